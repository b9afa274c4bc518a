"""PagedDecoder with prefixes, drafts, sampling and experts: calls at the edges
of what it takes. On the CPU over the operators in plain torch, and on the GPU
over the kernels."""
import pytest
import torch

import plain_more_serving
from neuralzip_amd.gpu.paged import PagedDecoder
from test_paged_decoder import prompt, small_model


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        plain_more_serving.install(monkeypatch)
    return request.param


@pytest.mark.parametrize("count", [0, 1, 3])
def test_numbers_are_two(device, count):
    """One vector would leave the other's numbers of the step before, which
    must not be used twice."""
    decoder = PagedDecoder(small_model(device), requests=2, max_length=40, temperature=0.8, drafts=1)
    decoder.add(prompt(5))
    sizes = (4, 2, 2)
    given = tuple(torch.full((n,), 0.5, dtype=torch.float64, device=device) for n in sizes)
    lengths = decoder.tables.lengths.tolist()
    with pytest.raises(ValueError, match="float64 vectors of 4 and 2"):
        decoder.step(numbers=given[:count])
    with pytest.raises(ValueError, match="float64 vectors of 4 and 2"):
        decoder.step(numbers=([0.5] * 4, [0.5] * 2))
    assert decoder.tables.lengths.tolist() == lengths
    decoder.step(numbers=given[:2])
    decoder.step(numbers=list(given[:2]))
    assert decoder.tables.lengths.tolist() == [lengths[0] + 2, 0]
