"""PagedDecoder's bookkeeping, on small random models: on the CPU over the
operators in plain torch (plain_serving), and on the GPU over the kernels."""
import contextlib

import pytest
import torch

import plain_serving
from neuralzip_amd.gpu import paged
from neuralzip_amd.gpu.paged import PagedDecoder

VOCAB = 200
SIZES = dict(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, intermediate_size=96, num_hidden_layers=3,
             vocab_size=VOCAB, max_position_embeddings=256, tie_word_embeddings=False, pad_token_id=0, bos_token_id=1,
             eos_token_id=2)


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        plain_serving.install(monkeypatch)
    return request.param


def small_model(device, kind="llama", **config):
    from transformers import CONFIG_MAPPING, AutoModelForCausalLM
    torch.manual_seed(5)
    model = AutoModelForCausalLM.from_config(CONFIG_MAPPING[kind](**dict(SIZES, **config)))
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.dim() > 1:
                p.copy_(torch.randn(p.shape) * 0.15)
            else:
                p.add_(torch.randn(p.shape) * 0.1)
    return model.float().to(device).eval()


def prompt(n, seed=1):
    return torch.randint(3, VOCAB, (n,), generator=torch.Generator().manual_seed(seed))


def own_logits(model, ids):
    """The model's own logits after `ids`."""
    with torch.no_grad():
        return model(input_ids=torch.as_tensor(ids, device=model.device)[None], use_cache=False).logits[0, -1]


def agree(got, want):
    """Logits of a few layers' float32 sums of at most some hundred terms, in
    two orders: they differ by far less than 1e-3 of the largest."""
    return bool((got - want).abs().max() <= 1e-3 * want.abs().max())


@pytest.mark.parametrize("most", [20, 32, 33])
def test_requests_at_max_length_stay_as_they_are(device, most):
    """Whether or not max_length fills its pages: a request that has reached
    it gets no more tokens, nothing of its keys changes and nothing of the
    next request's history is written."""
    model = small_model(device)
    decoder = PagedDecoder(model, requests=2, max_length=most, repetition=1.3)
    long, short = prompt(most - 2, 1), prompt(3, 2)
    first, second = decoder.add(long), decoder.add(short)
    decoder.step(), decoder.step()
    assert decoder.tables.lengths.tolist() == [most, 5]
    keys, history = decoder.cache.clone(), decoder._history[first].clone()
    pages = decoder.tables.tables[first, :-(-most // 16)].long()
    for i in range(4):
        decoder.step()
        assert decoder.tables.lengths.tolist() == [most, 6 + i]
    assert torch.equal(decoder.cache[:, :, pages], keys[:, :, pages]) and torch.isfinite(decoder.cache).all()
    assert torch.equal(decoder._history[first], history)
    assert decoder._history[second, :3].tolist() == short.tolist()
