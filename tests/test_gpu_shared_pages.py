"""Requests whose table rows begin with the same pages, over PageTables, which
takes every page for its request's own: ended by a trim to the shared tokens and
a length of 0, they give back what is theirs and nothing else."""
import pytest
import torch

from neuralzip_amd.gpu import serving
from test_gpu_serving import DEVICE, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own", [[1, 1, 1], [16, 17, 40], [0, 5, 33]])
def test_requests_behind_shared_pages_end(own):
    book, shared = serving.PageTables(4, 8, 16, 20, device=DEVICE), 48
    book.extend(ints([0, 0, 0, 50]), 50)                 # the prefix, in a row of its own: three whole pages
    prefix = book.tables[3, :4].tolist()
    for r in range(3):
        book.tables[r, :3] = book.tables[3, :3]
        book.lengths[r] = shared
    assert (book.extend(ints(own + [0]), 200).status == serving.PAGES_OK).all()
    left = 20 - 4 - sum(-(-n // 16) for n in own)
    assert int(book.n_free) == left

    def pages():
        used = prefix + book.free[:int(book.n_free)].tolist()
        for r, n in enumerate(book.lengths.tolist()[:3]):
            used += book.tables[r, 3:max(3, -(-n // 16))].tolist()
        return sorted(used)
    assert pages() == list(range(20))
    # drafts refused: never below what is shared
    book.trim(ints([shared + max(n - 2, 0) for n in own] + [50]))
    assert pages() == list(range(20))
    for r in (1, 0, 2):
        keep = book.lengths.clone()
        keep[r] = shared
        book.trim(keep)
        book.lengths[r] = 0
        assert pages() == list(range(20))
    assert book.lengths.tolist() == [0, 0, 0, 50] and int(book.n_free) == 16
    book.release(torch.tensor([False, False, False, True], device=DEVICE))
    assert sorted(book.free.tolist()) == list(range(20)) and int(book.n_free) == 20
