"""Shared attention, verification, routing and experts on tensors whose parts
lie more than 2^31 or 2^32 elements from one another: the same bits as from dense
ones."""
import pytest
import torch

from neuralzip_amd.gpu import serving
from test_gpu_serving import DEVICE, ints, randn
from test_gpu_shared import shared_case

pytestmark = pytest.mark.gpu

FAR = (1 << 31) + 64


@pytest.fixture
def memory():
    yield [torch.empty(2 * FAR + 16384, dtype=torch.bfloat16, device=DEVICE) for _ in range(2)]
    torch.cuda.empty_cache()


def test_shared_attention_on_far_pages():
    pages, kv_heads, page, dim = 70_000, 4, 256, 64
    assert (pages - 3) * kv_heads * page * dim > 1 << 32
    keys, values = (torch.empty(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=DEVICE) for _ in range(2))
    small = [randn(4, kv_heads, page, dim, seed=s, dtype=torch.bfloat16) for s in (1, 2)]
    places = [pages - 1, 0, pages - 3, pages - 2]
    for i, p in enumerate(places):
        keys[p], values[p] = small[0][i], small[1][i]
    # two pages shared, then one of its own for each of two requests, of three rows and one
    tables = [[0, 1, 2], [0, 1, 3]]
    contexts, of = ints([650, 651, 652, 530]), ints([0, 0, 0, 1])
    q = randn(4, 8, dim, seed=3, dtype=torch.bfloat16)
    plan = serving.SharedPlan(contexts, heads=8, kv_heads=kv_heads, requests=of, groups=ints([0, 0]), shared=ints([512]))
    want = serving.paged_attention(q, *small, ints(tables), plan)
    got = serving.paged_attention(q, keys, values, ints([[places[i] for i in row] for row in tables]), plan)
    assert torch.equal(got, want)
    del keys, values
    torch.cuda.empty_cache()


def test_shared_attention_of_far_rows(memory):
    q, keys, values, tables, _, contexts, of, groups = shared_case(torch.bfloat16, 4, 2, 64, 16, [(0, 3, 20, 2), (0, 3, 5, 1)])
    plan = serving.SharedPlan(ints(contexts), heads=4, kv_heads=2, requests=ints(of), groups=ints(groups), shared=ints([48]))
    want = serving.paged_attention(q, keys, values, tables, plan)
    wide, out = (m.as_strided((3, 4, 64), (FAR, 64, 1)) for m in memory)
    wide.copy_(q)
    assert torch.equal(serving.paged_attention(wide, keys, values, tables, plan, out=out), want)


def test_verification_of_far_rows(memory):
    logits, tokens = randn(3, 5000, seed=1, dtype=torch.bfloat16, scale=3.0), torch.tensor([0, 7, 9], device=DEVICE)
    q = randn(3, 5000, seed=2).softmax(-1)
    accept, sample = (torch.full((n,), u, dtype=torch.float64, device=DEVICE) for n, u in ((3, 0.1), (1, 0.6)))
    wide = memory[0].as_strided((3, 5000), (FAR, 1))
    wide.copy_(logits)
    far = memory[1].view(torch.float32).as_strided((3, 5000), (FAR // 2, 1))
    far.copy_(q)
    for draft, dense in ((None, None), (far, q)):
        for drafts in ([0, 7, 9], [0, int(logits[0].argmax()), int(logits[1].argmax())]):
            tokens.copy_(torch.tensor(drafts))
            for starts in ([0, 3], [2, 3]):
                got, want = (serving.verify_drafts(x, tokens, ints(starts), accept, sample, draft_probs=p)
                             for x, p in ((wide, draft), (logits, dense)))
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_experts_of_far_rows_and_far_experts(memory):
    x, gate_up, down = (randn(*s, seed=i, dtype=torch.bfloat16) for i, s in enumerate(((3, 64), (3, 96, 64), (3, 64, 48))))
    router = randn(3, 64, seed=5, dtype=torch.bfloat16)
    ids, weights = serving.route_experts(x, router, 2)
    want = serving.expert_mlp(x, ids, weights, gate_up, down)
    far_x, out = (m.as_strided((3, 64), (FAR, 1)) for m in memory)
    far_x.copy_(x)
    for got, same in zip(serving.route_experts(far_x, router, 2), (ids, weights)):
        assert torch.equal(got, same)
    assert torch.equal(serving.expert_mlp(far_x, ids, weights, gate_up, down, out=out), want)
    # rows end before 128, experts' matrices begin there
    far_up, far_down = (m.as_strided(t.shape, (FAR, t.shape[2], 1), 128) for m, t in zip(memory, (gate_up, down)))
    far_up.copy_(gate_up), far_down.copy_(down)
    assert torch.equal(serving.expert_mlp(far_x, ids, weights, far_up, far_down, out=out), want)
