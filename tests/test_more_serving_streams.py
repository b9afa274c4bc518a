"""Memory of shared plans', trims', verifications' and experts' calls on a
stream of their own: what a call was given is kept until the stream is done
with it. Without a GPU the records are watched; with one, a busy stream reads
what the caller has let go."""
import pytest
import torch

from neuralzip_amd.gpu import serving
from test_serving_streams import DEVICE, Lane, Watched, addresses, calls, kept, random  # noqa: F401


def test_trims_and_routes_keep_their_tensors(calls):  # noqa: F811
    book, lane, keep = serving.PageTables(3, 4, 16, 8, device="cpu"), Lane(), torch.zeros(3, dtype=torch.int32)
    book.trim(keep)
    assert not Watched.records
    book.trim(keep, stream=lane)
    state = addresses(book.lengths, book.tables, book.free, book.n_free)
    assert {a for a, s in Watched.records} >= state | addresses(keep) and all(s is lane for _, s in Watched.records)
    Watched.records = []
    x, weight, bias = torch.zeros(2, 64), torch.zeros(4, 64), torch.zeros(4)
    serving.route_experts(x, weight, 2, bias=bias)
    assert not Watched.records
    serving.route_experts(x, weight, 2, bias=bias, stream=lane)
    assert {a for a, _ in Watched.records} >= addresses(x, weight, bias)


def test_experts_keep_their_tensors(calls):  # noqa: F811
    x, ids, weights = torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2)
    gate_up, down, out, lane = torch.zeros(4, 96, 64), torch.zeros(4, 64, 48), torch.zeros(2, 64), Lane()
    serving.expert_mlp(x, ids, weights, gate_up, down)
    assert not Watched.records
    serving.expert_mlp(x, ids, weights, gate_up, down, out=out, stream=lane)
    assert {a for a, _ in Watched.records} >= addresses(x, ids, weights, gate_up, down, out)


# ---------------------------------------------------------------- on the GPU

@pytest.mark.gpu
def test_experts_read_what_the_caller_has_let_go():
    x, gate_up, down = (random(*s, seed=i) for i, s in enumerate(((9, 128), (8, 192, 128), (8, 128, 96))))
    ids, weights = torch.randint(0, 8, (9, 2), device=DEVICE), torch.rand(9, 2, device=DEVICE)
    tensors = [x, ids, weights, gate_up, down]
    del x, ids, weights, gate_up, down
    assert kept(tensors, serving.expert_mlp)
    assert kept([random(9, 128, seed=4), random(8, 128, seed=5)], lambda x, router, stream: serving.route_experts(x, router, 2, stream=stream)[1])


@pytest.mark.gpu
def test_verifications_read_what_the_caller_has_let_go():
    logits, probs = random(6, 5000, seed=1), torch.rand(6, 5000, device=DEVICE)
    tokens, starts = torch.arange(6, device=DEVICE), torch.tensor([0, 3, 6], dtype=torch.int32, device=DEVICE)
    accept, sample = torch.rand(6, device=DEVICE, dtype=torch.float64), torch.rand(2, device=DEVICE, dtype=torch.float64)
    temperature = torch.full((2,), 0.7, device=DEVICE)

    def call(*tensors, stream):
        accepted, following = serving.verify_drafts(*tensors[:5], draft_probs=tensors[5], temperature=tensors[6], stream=stream)
        if stream is None:
            return torch.cat((accepted.long(), following))
        with torch.cuda.stream(stream):
            return torch.cat((accepted.long(), following))
    tensors = [logits, tokens, starts, accept, sample, probs, temperature]
    del logits, tokens, starts, accept, sample, probs, temperature
    assert kept(tensors, call)


@pytest.mark.gpu
def test_shared_plans_read_what_the_caller_has_let_go():
    keys, values = random(12, 2, 16, 64, seed=1), random(12, 2, 16, 64, seed=2)
    q = random(6, 8, 64, seed=3)
    contexts = torch.tensor([40, 41, 60, 61, 50, 51], dtype=torch.int32, device=DEVICE)
    requests = torch.tensor([0, 0, 1, 1, 2, 2], dtype=torch.int32, device=DEVICE)
    tables = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 6, 7]], dtype=torch.int32, device=DEVICE)
    groups, shared = (torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in ([0, 0, 0], [32]))

    def call(q, keys, values, tables, contexts, requests, groups, shared, stream):
        plan = serving.SharedPlan(contexts, heads=8, kv_heads=2, requests=requests, groups=groups, shared=shared,
                                  stream=stream)
        return serving.paged_attention(q, keys, values, tables, plan, stream=stream)
    tensors = [q, keys, values, tables, contexts, requests, groups, shared]
    del q, keys, values, tables, contexts, requests, groups, shared
    assert kept(tensors, call)


@pytest.mark.gpu
def test_plans_used_on_another_stream_than_their_own():
    keys, values, q = random(40, 2, 16, 64, seed=1), random(40, 2, 16, 64, seed=2), random(4, 8, 64, seed=3)
    contexts = torch.tensor([600, 601, 602, 603], dtype=torch.int32, device=DEVICE)
    requests = torch.zeros(4, dtype=torch.int32, device=DEVICE)
    tables = torch.randperm(40, device=DEVICE).int()[None].contiguous()
    plan = serving.SharedPlan(contexts, heads=8, kv_heads=2, requests=requests)
    want = serving.paged_attention(q, keys, values, tables, plan)
    lanes = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    # calls with one plan may overlap: each stream has its scratch
    outs = []
    for _ in range(4):
        for lane in lanes:
            outs.append(serving.paged_attention(q, keys, values, tables, plan, stream=lane))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)
