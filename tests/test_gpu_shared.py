"""Attention over shared keys (SharedPlan) and trimmed pages on the GPU against
plain implementations in 64 bits (whole numbers: in loops). The bound is that
of the other plan's attention, whose sums these are in another order."""
import random

import pytest
import torch

from neuralzip_amd.gpu import serving
from test_gpu_serving import (DEVICE, TYPES, attention_bound, filled_tables, ints, pages_of, plain_attention, randn)

pytestmark = pytest.mark.gpu


def shared_case(dtype, heads, kv_heads, dim, page, requests, seed=0, sharp=1.0, spare=2):
    """`requests`: (group, pages of its prefix, own tokens, rows) each; rows see
    one key fewer per row before the last. Everything that no context reaches
    holds NaN. Returns q, caches, tables, their host form, contexts, rows'
    requests and requests' groups."""
    rng = random.Random(seed)
    prefixes = {group: first for group, first, _, _ in requests if group >= 0}
    used = [pages_of(own, page) for _, _, own, _ in requests]
    order = list(range(sum(used) + sum(prefixes.values()) + spare))
    rng.shuffle(order)
    total = len(order)
    shared = {group: [order.pop() for _ in range(first)] for group, first in prefixes.items()}
    width = max(1, max(pages_of(own, page) + (first if group >= 0 else 0) for group, first, own, _ in requests)) + 1
    keys, values = (torch.full((total, kv_heads, page, dim), float("nan"), dtype=dtype, device=DEVICE) for _ in range(2))

    def fill(p, live):
        keys[p, :, :live] = randn(kv_heads, live, dim, seed=seed + 17 * p, dtype=dtype)
        values[p, :, :live] = randn(kv_heads, live, dim, seed=seed + 17 * p + 1, dtype=dtype)
    for pages in shared.values():
        for p in pages:
            fill(p, page)
    tables, contexts, of = [], [], []
    for r, (group, first, own, rows) in enumerate(requests):
        row = list(shared[group]) if group >= 0 else []
        before = len(row) * page
        for i in range(pages_of(own, page)):
            p = order.pop()
            row.append(p)
            fill(p, min(page, own - i * page))
        tables.append(row + [-1] * (width - len(row)))
        contexts += [max(0, before + own - rows + 1 + i) for i in range(rows)]
        of += [r] * rows
    q = randn(len(of), heads, dim, seed=seed + 1, dtype=dtype, scale=sharp)
    return q, keys, values, ints(tables), tables, contexts, of, [group for group, _, _, _ in requests]


def check_shared(dtype, heads, kv_heads, dim, page, requests, seed=0, sharp=1.0, scale=None, lengths=None):
    q, keys, values, tables, host, contexts, of, groups = shared_case(dtype, heads, kv_heads, dim, page, requests, seed,
                                                                      sharp)
    extra = {}
    if any(group >= 0 for group in groups):
        prefix = dict((group, first * page) for group, first, _, _ in requests if group >= 0)
        lengths = lengths or [prefix.get(g, 0) for g in range(max(groups) + 1)]
        extra = dict(groups=ints(groups), shared=ints(lengths))
    plan = serving.SharedPlan(ints(contexts), heads=heads, kv_heads=kv_heads, requests=ints(of), **extra)
    out = serving.paged_attention(q, keys, values, tables, plan, scale=scale)
    want, size, most = plain_attention(q, keys, values, host, contexts, of, dim ** -0.5 if scale is None else scale)
    bound = attention_bound(want, size, most, contexts, dim, dtype)
    assert ((out.double() - want).abs() <= bound).all(), ((out.double() - want).abs() / bound).max()
    # the same plan again, and made anew in its memory
    again = serving.paged_attention(q, keys, values, tables, plan, scale=scale, out=torch.empty_like(q))
    assert torch.equal(out, again)
    plan.update(ints(contexts), requests=ints(of), **extra)
    assert torch.equal(out, serving.paged_attention(q, keys, values, tables, plan, scale=scale))
    return plan


# one prefix for three, another for two, one that a single request has, and requests without
MIXED = [(0, 3, 5, 1), (1, 5, 0, 1), (0, 3, 1, 3), (-1, 0, 40, 2), (2, 2, 17, 4), (1, 5, 33, 5), (-1, 0, 0, 1),
         (0, 3, 64, 1), (-1, 0, 3, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 128, 160, 256])
def test_shared_keys_of_every_head_size(dtype, dim):
    check_shared(dtype, 4, 2, dim, 16, MIXED, seed=dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (3, 3), (8, 1), (14, 2), (32, 8), (16, 1), (17, 1), (71, 1),
                                             (40, 2), (33, 1), (64, 2)])
def test_shared_keys_of_grouped_heads(dtype, heads, kv_heads):
    check_shared(dtype, heads, kv_heads, 64, 32, [(0, 2, 7, 1), (0, 2, 40, 2), (-1, 0, 33, 3), (0, 2, 1, 1)], seed=heads)


@pytest.mark.parametrize("page", [16, 64, 256, 1024])
def test_shared_keys_of_every_page_size(page):
    check_shared(torch.bfloat16, 4, 2, 128, page, [(0, 1, 1, 1), (0, 1, page, 2), (0, 1, page + 1, 1), (-1, 0, 5, 5)],
                 seed=page)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("requests", [[(-1, 0, 5000, 9)], [(0, 300, 700, 2)] * 12, [(0, 100, 1, 1)] * 130,
                                      [(i % 7, 20 + i % 7, 30 * i, 1 + i % 3) for i in range(1, 40)],
                                      [(-1, 0, 0, 1)] * 5, [(-1, 0, 1, 1)], [(0, 4, 0, 1)] * 3],
                         ids=["drafts", "prefix", "many", "groups", "empty", "one", "nothing-own"])
def test_shared_keys_split_over_long_contexts(dtype, requests):
    check_shared(dtype, 8, 2, 64, 16, requests, seed=len(requests))


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_keys_of_sharp_and_flat_scores(dtype):
    for more in (dict(sharp=30.0), dict(sharp=1e-3), dict(scale=0.0), dict(scale=-0.3)):
        check_shared(dtype, 4, 1, 64, 16, [(0, 30, 200, 2), (0, 30, 33, 3)], **more)


@pytest.mark.parametrize("lengths", [[1], [15], [47], [48], [0], [-5]])
def test_prefixes_that_end_anywhere(lengths):
    """Fewer keys may be declared than are shared."""
    check_shared(torch.bfloat16, 8, 2, 64, 16, [(0, 3, 20, 1), (0, 3, 2, 2), (0, 3, 0, 1)], lengths=lengths)


def test_declared_prefixes_longer_than_contexts():
    """Past a row's context nothing is seen, whatever its group shares."""
    q, keys, values, tables, host, contexts, of, _ = shared_case(torch.float16, 4, 2, 64, 16, [(0, 6, 8, 1)] * 4)
    contexts = [90, 0, 5, 33]
    for declared in (96, 10 ** 6, 2 ** 31 - 1):
        plan = serving.SharedPlan(ints(contexts), heads=4, kv_heads=2, requests=ints(of), groups=ints([0] * 4),
                                  shared=ints([declared]))
        out = serving.paged_attention(q, keys, values, tables, plan)
        want, size, most = plain_attention(q, keys, values, host, contexts, of, 64 ** -0.5)
        assert ((out.double() - want).abs() <= attention_bound(want, size, most, contexts, 64, torch.float16)).all()


@pytest.mark.parametrize("rows", [1, 63, 64, 65, 1023, 1024, 1025, 2048])
def test_plans_of_many_rows(rows):
    requests = [(i % 5 if i % 3 else -1, 1 + i % 5, i % 4, 1) for i in range(rows)]
    check_shared(torch.bfloat16, 2, 1, 32, 16, requests, seed=rows)


def test_many_rows_of_one_request_and_many_groups():
    check_shared(torch.bfloat16, 4, 1, 32, 16, [(-1, 0, 2000, 1000), (-1, 0, 70, 48)])
    check_shared(torch.bfloat16, 4, 1, 32, 16, [(i // 2, 1, 1 + i % 20, 1) for i in range(2000)])


def test_plans_cover_every_row_and_key_once():
    for requests in (MIXED, [(0, 100, 300, 2)] * 20, [(-1, 0, 3000, 40)]):
        for heads, kv_heads in ((8, 2), (40, 1), (4, 4)):
            *_, contexts, of, groups = shared_case(torch.bfloat16, heads, kv_heads, 16, 16, requests)
            first = {g: n * 16 for g, n, _, _ in requests if g >= 0}
            extra = dict(groups=ints(groups), shared=ints([first.get(g, 0) for g in range(max(groups) + 1)])) \
                if first else {}
            plan = serving.SharedPlan(ints(contexts), heads=heads, kv_heads=kv_heads, requests=ints(of), **extra)
            order = plan.order.tolist()
            seen = [[0] * max(contexts + [1]) for _ in of]
            for member, n, request, begin, end, _, _, _ in plan.items.tolist():
                for row in order[member:member + n]:
                    assert of[row] == request or groups[of[row]] == groups[request] >= 0
                    assert end <= max(contexts[row], 0) or begin == end
                    for t in range(begin, end):
                        seen[row][t] += 1
            for row, n in zip(seen, contexts):
                assert row[:n] == [1] * n


@pytest.mark.parametrize("rows, shared", [(2, None), (2048, None), (2, 2 ** 31 - 1), (2048, 2 ** 31 - 1), (300, 2 ** 30 + 5)])
def test_plans_of_the_longest_contexts(rows, shared):
    """Counts of items and ends of keys stay inside 32 bits. (Only planned.)"""
    extra = dict(groups=ints([0] * rows), shared=ints([shared])) if shared else {}
    plan = serving.SharedPlan(ints([2 ** 31 - 1] * rows), heads=8, kv_heads=8, **extra)
    order, seen = plan.order.tolist(), [[] for _ in range(rows)]
    for member, n, _, begin, end, _, _, _ in plan.items.tolist():
        for row in order[member:member + n]:
            seen[row].append((begin, end))
    for items in seen:
        items.sort()
        assert items[0][0] == 0 and items[-1][1] == 2 ** 31 - 1
        assert all(a[1] == b[0] for a, b in zip(items, items[1:]))


def test_what_is_not_finite_stays_where_it_is_seen():
    """A key that one row sees and its neighbour does not may have any value."""
    q, keys, values, tables, host, contexts, of, _ = shared_case(torch.bfloat16, 4, 1, 64, 16, [(-1, 0, 45, 4)] * 2)
    page, place = host[0][44 // 16], 44 % 16     # the last row's own key
    for bad in (float("inf"), float("nan")):
        v = values.clone()
        v[page, :, place] = bad
        plan = serving.SharedPlan(ints(contexts), heads=4, kv_heads=1, requests=ints(of))
        out = serving.paged_attention(q, keys, v, tables, plan)
        clean = serving.paged_attention(q, keys, values, tables, plan)
        assert not torch.isfinite(out[3]).any()
        keep = [0, 1, 2, 4, 5, 6, 7]
        assert torch.equal(out[keep], clean[keep])


def test_masked_pages_and_requests():
    q, keys, values, tables, host, contexts, of, _ = shared_case(torch.bfloat16, 4, 2, 64, 16, [(0, 3, 20, 2)] * 3)
    for r in range(3):
        host[r][1] = 10 ** 6                     # a page that there is not: masked
    of = [0, 0, 1, 1, -1, 7]
    plan = serving.SharedPlan(ints(contexts), heads=4, kv_heads=2, requests=ints(of), groups=ints([0] * 3),
                              shared=ints([48]))
    out = serving.paged_attention(q, keys, values, ints(host), plan)
    assert (out[4:] == 0).all()
    # without the masked page's 16 keys
    kept = [[row[0]] + row[2:] for row in host]
    want, size, most = plain_attention(q[:4], keys, values, kept, [n - 16 for n in contexts[:4]], of[:4], 64 ** -0.5)
    assert ((out[:4].double() - want).abs() <= attention_bound(want, size, most, contexts, 64, torch.bfloat16)).all()


def test_strided_caches_and_outputs():
    q, keys, values, tables, host, contexts, of, groups = shared_case(torch.float16, 6, 2, 48, 16, MIXED)
    wide = torch.full((*keys.shape[:3], 2, 64), float("nan"), dtype=q.dtype, device=DEVICE).transpose(1, 2)
    wide[..., 0, 8:56], wide[..., 1, 8:56] = keys.transpose(1, 2), values.transpose(1, 2)
    k, v = (wide[..., i, 8:56].transpose(1, 2) for i in range(2))
    extra = dict(groups=ints(groups), shared=ints([48, 80, 32]))
    plan = serving.SharedPlan(ints(contexts), heads=6, kv_heads=2, requests=ints(of), **extra)
    out = torch.zeros(len(of), 8, 64, dtype=q.dtype, device=DEVICE)
    view = serving.paged_attention(q, k, v, tables, plan, out=out[:, 1:7, 8:56])
    assert torch.equal(view, serving.paged_attention(q, keys, values, tables, plan))
    out[:, 1:7, 8:56] = 0
    assert (out == 0).all()


def test_a_captured_plan_follows_its_contexts():
    """Plan and attention in one graph, replayed over growing requests with
    eager work between."""
    q, keys, values, tables, host, contexts, of, groups = shared_case(torch.bfloat16, 8, 2, 64, 16,
                                                                      [(0, 4, 60, 2), (0, 4, 60, 2), (-1, 0, 60, 2)])
    now, extra = ints([1] * 6), dict(groups=ints(groups), shared=ints([64]))
    plan = serving.SharedPlan(now, heads=8, kv_heads=2, requests=ints(of), **extra)
    out = torch.empty_like(q)
    requests = ints(of)
    serving.paged_attention(q, keys, values, tables, plan, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(now, requests=requests, **extra)
        serving.paged_attention(q, keys, values, tables, plan, out=out)
    for grown in ([65, 66, 70, 71, 1, 2], contexts, [0, 1, 64, 65, 59, 60], [124, 123, 1, 1, 0, 0]):
        now.copy_(ints(grown))
        graph.replay()
        torch.cuda.synchronize()
        want, size, most = plain_attention(q, keys, values, host, grown, of, 64 ** -0.5)
        assert ((out.double() - want).abs() <= attention_bound(want, size, most, contexts, 64, torch.bfloat16)).all()
        eager = serving.SharedPlan(ints(grown), heads=8, kv_heads=2, requests=requests, **extra)
        assert torch.equal(out, serving.paged_attention(q, keys, values, tables, eager))


def test_plans_of_no_rows_and_no_groups():
    none = ints([])
    plan = serving.SharedPlan(none, heads=4, kv_heads=2, requests=none)
    q, caches = randn(0, 4, 64), [randn(3, 2, 16, 64) for _ in range(2)]
    assert serving.paged_attention(q, *caches, ints([[0, 1]]), plan).shape == (0, 4, 64)
    q = randn(2, 4, 64, seed=1)
    one = serving.SharedPlan(ints([20, 9]), heads=4, kv_heads=2, groups=ints([-1, 7]), shared=none)
    two = serving.AttentionPlan(ints([20, 9]), heads=4, kv_heads=2)
    tables = ints([[0, 1], [2, 0]])
    got, want = (serving.paged_attention(q, *caches, tables, plan) for plan in (one, two))
    assert (got - want).abs().max() <= 2.0 ** -18 * caches[1].abs().max()


@pytest.mark.parametrize("change, message", [
    (dict(contexts=[3, 4, 5]), "contexts"), (dict(requests=[0]), "requests"), (dict(groups=[0]), "groups"),
    (dict(shared=[1, 2]), "shared"), (dict(groups=None, shared=None), "as when the plan was made")])
def test_updates_of_other_sizes_are_refused(change, message):
    given = dict(contexts=[3, 4], requests=[0, 1], groups=[0, 0], shared=[2])
    plan = serving.SharedPlan(**{k: ints(v) for k, v in given.items()}, heads=2, kv_heads=1)
    with pytest.raises(ValueError, match=message):
        plan.update(**{k: None if v is None else ints(v) for k, v in dict(given, **change).items()})


def test_refusals_that_need_the_device():
    with pytest.raises(ValueError, match="2048 rows"):
        serving.SharedPlan(ints([1] * 2049), heads=2, kv_heads=1)
    with pytest.raises(ValueError, match="go together"):
        serving.SharedPlan(ints([1]), heads=2, kv_heads=1, groups=ints([0]))
    with pytest.raises(ValueError, match="vectors"):
        serving.SharedPlan(ints([1]), heads=2, kv_heads=1, groups=ints([[0]]), shared=ints([1]))
    plan = serving.SharedPlan(ints([1, 2]), heads=2, kv_heads=1)
    q, caches, tables = randn(2, 2, 64), [randn(3, 1, 16, 64) for _ in range(2)], ints([[0], [1]])
    with pytest.raises(ValueError, match="q must be"):
        serving.paged_attention(randn(3, 2, 64), *caches, tables, plan)
    with pytest.raises(ValueError, match="Caches must"):
        serving.paged_attention(q, caches[0], caches[1][:2], tables, plan)
    with pytest.raises(ValueError, match="tables must"):
        serving.paged_attention(q, *caches, tables.long(), plan)
    with pytest.raises(ValueError, match="no backward"):
        serving.paged_attention(q.clone().requires_grad_(), *caches, tables, plan)


def test_a_side_stream():
    q, keys, values, tables, _, contexts, of, groups = shared_case(torch.bfloat16, 8, 2, 64, 16, MIXED)
    extra = dict(groups=ints(groups), shared=ints([48, 80, 32]))
    plan = serving.SharedPlan(ints(contexts), heads=8, kv_heads=2, requests=ints(of), **extra)
    want = serving.paged_attention(q, keys, values, tables, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = serving.SharedPlan(ints(contexts), heads=8, kv_heads=2, requests=ints(of), stream=side, **extra)
    got = serving.paged_attention(q, keys, values, tables, other, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


# ---------------------------------------------------------------------- trim

def plain_trim(lengths, keep, tables, free, n_free, page):
    free, top, after = list(free), n_free, []
    for r, (n, k) in enumerate(zip(lengths, keep)):
        k = min(max(k, 0), n)
        for j in range(pages_of(k, page), pages_of(n, page)):
            free[top] = tables[r][j]
            top += 1
        after.append(k)
    return after, free, top


@pytest.mark.parametrize("requests", [1, 5, 63, 64, 65, 257, 1025])
@pytest.mark.parametrize("advance", [False, True])
def test_trim_follows_the_rules(requests, advance):
    rng = random.Random(requests)
    lengths = [rng.choice((0, 1, 16, 17, 100, 500)) for _ in range(requests)]
    keep = [rng.choice((-3, 0, 1, 15, 16, 17, 90, 99, 100, 2 ** 31 - 1)) for _ in range(requests)]
    book, tables, free, n_free = filled_tables(lengths, 16, 33, 7, seed=requests)
    after, stack, top = plain_trim(lengths, keep, tables, free, n_free, 16)
    out = book.trim(ints(keep), advance=advance)
    assert out.lengths.tolist() == after and out.n_free.item() == top and book.free.tolist() == stack
    assert book.lengths.tolist() == (after if advance else lengths)
    assert book.n_free.item() == (top if advance else n_free) and book.tables.tolist() == tables


def test_trimmed_pages_are_given_out_again():
    book = serving.PageTables(3, 8, 16, 12, device=DEVICE)
    book.extend(ints([40, 17, 60]), 200)
    pages = book.tables.tolist()
    book.trim(ints([33, 16, 0]))
    assert book.lengths.tolist() == [33, 16, 0] and book.n_free.item() == 12 - 3 - 1
    step = book.extend(ints([0, 1, 100]), 200)
    assert step.status.tolist() == [0, 0, 0]
    taken = book.tables.tolist()
    used = taken[0][:3] + taken[1][:2] + taken[2][:7]
    assert sorted(used) == list(range(12)) and taken[0][:3] == pages[0][:3] and taken[1][:1] == pages[1][:1]
