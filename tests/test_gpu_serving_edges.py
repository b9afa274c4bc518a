"""Edges of the serving-step operators on the GPU, beside test_gpu_serving.py,
whose plain forms and tolerances they use."""
import pytest
import torch

from neuralzip_amd.gpu import serving
from test_gpu_serving import DEVICE, ints, unit

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits, tail", [(45.0, 60000.0), (60.0, -60000.0), (130.0, 60000.0)])
def test_attention_of_many_keys_of_next_to_no_weight(dtype, bits, tail):
    """100000 keys of 2^-bits of the first one's weight, with values as large
    as fp16 has, beside a value of 0, in as many rows as leave each row in one
    item. Its four wavefronts take every fourth 32 keys and weigh them against
    their own largest; in the one with the first key fp16 holds weights in
    multiples of 2^-39 of the largest, so each is off by at most 2^-40 of it.
    bf16 and fp32 reach down to 2^-126."""
    n, dim, page, rows = 100_001, 64, 1024, 256
    pages = -(-n // page)
    keys, values = (torch.zeros(pages, 1, page, dim, dtype=dtype, device=DEVICE) for _ in range(2))
    values += tail
    keys[0, 0, 0, 0], values[0, 0, 0] = 1.0, 0.0
    q = torch.zeros(rows, 1, dim, dtype=dtype, device=DEVICE)
    q[..., 0] = bits * 0.6931
    plan = serving.AttentionPlan(ints([n] * rows), heads=1, kv_heads=1)
    assert (plan.items[:rows, 5] == 1).all()
    tables = torch.arange(pages, dtype=torch.int32, device=DEVICE)[None].expand(rows, -1).contiguous()
    got = serving.paged_attention(q, keys, values, tables, plan, scale=1.0).double()
    weight = (-q[0, 0, 0].double()).exp() * (n - 1)
    want, size = (weight / (1 + weight) * values[0, 0, 1, 0].double()).item(), abs(values[0, 0, 1, 0].item())
    # bf16 splits a weight in two halves of 8 bits; the sums of 32 bits err by n roundings
    bound = unit(dtype) * abs(want) + abs(want) * (2.0 ** -14 + n * 2.0 ** -24) + 2.0 ** -25
    if dtype == torch.float16:
        bound += (n / 4 + 32) * 2.0 ** -40 * size
    assert ((got - want).abs() <= bound).all(), (got.flatten()[0].item(), want, bound)


def test_attention_passes_on_infinite_values_of_full_weight():
    """Weights that 16 bits hold whole (here 1, 1/2 and 1/4 of the largest)
    leave no rest, which must not turn an infinite value into NaN."""
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        keys, values = (torch.zeros(1, 1, 16, 64, dtype=dtype, device=DEVICE) for _ in range(2))
        for i, weight in enumerate((0.0, -0.6931, -1.3863)):
            keys[0, 0, i, 0] = weight
            values[0, 0, i, i] = float("-inf") if i == 1 else float("inf")
        q = torch.zeros(1, 1, 64, dtype=dtype, device=DEVICE)
        q[..., 0] = 1.0
        plan = serving.AttentionPlan(ints([3]), heads=1, kv_heads=1)
        out = serving.paged_attention(q, keys, values, ints([[0]]), plan, scale=1.0)[0, 0]
        assert out[:3].tolist() == [float("inf"), float("-inf"), float("inf")] and not out[3:].any()


def test_attention_of_scores_that_are_minus_infinity():
    """Such keys have no weight, as masked ones; a row of nothing else gives zeros."""
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        keys = torch.zeros(2, 1, 16, 64, dtype=dtype, device=DEVICE)
        values = torch.ones(2, 1, 16, 64, dtype=dtype, device=DEVICE)
        keys[0, 0, :, 0], keys[1, 0, 1:, 0], values[1, 0, 0] = float("-inf"), float("-inf"), 3.0
        q = torch.zeros(2, 1, 64, dtype=dtype, device=DEVICE)
        q[..., 0] = 1.0
        plan = serving.AttentionPlan(ints([16, 9]), heads=1, kv_heads=1)
        out = serving.paged_attention(q, keys, values, ints([[0], [1]]), plan)
        assert not out[0].any() and (out[1] == 3).all()


@pytest.mark.parametrize("heads, kv_heads", [(32, 8), (8, 1), (64, 2)])
@pytest.mark.parametrize("contexts", [[0], [128], [129], [257], [2001], [8191], [8192], [8193], [100_000], [0, 0, 5000],
                                      [129] * 40, [200] * 1500, [100_000, 7] * 40, list(range(1, 8192, 128)),
                                      [2 ** 31 - 1, 5], [30, 400, 50, 9000] * 300])
def test_plans_keep_their_bounds(contexts, heads, kv_heads):
    """The longest item, the number of items and the even cut of rows, as
    nz_attention_plan's declaration has them."""
    plan = serving.AttentionPlan(ints(contexts), heads=heads, kv_heads=kv_heads)
    target = 256 // (kv_heads * -(-(heads // kv_heads) // 16))
    n, keys, longest = -(-len(contexts) // target) * target, sum(contexts), max(contexts)
    least = min(max(-(-(-(-longest // 32)) // 16), 4), 16)

    def shortest(limit):
        """In 32 keys; items get fewer as they get longer."""
        low, high = least, max(least, -(-longest // 32))
        while low < high:
            middle = (low + high) // 2
            if sum(max(-(-c // (32 * middle)), 1) for c in contexts) <= limit:
                high = middle
            else:
                low = middle + 1
        return low
    length = 32 * shortest(n)
    if length > 32 * least and 2 * length * n > 3 * keys and 2 * length * target > keys:
        n, length = n + target, 32 * shortest(n + target)
    items = [item for item in plan.items.tolist() if item[0] >= 0]
    assert len(contexts) <= len(items) <= n <= plan.capacity
    for row, context in enumerate(contexts):
        sizes = [item[3] - item[2] for item in items if item[0] == row]
        assert sum(sizes) == context and len(sizes) <= max(-(-context // length), 1)
        assert len(set(sizes[:-1])) <= 1 and all(0 < sizes[-1] <= s <= length for s in sizes[:-1])
        assert all(s % 32 == 0 and 2 * s > length for s in sizes[:-1]) and sizes[-1] <= length
