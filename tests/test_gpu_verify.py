"""verify_drafts on the GPU against the definition in 64 bits, request by
request. Its results are whole numbers and have to be equal: the sums that they
are taken from differ by a few times 2^-53 of their size, and so does the
chance that a number falls between two of them."""
import math

import numpy as np
import pytest
import torch

from neuralzip_amd.gpu import serving

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def chances(logits, t):
    """A row's probabilities (zeros where nothing is left)."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    if not t > 0:
        p = np.zeros_like(x)
        p[int(x.argmax())] = 1.0
        return p
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / t)))
    return p / p.sum()


def definition(logits, tokens, starts, accept, sample, probs, temperature):
    accepted, following = [], []
    vocab = logits.shape[1]
    for r in range(len(starts) - 1):
        first, end = starts[r], starts[r + 1]
        if first >= end:
            accepted.append(0), following.append(-1)
            continue
        t = 1.0 if temperature is None else temperature[r]
        for row in range(first, end):
            p = chances(logits[row], t)
            weights = p
            if row + 1 == end:
                break
            d = tokens[row + 1]
            if not 0 <= d < vocab or p.sum() == 0:
                break
            q = probs[row].astype(np.float64) if probs is not None else (np.arange(vocab) == d).astype(np.float64)
            if not accept[row] * q[d] < p[d]:
                with np.errstate(invalid="ignore"):
                    weights = np.where(p > q, p - q, 0.0)
                weights = weights if weights.sum() > 0 else p
                break
        sums = np.cumsum(weights)
        over = np.flatnonzero((sums > sample[r] * sums[-1]) & (weights > 0))
        some = np.flatnonzero(weights > 0)
        accepted.append(row - first)
        following.append(int(over[0]) if len(over) else int(some[-1]) if len(some) else -1)
    return accepted, following


def run(logits, tokens, starts, accept, sample, probs=None, temperature=None):
    def on(x, dtype):
        return None if x is None else torch.as_tensor(np.asarray(x), dtype=dtype).to(DEVICE)
    logits = logits.to(DEVICE)
    got = serving.verify_drafts(logits, on(tokens, torch.int64), on(starts, torch.int32), on(accept, torch.float64),
                                on(sample, torch.float64), draft_probs=on(probs, torch.float32),
                                temperature=on(temperature, torch.float32))
    return got[0].tolist(), got[1].tolist()


def check(logits, tokens, starts, accept, sample, probs=None, temperature=None):
    t = None if temperature is None else np.float32(temperature).astype(np.float64)
    want = definition(logits.double().numpy(), tokens, starts, accept, sample, probs, t)
    assert run(logits, tokens, starts, accept, sample, probs, temperature) == tuple(want)
    return want


def case(dtype, vocab, drafts, probs, seed=0, pad=2, sharp=3.0):
    """Random logits, drafts that are likely to be accepted, some not."""
    rng = np.random.default_rng(seed)
    starts = np.concatenate(([0], np.cumsum([k + 1 for k in drafts]))).tolist()
    rows = starts[-1] + pad
    logits = torch.from_numpy(sharp * rng.standard_normal((rows, vocab))).to(dtype)
    p = np.stack([chances(x, 1.0) for x in logits.double().numpy()]) if rows else np.zeros((0, vocab))
    q = None
    if probs:
        q = np.maximum(p * np.exp(0.3 * rng.standard_normal(p.shape)), 1e-30)
        q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    tokens = np.zeros(rows, dtype=np.int64)
    for row in range(rows - 1):
        chance = q[row].astype(np.float64) if probs else p[row]
        tokens[row + 1] = rng.choice(vocab, p=chance / chance.sum()) if rng.random() < 0.8 else p[row].argmax()
    return (logits, tokens.tolist(), starts, rng.random(rows) * (1.0 if probs else 0.3), rng.random(len(drafts)), q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 300, 4095, 4096, 4097, 9001])
@pytest.mark.parametrize("probs", [False, True])
def test_drafts_against_the_definition(dtype, vocab, probs):
    seen = set()
    for seed in range(4):
        drafts = [0, 3, -1, 5, 1, 2, 0, -1, 4, 17, 40]
        one = case(dtype, vocab, drafts, probs, seed=seed + vocab)
        rng = np.random.default_rng(seed)
        for temperature in (None, rng.random(len(drafts)) + 0.3, [0.0, 1.0, 0.0, -1.0, 2.0, 0.1, 0.7, 0.0, 1e-6, 1.0, 50.0]):
            seen.update(check(*one, temperature=temperature)[0])
    if vocab >= 300:
        assert len(seen) > 1      # drafts were accepted and refused


def test_many_requests():
    for n in (63, 64, 65, 700, 5000):
        drafts = [(i * 7) % 4 - 1 for i in range(n)]
        check(*case(torch.bfloat16, 40, drafts, False, seed=n))


@pytest.mark.parametrize("vocab", [151936, 1 << 22])
def test_large_vocabularies(vocab):
    check(*case(torch.bfloat16, vocab, [1, 0], True, pad=0))
    check(*case(torch.float32, vocab, [2], False, pad=0, sharp=0.1))


def even(vocab, dtype=torch.float32, rows=1):
    """Logits of 2^-k each: sums of them are exact."""
    return torch.zeros(rows, vocab, dtype=dtype)


def test_numbers_on_the_border():
    # the first token at which the sum exceeds the number
    for i in range(8):
        assert run(even(8), [0], [0, 1], [0.0], [i / 8]) == ([0], [i])
        assert run(even(8), [0], [0, 1], [0.0], [i / 8 + 2.0 ** -50]) == ([0], [i])
    assert run(even(1 << 14), [0], [0, 1], [0.0], [4096 / (1 << 14)]) == ([0], [4096])
    assert run(even(1 << 14), [0], [0, 1], [0.0], [4096 / (1 << 14) - 2.0 ** -50]) == ([0], [4095])
    assert run(even(8), [0], [0, 1], [0.0], [1.0 - 2.0 ** -53]) == ([0], [7])
    assert run(even(8), [0], [0, 1], [0.0], [1.0]) == ([0], [7])       # not from [0, 1): the last token
    # accepted only below p: certain drafts of p = 1/8
    two = even(8, rows=2)
    assert run(two, [0, 5], [0, 2], [0.125, 0.0], [0.5])[0] == [0]
    assert run(two, [0, 5], [0, 2], [math.nextafter(0.125, 0.0), 0.0], [0.5])[0] == [1]
    # without token 5, seven are left
    assert run(two, [0, 5], [0, 2], [0.9, 0.0], [5.5 / 7]) == ([0], [6])
    assert run(two, [0, 5], [0, 2], [0.9, 0.0], [4.5 / 7]) == ([0], [4])
    assert run(two, [0, 7], [0, 2], [0.9, 0.0], [1.0 - 2.0 ** -53]) == ([0], [6])
    # q of a quarter: accepted below half of the numbers
    q = np.zeros((2, 8), dtype=np.float32)
    q[0, :4] = 0.25
    assert run(two, [0, 3], [0, 2], [0.5, 0.0], [0.0], q) == ([0], [4])
    assert run(two, [0, 3], [0, 2], [math.nextafter(0.5, 0.0), 0.0], [0.3], q) == ([1], [2])
    for i in range(4):
        assert run(two, [0, 3], [0, 2], [0.5, 0.0], [i / 4], q) == ([0], [4 + i])


def test_nothing_left_of_a_refusal():
    """Where the draft's probabilities are the model's, a refusal (by a number
    that is not below 1) picks from the model's."""
    q = np.full((2, 8), 0.125, dtype=np.float32)
    assert run(even(8, rows=2), [0, 3], [0, 2], [1.0, 0.0], [0.4], q) == ([0], [3])
    one = torch.tensor([[0.0, -math.inf], [0.0, 0.0]])
    assert run(one, [0, 0], [0, 2], [1.0, 0.0], [0.4]) == ([0], [0])    # the only token is refused
    assert run(one, [0, 0], [0, 2], [0.9, 0.0], [0.6]) == ([1], [1])


def test_tokens_that_are_no_drafts():
    logits, _, _, _, _, q = case(torch.float32, 50, [3], True)
    for bad in (-1, 50, 2 ** 40, -2 ** 62):
        for probs in (None, q):
            for u in (0.0, 0.3, 0.9):
                check(logits, [1, bad, 2, 3, 0, 0], [0, 4], [0.0] * 6, [u], probs)


def test_logits_that_are_not_finite():
    inf, nan = math.inf, math.nan
    rows = torch.tensor([[-inf] * 5, [nan] * 5, [0.0, inf, -inf, inf, 1.0], [nan, 1.0, -inf, 2.0, nan],
                         [-inf, -inf, 3.0, -inf, -inf]])
    for dtype in TYPES:
        for u in (0.0, 0.4, 0.6, 0.99):
            for t in (None, [0.7] * 5, [0.0] * 5, [inf] * 5):
                check(rows.to(dtype), [0] * 5, [0, 1, 2, 3, 4, 5], [0.5] * 5, [u] * 5, None,
                      [3.4e38] * 5 if t == [inf] * 5 else t)
                check(rows.to(dtype), [0, 3, 3, 3, 2], [0, 2, 4, 5, 5, 5], [0.5] * 5, [u] * 5, None,
                      [3.4e38] * 5 if t == [inf] * 5 else t)
    assert run(rows[:2], [0, 0], [0, 1, 2], [0.0] * 2, [0.5] * 2) == ([0, 0], [-1, -1])
    assert run(rows[2:3], [0], [0, 1], [0.0], [0.5], temperature=[inf]) == ([0], [3])


def test_draft_probabilities_that_are_not_finite():
    logits, tokens, starts, accept, sample, q = case(torch.float32, 60, [2, 2], True, pad=0)
    for bad in (math.nan, math.inf, -1.0):
        odd = q.copy()
        odd[:, ::3] = bad
        odd[0, tokens[1]] = bad
        check(logits, tokens, starts, accept, sample, odd)


def test_equal_logits_are_taken_from_the_front():
    logits = torch.zeros(3, 10000)
    logits[0, [7, 9000]], logits[1, [4096, 9999]], logits[2, 9999] = 5.0, 5.0, 5.0
    assert run(logits, [0, 7, 4096], [0, 3], [0.99] * 3, [0.9], temperature=[0.0]) == ([2], [9999])
    assert run(logits, [0, 9000, 4096], [0, 3], [0.0] * 3, [0.9], temperature=[0.0]) == ([0], [7])


def test_starts_that_mean_nothing_are_kept_inside():
    """Rows past the logits and starts that fall do no harm."""
    logits = torch.randn(6, 100)
    for starts in ([-5, 3, 900], [4, 2, 6], [100, 200, 300], [6, 6, 6], [0, 2 ** 31 - 1, 3]):
        accepted, following = run(logits, [0] * 6, starts, [0.5] * 6, [0.5] * 2)
        assert all(0 <= n <= 6 for n in accepted) and all(-1 <= v < 100 for v in following)


def test_strided_rows_and_no_rows():
    logits, tokens, starts, accept, sample, q = case(torch.bfloat16, 501, [2, 0, 3], True)
    wide = torch.full((logits.shape[0], 777), math.nan, dtype=torch.bfloat16, device=DEVICE)
    wide[:, 3:504] = logits.to(DEVICE)
    drafts = torch.full((logits.shape[0], 640), math.nan, device=DEVICE)
    drafts[:, 1:502] = torch.from_numpy(q).to(DEVICE)

    def on(x, dtype):
        return torch.as_tensor(np.asarray(x), dtype=dtype).to(DEVICE)
    got = serving.verify_drafts(wide[:, 3:504], on(tokens, torch.int64), on(starts, torch.int32),
                                on(accept, torch.float64), on(sample, torch.float64), draft_probs=drafts[:, 1:502])
    want = definition(logits.double().numpy(), tokens, starts, accept, sample, q, None)
    assert (got[0].tolist(), got[1].tolist()) == tuple(want)
    none = torch.zeros(0, 501)
    assert run(none, [], [0, 0, 0], [], [0.5, 0.5]) == ([0, 0], [-1, -1])
    assert run(none, [], [0], [], []) == ([], [])


def test_answers_are_distributed_as_the_model_s():
    """Over numbers that are even: the pairs (accepted, next token) of one draft
    by a draft model come to p, as the rule promises. 180 * 180 numbers on a
    grid: each token's share is off by at most a grid line per interval of
    each number, 8 * 2 / 180 in all."""
    vocab, n = 8, 180
    rng = np.random.default_rng(3)
    logits = torch.from_numpy(rng.standard_normal((1, vocab)))
    p = chances(logits.numpy()[0], 1.0)
    q = chances(rng.standard_normal(vocab), 1.0).astype(np.float32)
    q64 = q.astype(np.float64)
    share = np.zeros(vocab)
    grid = (np.arange(n) + 0.5) / n
    accept, sample = (x.ravel() for x in np.meshgrid(grid, grid))
    rows = logits.float().repeat(2 * n * n, 1)
    for d in range(vocab):
        tokens = np.tile([0, d], n * n)
        got = run(rows, tokens, 2 * np.arange(n * n + 1), np.repeat(accept, 2), sample, np.tile(q, (2 * n * n, 1)))
        accepted, following = np.array(got[0]), np.array(got[1])
        first = np.where(accepted == 1, d, following)
        share += q64[d] / q64.sum() * np.bincount(first, minlength=vocab) / (n * n)
    assert np.abs(share - p).max() <= 16 / n


def test_captured_and_replayed():
    """A graph of the call follows its inputs, with eager work between."""
    logits, tokens, starts, accept, sample, q = case(torch.float32, 5000, [3, 0, 2], True)

    def on(x, dtype):
        return torch.as_tensor(np.asarray(x), dtype=dtype).to(DEVICE)
    state = [logits.to(DEVICE), on(tokens, torch.int64), on(starts, torch.int32), on(accept, torch.float64),
             on(sample, torch.float64)]
    drafts = torch.from_numpy(q).to(DEVICE)
    serving.verify_drafts(*state, draft_probs=drafts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serving.verify_drafts(*state, draft_probs=drafts)
    for seed in range(4):
        other = case(torch.float32, 5000, [3, 0, 2] if seed % 2 else [1, 2, 2], True, seed=seed + 9)
        for t, x in zip(state + [drafts], (other[0], *(torch.as_tensor(np.asarray(v)) for v in other[1:5]),
                                           torch.from_numpy(other[5]))):
            t.copy_(x[:t.shape[0]].to(DEVICE))
        graph.replay()
        torch.cuda.synchronize()
        want = definition(other[0].double().numpy(), *other[1:5], other[5], None)
        assert (out[0].tolist(), out[1].tolist()) == tuple(want)
        eager = serving.verify_drafts(*state, draft_probs=drafts)
        assert torch.equal(eager[0], out[0]) and torch.equal(eager[1], out[1])


def test_a_side_stream():
    logits, tokens, starts, accept, sample, q = case(torch.float16, 3000, [3, 1], True)
    state = [logits.to(DEVICE)] + [torch.as_tensor(np.asarray(x), dtype=dtype).to(DEVICE) for x, dtype in
                                   ((tokens, torch.int64), (starts, torch.int32), (accept, torch.float64),
                                    (sample, torch.float64))]
    drafts, side = torch.from_numpy(q).to(DEVICE), torch.cuda.Stream()
    want = serving.verify_drafts(*state, draft_probs=drafts)
    side.wait_stream(torch.cuda.current_stream())
    got = serving.verify_drafts(*state, draft_probs=drafts, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("change, message", [
    (dict(logits=torch.zeros(4, 10)), "logits"),
    (dict(tokens="short"), "tokens"), (dict(accept="float"), "accept"), (dict(sample="short"), "sample"),
    (dict(starts="long"), "starts"), (dict(draft_probs="half"), "draft_probs"), (dict(temperature="short"), "temperature")])
def test_refusals_that_need_the_device(change, message):
    f64 = torch.float64
    state = dict(logits=torch.zeros(4, 10, device=DEVICE), tokens=torch.zeros(4, dtype=torch.int64, device=DEVICE),
                 starts=torch.tensor([0, 2, 4], dtype=torch.int32, device=DEVICE),
                 accept=torch.zeros(4, dtype=f64, device=DEVICE), sample=torch.zeros(2, dtype=f64, device=DEVICE),
                 draft_probs=torch.zeros(4, 10, device=DEVICE), temperature=torch.ones(2, device=DEVICE))
    for name, how in change.items():
        t = state[name]
        state[name] = how if torch.is_tensor(how) else \
            {"short": t[:-1], "float": t.float(), "long": t.long(), "half": t.half()}[how]
    with pytest.raises(ValueError, match=message):
        serving.verify_drafts(**state)
