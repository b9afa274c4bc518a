"""verify_drafts where weights are at the ends of 64 bits, against the
definition in 64 bits: logits next to one another at low temperatures, logits
as far apart as 32 bits allow at high ones. Results are whole numbers and have
to be equal."""
import itertools
import math

import numpy as np
import pytest
import torch

from test_gpu_verify import chances, check, run

pytestmark = pytest.mark.gpu

MOST = float(np.finfo(np.float32).max)
# Some whose neighbour below is half of 2^-23 of them away, some of which it is
# nearly all; negative ones, a subnormal one and those at both ends.
TOPS = [16.0, 12.0, 1.75, 1.0, 100.0, 30.0, 1e6, 1.5e10, 3e38, -16.0, -12.0, -1e6, 1e-40, 2.0 ** -126, 0.0, MOST]
TEMPERATURES = [1e-6, 1e-7, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20, 1e-38, 1e-45, 1.0]


def below(top, steps):
    x = np.float32(top)
    for _ in range(steps):
        x = np.nextafter(x, np.float32(-np.inf))
    return float(x)


@pytest.mark.parametrize("top", TOPS)
@pytest.mark.parametrize("place", [3, 5000])
def test_logits_next_to_the_largest(top, place):
    """The runner-up one and two steps below, in the largest one's chunk and in
    another: as a row of its own, and behind a draft of the largest, which is
    accepted by its number or refused by it."""
    for steps, t in itertools.product((1, 2), TEMPERATURES):
        row = torch.full((3, 5003), -math.inf)
        row[:, 1], row[:, place], row[:, 2] = top, below(top, steps), below(top, 3 * steps)
        for u in (0.0, 0.4, 0.6, 0.99):
            check(row[:1], [0], [0, 1], [0.0], [u], temperature=[t])
            for draft, accept in ((1, 0.4), (1, 1.0), (place, 0.0), (place, 0.9)):
                check(row, [0, draft, 1], [0, 3], [accept, 0.3, 0.0], [u], temperature=[t])
                q = np.zeros((3, 5003), dtype=np.float32)
                q[:, 1], q[:, place] = 0.5, 0.25
                check(row, [0, draft, 1], [0, 3], [accept, 0.3, 0.0], [u], q, [t])


def test_the_last_weights_that_64_bits_hold():
    """Behind the refusal of the largest logit (by a number that is not below
    1) its runner-up is picked as long as it has a weight."""
    row = torch.zeros(2, 5000)
    for place, gap in itertools.product((7, 4999), (700.0, 744.0, 745.0, 745.5, 746.0, 2000.0, 1e30)):
        row[:], row[:, 1], row[:, place] = -math.inf, 0.0, -gap
        assert run(row, [0, 1], [0, 2], [1.0, 0.0], [0.5]) == ([0], [place if gap < 745.2 else 1])


@pytest.mark.parametrize("t", [1e38, 3e38, 3.4e38, MOST])
def test_logits_far_apart_at_high_temperatures(t):
    rng = np.random.default_rng(1)
    row = torch.from_numpy(rng.uniform(-3.4e38, 3.4e38, (4, 300)).astype(np.float32))
    row[:, 7], row[:, 9], row[:, 11] = MOST, -MOST, -math.inf
    for u in rng.random(20):
        check(row, [0, 9, 9, 5], [0, 2, 4], [0.001, 0.0, 0.9, 0.5], [u, 1 - u], temperature=[t, t])
    two = torch.tensor([[3e38, -3e38]])
    share = 1 / (1 + math.exp(-6e38 / float(np.float32(t))))
    for u in (share - 1e-5, share + 1e-5):
        assert run(two, [0], [0, 1], [0.0], [u], temperature=[t]) == ([0], [int(u > share)])


def test_an_infinite_temperature():
    """Every finite logit is as likely as any other."""
    row = torch.tensor([[3e38, -3e38, -math.inf, 0.0, math.nan, 1.0]])
    for i, token in enumerate((0, 1, 3, 5)):
        assert run(row, [0], [0, 1], [0.0], [i / 4 + 0.01], temperature=[math.inf]) == ([0], [token])


def test_the_first_of_the_largest_wherever_it_lies():
    """Without a temperature, in every thread of a chunk, alone and with equals
    behind it in its own wavefront, the next ones and the next chunk."""
    for behind in (None, 1, 700, 3000, 4096):
        row = torch.zeros(513, 9000)
        places = [8 * i + i % 8 for i in range(513)]
        for i, place in enumerate(places):
            row[i, place] = 2.0
            if behind is not None:
                row[i, place + behind] = 2.0
        got = run(row, [0] * 513, list(range(514)), [0.0] * 513, [0.9] * 513, temperature=[0.0] * 513)
        assert got == ([0] * 513, places)


def test_tokens_in_every_chunk():
    """Equal weights: the token is the number's place, in each of a row's chunks,
    whose sums of those before another thread hands on."""
    vocab, step = 1 << 16, 1021
    tokens = list(range(0, vocab, step))
    n = len(tokens)
    row = torch.zeros(n, vocab, dtype=torch.bfloat16)
    got = run(row, [0] * n, list(range(n + 1)), [0.0] * n, [t / vocab for t in tokens])
    assert got == ([0] * n, tokens)


def answer_shares(p, q, rest_of):
    """How often each token is a request's first one, over a draft drawn from q
    that is kept with probability min(1, p / q), or replaced by a token with
    weights rest_of(draft) otherwise."""
    share = np.zeros(len(p))
    for d in range(len(p)):
        kept = min(1.0, p[d] / q[d])
        rest = rest_of(d)
        share[d] += q[d] * kept
        share += q[d] * (1.0 - kept) * rest / rest.sum()
    return share


def test_first_tokens_are_distributed_as_the_model_s():
    """The draft is accepted below p / q and not above it, which gives its share
    exactly; the token after a refusal is counted over n even numbers, each
    token's share off by less than a number's, 1 / n. Rules that pick that token
    from p, or from p without the draft, are far outside that bound."""
    vocab, n = 8, 2000
    rng = np.random.default_rng(3)
    logits = torch.from_numpy(rng.standard_normal((1, vocab))).float()
    p, q32 = chances(logits.double().numpy()[0], 1.0), chances(rng.standard_normal(vocab), 1.0).astype(np.float32)
    q = q32.astype(np.float64)       # (its sum is 1 to within vocab * 2^-25)
    bound = 1.0 / n + vocab * 2.0 ** -24
    outside = np.eye(vocab)
    for wrong in (lambda d: p, lambda d: p * (1.0 - outside[d])):
        assert np.abs(answer_shares(p, q, wrong) - p).max() > 20 * bound
    assert np.abs(answer_shares(p, q, lambda d: np.maximum(p - q, 0.0)) - p).max() < bound / 10
    sample = (np.arange(n) + 0.5) / n
    counts = {}
    for d in range(vocab):
        def at(accept, samples):
            rows = 2 * len(samples)
            return run(logits.repeat(rows, 1), [0, d] * len(samples), list(range(0, rows + 1, 2)), [accept, 0.0] * len(samples),
                       samples, np.tile(q32, (rows, 1)))
        limit = p[d] / q[d]
        assert at(min(limit, 1.0) * (1 - 1e-12), [0.5])[0] == [1]
        counts[d] = np.zeros(vocab)
        if limit < 1.0:
            accepted, following = at(limit * (1 + 1e-12), sample)
            assert accepted == [0] * n
            counts[d] = np.bincount(following, minlength=vocab).astype(np.float64)
    assert any(c.sum() for c in counts.values())
    share = answer_shares(p, q, lambda d: counts[d] if counts[d].sum() else np.ones(vocab))
    assert np.abs(share - p).max() <= bound
