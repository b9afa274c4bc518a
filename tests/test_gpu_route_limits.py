"""route_experts where scores or biases are NaN or infinite: NaN is behind every
other expert, whatever the scoring and the bias."""
import math

import pytest
import torch

from neuralzip_amd.gpu import serving

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
INF, NAN = math.inf, math.nan


def route(scores, bias=None, **more):
    """All experts in order, and their weights, of one token with these scores."""
    weight = torch.zeros(len(scores), 8, device=DEVICE)
    weight[:, 0] = torch.tensor(scores)
    x = torch.zeros(1, 8, device=DEVICE)
    x[0, 0] = 1.0
    bias = None if bias is None else torch.tensor(bias, device=DEVICE)
    ids, weights = serving.route_experts(x, weight, min(len(scores), 32), bias=bias, **more)
    return ids[0].tolist(), weights[0].tolist()


def definition(scores, bias, scoring):
    rank = [s if scoring == "softmax" else (NAN if math.isnan(s) else 1 / (1 + math.exp(-s)) if s > -700 else 0.0) for s in scores]
    rank = [r + b for r, b in zip(rank, bias or [0.0] * len(rank))]
    return sorted(range(len(rank)), key=lambda e: (math.isnan(rank[e]), 0.0 if math.isnan(rank[e]) else -rank[e], e))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scores, bias", [
    ([0.5, NAN, -2.0, -INF, 1.0], None), ([0.5, NAN, -2.0, -INF, 1.0], [0.0, 9.0, 0.0, 0.0, 0.0]),
    ([NAN, -INF, NAN, -INF, -INF], None), ([NAN, -INF, NAN, -INF, -1.0], [5.0, 0.0, INF, 0.0, 0.0]),
    ([0.5, 1.0, 2.0, 3.0], [NAN, 0.0, -INF, 0.0]), ([0.0, NAN, -1000.0, -800.0], None), ([NAN, NAN, NAN], [1.0, 2.0, 3.0]),
    ([INF, 1.0, NAN, -INF], [-1.0, 0.5, 0.0, 0.0]), ([NAN] + [-INF] * 30, None)])
def test_nan_is_behind_every_expert(scores, bias, scoring):
    for normalize in (False, True):
        ids, weights = route(scores, bias, scoring=scoring, normalize=normalize)
        assert ids == definition(scores, bias, scoring)
        live = [s for s in scores if not math.isnan(s) and s > -INF]
        if live:
            assert all(w == 0.0 for e, w in zip(ids, weights) if math.isnan(scores[e]))
            assert all(math.isfinite(w) for w in weights)


def test_nan_among_many_experts():
    """More experts than are chosen, several threads an expert and one."""
    for experts in (40, 100, 600, 1024):
        scores = [NAN if e % 3 == 0 else ((e * 7) % 11) / 8 - 0.5 for e in range(experts)]
        want = definition(scores, None, "softmax")[:32]
        assert route(scores)[0] == want
        bias = [100.0 if e % 3 == 0 else 0.0 for e in range(experts)]
        assert route(scores, bias, scoring="sigmoid")[0] == definition(scores, bias, "sigmoid")[:32]
