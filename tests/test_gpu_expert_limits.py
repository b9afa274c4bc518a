"""expert_mlp where weights or activations are infinite: the results are the
formula's, infinite or NaN as in exact arithmetic with infinities."""
import math

import pytest
import torch

from neuralzip_amd.gpu import serving

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def layer(dtype, x, gate, up, down, inter=40, hidden=72):
    """One token of one expert whose inner element i is act(gate[i] x) * (up[i]
    x), from the token's first element alone. `down` maps places of the output
    to {inner element: weight}; all others are 0."""
    t = torch.zeros(1, hidden, dtype=dtype, device=DEVICE)
    t[0, 0] = x
    gate_up, weights = torch.zeros(1, 2 * inter, hidden), torch.zeros(1, hidden, inter)
    for i, value in gate.items():
        gate_up[0, i, 0] = value
    for i, value in up.items():
        gate_up[0, inter + i, 0] = value
    for place, row in down.items():
        for i, value in row.items():
            weights[0, place, i] = value
    one = torch.ones(1, 1, device=DEVICE)
    ids = torch.zeros(1, 1, dtype=torch.int32, device=DEVICE)
    return serving.expert_mlp(t, ids, one, gate_up.to(DEVICE, dtype), weights.to(DEVICE, dtype))[0].tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("value", [40.0, 40.25, 1.0 / 3])
def test_infinite_weights(dtype, sign, value):
    """Of activations that 16 bits hold exactly, and of ones that they do not:
    40 * value, as silu(40) is 40 in 32 bits."""
    inner = (0, 7, 39)
    out = layer(dtype, 1.0, {i: 40.0 for i in inner}, {i: sign * value for i in inner},
                {0: {0: math.inf}, 1: {7: -math.inf}, 2: {39: math.inf, 0: 1.0}, 71: {0: math.inf, 7: -math.inf},
                 5: {3: math.inf}, 6: {0: 1.0}})
    assert out[:3] == [sign * math.inf, -sign * math.inf, sign * math.inf]
    # infinities of both signs, and an infinite weight of an activation of 0
    assert math.isnan(out[71]) and math.isnan(out[5])
    assert math.isfinite(out[6]) and out[10:71] == [0.0] * 61


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_activations(dtype):
    """Where the token's element is infinite, all activations are: their
    products with weights of one sign are too, those with 0 are NaN."""
    inner = {i: 1.0 for i in range(40)}
    out = layer(dtype, math.inf, inner, inner, {0: dict(inner), 1: {i: -0.5 for i in inner},
                                                2: {**inner, 39: math.inf},
                                                3: {**inner, 4: -1.0}})
    assert out[:3] == [math.inf, -math.inf, math.inf]
    assert all(math.isnan(v) for v in out[3:])


def test_an_infinite_activation_beside_finite_ones():
    """fp16 activations are scaled by the largest of them; an infinite one must
    not make others, finite but past fp16's range, infinite."""
    t = torch.zeros(1, 8, dtype=torch.float16, device=DEVICE)
    t[0, 0] = 60000.0
    gate_up, down = torch.zeros(1, 16, 8), torch.zeros(1, 8, 8)
    gate_up[0, 0, 0] = gate_up[0, 8, 0] = math.inf      # infinite
    gate_up[0, 1, 0] = gate_up[0, 9, 0] = 60000.0       # 1.3e19
    down[0, :, 0], down[0, 0, 1], down[0, 1, 1] = 1.0, -1.0, 1.0
    ids, one = torch.zeros(1, 1, dtype=torch.int32, device=DEVICE), torch.ones(1, 1, device=DEVICE)
    out = serving.expert_mlp(t, ids, one, gate_up.half().to(DEVICE), down.half().to(DEVICE))[0]
    assert out.tolist() == [math.inf] * 8
