"""Routing with a bias on the logits: alone, with groups, and where logit and bias leave f32 when they are added."""
import math

import pytest
import torch

from tests.test_gpu_route_logits import SIGMOID, SOFTMAX, check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("T,E,k", [(1, 8, 8), (1, 256, 8), (40, 64, 6), (70, 512, 32), (600, 384, 8), (33, 129, 3)])
def test_without_groups(gpu_backend, dtype, score, T, E, k):
    bias = logits(1, E, 3)[0]
    check(gpu_backend, logits(T, E, 4, dtype), k, score, logit_bias=bias, norm=bool(T % 2), scale=2.5)
    check(gpu_backend, logits(T, E, 5, dtype), k, score, logit_bias=bias, select_bias=logits(1, E, 6)[0] * 0.1)


@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
def test_closed_by_either(gpu_backend, score):
    z, bias = logits(30, 64, 7), logits(1, 64, 8)[0]
    z[:, ::3], z[4] = -math.inf, -math.inf
    bias[1::3], bias[2] = -math.inf, math.nan
    got = check(gpu_backend, z, 30, score, logit_bias=bias, norm=True)
    assert (got.idx[0] >= 0).sum() == 20 and (got.idx[4] == -1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("G,kept", [(1, 1), (4, 3)])
def test_lowest_and_largest_values(gpu_backend, dtype, score, G, kept):
    """Masks of the lowest finite value in logits and in the bias: their sum is a number, below every other, and closes nothing."""
    low, f32 = torch.finfo(dtype).min, torch.finfo(torch.float32)
    z = logits(8, 16, 9)
    z[0, :], z[1, 3:], z[2, ::2] = low, low, low
    z[3], z[3, 5] = -math.inf, low          # the only open expert
    z[4], z[4, [5, 6]] = -math.inf, low     # two, one of them with a bias
    z[5], z[5, [2, 9]] = -math.inf, -low    # largest and largest
    z[6] = low
    z[6, 1] = -math.inf
    z = z.to(dtype)
    bias = torch.zeros(16, device="cuda")
    bias[[3, 5, 6, 12]], bias[9] = f32.min, f32.max
    for select in (None, torch.linspace(0, 3, 16, device="cuda")):
        got = check(gpu_backend, z, 6, score, logit_bias=bias, select_bias=select, G=G, kept=kept)
        assert got.idx[3, 0] == 5 and set(got.idx[4, :2].tolist()) == {5, 6}
