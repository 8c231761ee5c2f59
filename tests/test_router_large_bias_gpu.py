"""Balance biases at the end of fp32's range, as programs use them to force or to ban experts: the sum of a group's two best
is a number in 64 bits, and the choice goes by it."""
import math

import pytest
import torch

from .test_router_gpu import check

pytestmark = pytest.mark.gpu
LAST = torch.finfo(torch.float32).max


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("experts", [32, 36])
def test_banned_experts(native_lib, score, experts):
    """A group whose experts are all banned comes before one whose experts are all masked."""
    x = torch.randn(50, experts, device="cuda")
    size = experts // 4
    bias = torch.full((experts,), -LAST, device="cuda")
    x[:, :size] = -math.inf
    bias[2 * size + 3] = 0.0
    chosen, _ = check(x, size + 2, score=score, bias=bias, groups=4, topk_groups=2)
    assert (chosen[:, 0] == 2 * size + 3).all() and (chosen >= size).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_forced_experts(native_lib, score):
    x = torch.randn(50, 64, device="cuda")
    bias = torch.zeros(64, device="cuda")
    bias[[1, 2]] = 0.6 * LAST
    bias[[41, 42]] = LAST
    chosen, _ = check(x, 3, score=score, bias=bias, groups=8, topk_groups=1)
    assert (chosen[:, :2] // 8 == 5).all()
    check(x, 6, score=score, bias=bias, groups=8, topk_groups=3)
    check(x, 6, score=score, bias=bias, groups=8, topk_groups=3, group_score="max")
