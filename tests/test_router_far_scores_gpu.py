"""Renormalised weights of tokens whose chosen experts all have scores next to nothing: w_i = s_i / sum s is of order 1
however small the scores are, and so is its gradient. The reference works with logarithms of the scores in 64 bits.

Tolerance: a weight is an exponential of an fp32 difference of logits (half a step of |x - max|; of at most 45 against a
softmax's best, and against the best of the chosen where those are farther below) and a sum of topk of them, off by at
most (|x - max| + topk + 16) half steps of fp32 (2^-24), twice that with the quotient; a gradient of k slots adds k
products, and a softmax's other experts see the rounding of the slots' sum, which is 0 by the formula."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F = 2.0 ** -24


def log_scores(x, score):
    x = x.double()
    return torch.nn.functional.logsigmoid(x) if score == "sigmoid" else torch.log_softmax(x, 1)


def weights_of(x, experts, score, scale):
    return scale * torch.softmax(log_scores(x, score).gather(1, experts.long()), 1)


def gradient_of(dw, x, experts, score, scale):
    w = weights_of(x, experts, score, 1.0)
    d = scale * w * (dw.double() - (dw.double() * w).sum(1, keepdim=True))
    if score == "sigmoid":
        d = d * torch.sigmoid(-x.double()).gather(1, experts.long())
    return torch.zeros(x.shape, dtype=torch.float64, device=x.device).scatter_add_(1, experts.long(), d)


def check(x, k, score, scale, **kw):
    from pipelink_b200 import router
    experts, weights = router.route_topk(x, k, score=score, scale=scale, **kw)
    want = weights_of(x, experts, score, scale)
    at = x.double().gather(1, experts.long())
    low = at.amin(1, keepdim=True)
    spread = at.amax(1, keepdim=True) - low
    if score == "softmax":
        spread = torch.maximum(spread, (x.double().amax(1, keepdim=True) - low).clamp_max(45))
    tol = 2 * (spread + k + 16) * F
    assert ((weights.double() - want).abs() <= tol * want).all(), float(((weights.double() - want).abs() / (tol * want)).max())
    dw = torch.randn(x.shape[0], k, device="cuda") * 3
    got = router.route_topk_bwd(dw, x, experts, score=score, scale=scale)
    want = gradient_of(dw, x, experts, score, scale)
    size = scale * dw.double().abs().sum(1, keepdim=True)              # of a slot's gradient before the mean is taken off
    share = torch.zeros_like(want).scatter_(1, experts.long(), weights.double() / scale)
    if score == "softmax":
        share = torch.maximum(share, log_scores(x, score).exp())
    tol = 4 * tol * size * share + 2.0 ** -8 * want.abs() * (x.dtype == torch.bfloat16)
    assert got.dtype == x.dtype and ((got.double() - want).abs() <= tol + 1e-37).all()
    return experts, weights


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("level", [-20.0, -80.0, -87.0, -88.0, -88.5, -100.0, -600.0])
def test_sigmoids_far_below_zero(native_lib, level, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (level + torch.randn(70, 64, generator=g, device="cuda")).to(dtype)
    check(x, 8, "sigmoid", 2.5)
    check(x, 8, "sigmoid", 1.0, groups=8, topk_groups=3)
    check(x, 5, "sigmoid", 100.0, bias=torch.linspace(1, 0, 64, device="cuda"))
    check(x[:, :33], 20, "sigmoid", 1.0)


def test_scores_that_vanish_in_64_bits(native_lib):
    """exp(-700) and less counts as 0, so that a type's lowest number masks an expert as -inf does."""
    from pipelink_b200 import router
    x = -1000 + torch.randn(9, 64, device="cuda")
    experts, weights = router.route_topk(x, 4, score="sigmoid")
    assert (weights == 0).all() and (router.route_topk_bwd(torch.ones_like(weights), x, experts, score="sigmoid") == 0).all()
    x[:, 5] = -90.0
    experts, weights = router.route_topk(x, 4, score="sigmoid")
    assert (experts[:, 0] == 5).all() and (weights[:, 0] == 1).all() and (weights[:, 1:] == 0).all()
    x = torch.full((9, 64), torch.finfo(torch.float32).min, device="cuda")
    x[:, :2] = 0.0
    bias = torch.zeros(64, device="cuda")
    bias[:2] = -2.0
    experts, weights = router.route_topk(x, 4, bias=bias)
    assert (experts >= 2).all() and (weights == 0).all()
    assert (router.route_topk_bwd(torch.ones_like(weights), x, experts) == 0).all()


@pytest.mark.parametrize("gap", [20.0, 90.0, 104.0, 300.0])
def test_a_bias_that_drops_the_best_of_a_softmax(native_lib, gap):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(65, 96, generator=g, device="cuda")
    x[:, :4] += gap
    bias = torch.zeros(96, device="cuda")
    bias[:4] = -3.0
    experts, _ = check(x, 6, "softmax", 1.5, bias=bias)
    assert (experts >= 4).all()
    # by groups: the first group holds the best expert and loses by the sum of its two best
    bias = torch.zeros(96, device="cuda")
    bias[:48] = -4.0
    check(x, 6, "softmax", 1.0, bias=bias, groups=2, topk_groups=1)


def test_masked_repeated_and_foreign_experts_far_below_zero(native_lib):
    from pipelink_b200 import router
    x = torch.full((5, 40), -math.inf, device="cuda")
    x[0, 3], x[1, 3], x[1, 9] = -95.0, -95.0, -96.0
    x[2:] = -93.0
    experts, weights = router.route_topk(x, 2, score="sigmoid")
    assert experts[0, 0] == 3 and weights[0].tolist() == [1.0, 0.0] and experts[1].tolist() == [3, 9]
    assert abs(float(weights[1, 0]) - 1 / (1 + math.exp(-1))) <= 32 * F and weights[2].tolist() == [0.5, 0.5]
    chosen = torch.tensor([[3, 0], [3, 9], [7, 7], [5, 40], [-1, 41]], dtype=torch.int32, device="cuda")
    dw = torch.tensor([[1.0, 2.0], [3.0, -1.0], [1.0, 3.0], [2.0, 5.0], [1.0, 1.0]], device="cuda")
    for score in ("sigmoid", "softmax"):
        got = router.route_topk_bwd(dw, x, chosen, score=score)
        assert torch.isfinite(got).all() and (got[0] == 0).all() and (got[2:].abs() <= 64 * F).all()
    got = router.route_topk_bwd(dw, x, chosen, score="sigmoid")
    w = 1 / (1 + math.exp(-1))
    assert abs(float(got[1, 3]) - 4 * w * (1 - w)) <= 256 * F and abs(float(got[1, 9]) + 4 * w * (1 - w)) <= 256 * F
    # an expert named twice counts twice: slots 7, 7 have half each, and their gradients cancel; NaN spreads as before
    x[2, 20] = math.nan
    assert torch.isnan(router.route_topk_bwd(dw, x, chosen, score="softmax")[2]).all()
    assert torch.isnan(router.route_topk_bwd(dw, x, chosen, score="sigmoid")[2, 20])
