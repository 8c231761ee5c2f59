"""Routing against its definition in 64 bits: the choice has to be equal, weights and gradients to fp32 arithmetic.

Tolerance: a score is exp of an fp32 difference and a sum over the experts, off by at most (|x - max| + experts + 16)
half steps of fp32 (2^-24), relative; renormalised weights and gradients add as many again."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F = 2.0 ** -24


def scores(x, score):
    x = x.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isneginf(top), 0.0, top))
    total = e.sum(1, keepdim=True)
    return torch.where(total == 0, 0.0, e / total)


def reference(x, k, score="softmax", bias=None, groups=1, topk_groups=1, group_score="top2", renormalize=True, scale=1.0):
    """Python lists over the experts of each token, compared as fp64 numbers."""
    s = scores(x, score).cpu()
    xs = x.double().cpu()
    c = s + (bias.double().cpu() if bias is not None else 0)
    if bias is None and groups == 1:
        c = xs.clone()                                     # the scores' order is the logits'
    c[torch.isneginf(xs)] = -math.inf
    out = []
    size = x.shape[1] // groups
    for row in c.tolist():
        row = [(-math.inf, -1) if v != v else (v, 0) for v in row]          # NaN below every number
        allowed = range(len(row))
        if groups > 1 and topk_groups < groups:
            def value(g):
                best = sorted((v for v, _ in row[g * size:(g + 1) * size]), reverse=True)[: 2 if group_score == "top2" else 1]
                return best[0] + (best[1] if len(best) > 1 and best[1] > -math.inf else 0.0)
            kept = sorted(range(groups), key=lambda g: (-value(g), g))[:topk_groups]
            allowed = [e for g in kept for e in range(g * size, (g + 1) * size)]
        out.append(sorted(allowed, key=lambda e: (-row[e][0], -row[e][1], e))[:k])
    experts = torch.tensor(out, dtype=torch.int64).reshape(len(out), k).to(x.device)
    w = s.to(x.device).gather(1, experts)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return experts, scale * w


def spread(x):
    """|x - max| over the unmasked experts, the largest of a row."""
    x = x.double()
    low = torch.where(torch.isneginf(x), math.inf, x).amin(1)
    return torch.nan_to_num(x.amax(1) - low, nan=0.0, posinf=0.0, neginf=0.0).clamp_min(0)


def check(x, k, **kw):
    from pipelink_b200 import router
    experts, weights = router.route_topk(x, k, **kw)
    want_e, want_w = reference(x, k, **kw)
    assert experts.dtype == torch.int32 and weights.dtype == torch.float32
    assert torch.equal(experts.long(), want_e), (experts.long() != want_e).nonzero()[:4]
    tol = 2 * (spread(x)[:, None] + x.shape[1] + 16) * F * want_w.abs() + 1e-37
    assert ((weights.double() - want_w).abs() <= tol).all(), float(((weights.double() - want_w).abs() / tol).max())
    return experts, weights


CASES = [
    (1, 1, 1, {}), (1, 64, 8, {}), (5, 8, 8, {}), (33, 60, 4, dict(score="sigmoid")), (300, 64, 6, dict(renormalize=False)),
    (257, 33, 5, dict(bias=True)), (100, 160, 6, dict(score="softmax", groups=8, topk_groups=3, group_score="max", renormalize=False, scale=16.0)),
    (513, 256, 8, dict(score="sigmoid", bias=True, groups=8, topk_groups=4, scale=2.5)), (65, 384, 32, dict(score="sigmoid", bias=True)),
    (40, 512, 10, dict(groups=32, topk_groups=1)), (64, 16, 3, dict(score="sigmoid", groups=16, topk_groups=5)),
    (20, 1024, 16, dict(bias=True, groups=4, topk_groups=4)), (31, 96, 7, dict(groups=3, topk_groups=2, bias=True)),
]


@pytest.mark.parametrize("tokens,experts,k,kw", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_choice_and_weights(native_lib, tokens, experts, k, kw, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens + experts)
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = 0.1 * torch.randn(experts, generator=g, device="cuda")
    check(torch.randn(tokens, experts, generator=g, device="cuda").to(dtype), k, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(bias=True), dict(score="sigmoid", bias=True, groups=8, topk_groups=3),
                                dict(groups=8, topk_groups=3, group_score="max"), dict(score="sigmoid", groups=4, topk_groups=2)])
def test_masked_experts_and_empty_rows(native_lib, kw):
    g = torch.Generator(device="cuda").manual_seed(1)
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = 0.3 * torch.randn(64, generator=g, device="cuda")
    x = torch.randn(200, 64, generator=g, device="cuda")
    x[torch.rand(200, 64, generator=g, device="cuda") < torch.rand(200, 1, generator=g, device="cuda")] = -math.inf
    x[7] = -math.inf
    x[8, 1:] = -math.inf
    x[9] = torch.finfo(torch.float32).min          # the type's lowest number is a number
    x[10, :40] = torch.finfo(torch.float32).min
    experts, weights = check(x, 6, **kw)
    assert (weights[7] == 0).all() and torch.isfinite(weights).all()


def test_nan_and_infinity(native_lib):
    """NaN ranks last, the named experts stay valid and distinct, and only the rows that hold one are touched."""
    from pipelink_b200 import router
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(6, 32, generator=g, device="cuda")
    clean = [t.clone() for t in router.route_topk(x, 4, score="sigmoid")]
    x[1, 3], x[2, 5], x[3] = float("nan"), float("inf"), float("nan")
    experts, weights = router.route_topk(x, 4, score="sigmoid")
    for row in (0, 4, 5):
        assert torch.equal(experts[row], clean[0][row]) and torch.equal(weights[row], clean[1][row])
    assert 3 not in experts[1].tolist() and torch.isfinite(weights[1]).all()
    assert experts[2, 0] == 5 and torch.isnan(weights[3]).all()
    for score in ("sigmoid", "softmax"):
        for kw in (dict(), dict(groups=4, topk_groups=2), dict(bias=torch.zeros(32, device="cuda"))):
            experts, weights = router.route_topk(x, 4, score=score, **kw)
            assert all(len(set(r)) == 4 and 0 <= min(r) and max(r) < 32 for r in experts.tolist())
            if score == "softmax":
                assert torch.isnan(weights[1:4]).all() and torch.isfinite(weights[4:]).all()


@pytest.mark.parametrize("kw", [dict(score="sigmoid"), dict(score="softmax"), dict(score="sigmoid", groups=8, topk_groups=4)])
def test_scores_closer_than_fp32(native_lib, kw):
    """Tens of thousands of tokens, some of whose scores with the bias differ by less than an fp32 step, and a
    construction where all do: a choice in fp32 would differ."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(20000, 64, generator=g, device="cuda")
    check(x, 8, bias=0.1 * torch.randn(64, generator=g, device="cuda"), **kw)
    # bias = what the first row's scores lack to 1, rounded to fp32: every choice value is 1 give or take 2^-25
    x = torch.randn(1, 64, generator=g, device="cuda")
    bias = (1 - scores(x, kw["score"])).float()[0]
    check(x.expand(70, 64), 8, bias=bias, **kw)


def test_ties_go_to_the_lowest_index(native_lib):
    x = torch.zeros(3, 96, device="cuda")
    x[1, ::2] = 1.0
    x[2, 50:] = -0.0
    for kw in (dict(), dict(score="sigmoid", bias=torch.zeros(96, device="cuda")), dict(groups=6, topk_groups=2)):
        experts, _ = check(x, 5, **kw)
        assert experts[0].tolist() == [0, 1, 2, 3, 4]
    coarse = torch.randn(500, 64, device="cuda").mul(4).round().div(4)
    check(coarse, 8)
    check(coarse, 8, score="sigmoid", bias=torch.zeros(64, device="cuda"), groups=8, topk_groups=3)
    check(coarse.bfloat16(), 8, bias=torch.full((64,), 0.25, device="cuda"))


def jacobian_reference(dw, x, experts, score, renormalize, scale):
    s = scores(x, score).requires_grad_(False)
    xd = x.double().clone().requires_grad_(True)
    s = torch.sigmoid(xd) if score == "sigmoid" else torch.softmax(xd, 1)
    w = s.gather(1, experts.long())
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    (scale * w * dw.double()).sum().backward()
    return xd.grad


@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 64, 8), (33, 60, 4), (300, 256, 8), (10, 1000, 32), (70, 512, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient(native_lib, tokens, experts, k, score, renormalize):
    from pipelink_b200 import router
    g = torch.Generator(device="cuda").manual_seed(experts)
    x = torch.randn(tokens, experts, generator=g, device="cuda")
    dw = torch.randn(tokens, k, generator=g, device="cuda")
    chosen, _ = router.route_topk(x, k, score=score)
    for dtype in (torch.float32, torch.bfloat16):
        xs = x.to(dtype)
        got = router.route_topk_bwd(dw, xs, chosen, score=score, renormalize=renormalize, scale=2.5)
        want = jacobian_reference(dw, xs, chosen, score, renormalize, 2.5)
        s = scores(xs, score)
        total = s.gather(1, chosen.long()).sum(1, keepdim=True) if renormalize else 1.0
        size = 2.5 * dw.double().abs().sum(1, keepdim=True) * 2 / total      # of dS, before cancellation
        tol = 4 * (experts + 32) * F * s * size * 2 + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0) + 1e-37
        assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())


def test_gradient_of_saturated_sigmoids(native_lib):
    """Far from 0 the slope s (1 - s) is small but as exact as anywhere: expf is off by two steps, the rest by one each."""
    from pipelink_b200 import router
    x = torch.linspace(-40, 40, 32, device="cuda")[None].contiguous()
    chosen = torch.arange(32, dtype=torch.int32, device="cuda")[None]
    dw = 1 + torch.rand(1, 32, device="cuda")
    got = router.route_topk_bwd(dw, x, chosen, score="sigmoid", renormalize=False)
    want = dw.double() * torch.sigmoid(x.double()) * torch.sigmoid(-x.double())
    assert ((got.double() - want).abs() <= 16 * F * want).all()


def test_gradient_of_masked_repeated_and_foreign_experts(native_lib):
    from pipelink_b200 import router
    x = torch.randn(4, 40, device="cuda")
    x[0] = -math.inf
    x[1, 2:] = -math.inf
    chosen = torch.tensor([[0, 1], [1, 0], [7, 7], [5, 39]], dtype=torch.int32, device="cuda")
    dw = torch.randn(4, 2, device="cuda")
    got = router.route_topk_bwd(dw, x, chosen)
    assert (got[0] == 0).all() and (got[1, 2:] == 0).all() and torch.isfinite(got).all()
    want = jacobian_reference(dw[1:], x[1:], chosen[1:], "softmax", True, 1.0)
    assert (got[1:].double() - want).abs().max() <= 1e-5
    plain = router.route_topk_bwd(dw, x, chosen, renormalize=False)
    want = jacobian_reference(dw[1:], x[1:], chosen[1:], "softmax", False, 1.0)
    assert (plain[1:].double() - want).abs().max() <= 1e-5
    foreign = chosen.clone()
    foreign[3, 1] = 40
    foreign[2, 0] = -1
    alone = router.route_topk_bwd(dw, x, foreign, score="sigmoid", renormalize=False)
    assert (alone[3].nonzero().flatten().tolist() == [5]) and alone[2].nonzero().flatten().tolist() == [7]


def test_strides_streams_and_graphs(native_lib):
    from pipelink_b200 import router
    wide = torch.randn(1111, 100, device="cuda")
    x = wide[:, 3:67]
    bias = 0.1 * torch.randn(64, device="cuda")
    kw = dict(score="sigmoid", bias=bias, groups=4, topk_groups=2)
    want = router.route_topk(x.contiguous(), 8, **kw)
    dw = torch.randn(1111, 8, device="cuda")
    want_g = router.route_topk_bwd(dw, x.contiguous(), want[0], score="sigmoid")
    same = lambda r, d: torch.equal(r[0], want[0]) and torch.equal(r[1], want[1]) and torch.equal(d, want_g)
    assert same(router.route_topk(x, 8, **kw), router.route_topk_bwd(dw, x, want[0], score="sigmoid"))
    assert same(router.route_topk(x.T.contiguous().T, 8, **kw), want_g)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            r = router.route_topk(x, 8, **kw)
            got.append((r, router.route_topk_bwd(dw, x, r[0], score="sigmoid")))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = router.route_topk(x, 8, **kw)
        got.append((r, router.route_topk_bwd(dw, x, r[0], score="sigmoid")))
    graph.replay()
    graph.replay()
    assert all(same(*g) for g in got)
    row = x[:1].expand(50, 64)
    assert torch.equal(router.route_topk(row, 8)[0], router.route_topk(row.contiguous(), 8)[0])


def test_no_tokens(native_lib):
    from pipelink_b200 import router
    x = torch.empty(0, 64, device="cuda")
    experts, weights = router.route_topk(x, 8)
    assert experts.shape == (0, 8) and router.route_topk_bwd(weights, x, experts).shape == (0, 64)
