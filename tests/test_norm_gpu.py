"""RMS norm, both directions, against the formula in 64 bits. Half a bf16 step is 2^-8 of the value; a sum of n fp32
terms is off by at most (n + 2) * 2^-24 of the sum of their magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H, F = 2.0 ** -8, 2.0 ** -24
SIZES = [(1, 1), (1, 8), (3, 7), (1, 2048), (130, 128), (5, 1001), (7, 4096), (300, 384), (2, 5121), (3, 8192), (2, 16384), (2, 20008), (1000, 64), (129, 520)]


def make(rows, width, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda")
    b = torch.bfloat16
    return draw(rows, width).to(b), (3 * draw(rows, width)).to(b), (1 + 0.1 * draw(width)).to(b), draw(rows, width).to(b)


def formula(h, w, eps):
    h = h.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    return rstd, h * rstd[:, None] * w.double()


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_forward(native_lib, rows, width, with_residual):
    from pipelink_b200 import mok, norm
    x, r, w, _ = make(rows, width, seed=rows + width)
    h = (x.float() + r.float()).to(torch.bfloat16) if with_residual else x
    rstd, y = formula(h, w, 1e-5)
    n = norm.rmsnorm_fwd(x, w, r if with_residual else None)
    assert torch.equal(n.hidden, h) and n.fp8 is None and n.sc is None
    assert ((n.rstd.double() - rstd).abs() <= (width + 8) * F * rstd).all()
    slack = (width + 16) * F
    assert ((n.y.double() - y).abs() <= (H + slack) * (1 + slack) * y.abs() + 1e-38).all()
    if width % 128 == 0:
        both = norm.rmsnorm_fwd(x, w, r if with_residual else None, out="both")
        only = norm.rmsnorm_fwd(x, w, r if with_residual else None, out="mxfp8")
        padded = torch.zeros(((rows + 127) // 128 * 128, width), dtype=torch.bfloat16, device="cuda")
        padded[:rows] = n.y
        q, sc, _, _ = mok.mxfp8_quantize(padded)
        assert only.y is None and torch.equal(both.y, n.y)
        for got in (both, only):
            assert torch.equal(got.fp8, q) and torch.equal(got.sc, sc) and torch.equal(got.hidden, h) and torch.equal(got.rstd, n.rstd)


@pytest.mark.parametrize("rows,width", SIZES + [(4097, 256), (700, 4096)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_backward(native_lib, rows, width, with_residual):
    from pipelink_b200 import norm
    h, dh, w, dy = make(rows, width, seed=rows * 3 + width)
    rstd, _ = formula(h, w, 1e-5)
    g, n = dy.double() * w.double(), h.double() * rstd[:, None]
    dot, mag = (g * n).mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
    dx = rstd[:, None] * (g - n * dot) + (dh.double() if with_residual else 0)
    got, dw = norm.rmsnorm_bwd(dy, h, rstd.float(), w, dh if with_residual else None)
    terms = rstd[:, None] * (g.abs() + n.abs() * mag * (width + 8)) + (dh.double().abs() if with_residual else 0)
    assert got.dtype == torch.bfloat16 and ((got.double() - dx).abs() <= H * dx.abs() * (1 + H) + 8 * F * terms + 1e-38).all()
    assert dw.dtype == torch.float32
    assert ((dw.double() - (dy.double() * n).sum(0)).abs() <= (rows + 8) * F * (dy.double() * n).abs().sum(0) + 1e-38).all()
    again, dw2 = norm.rmsnorm_bwd(dy, h, rstd.float(), w, dh if with_residual else None)
    assert torch.equal(again, got) and torch.equal(dw, dw2)


def test_gradient_against_differences(native_lib):
    from pipelink_b200 import norm
    h, _, w, dy = make(4, 40, seed=8)
    rstd, _ = formula(h, w, 1e-5)
    dx, dw = norm.rmsnorm_bwd(dy, h, rstd.float(), w)
    u, uw = torch.randn(4, 40, device="cuda", dtype=torch.float64), torch.randn(40, device="cuda", dtype=torch.float64)
    loss = lambda e, ew: (formula(h.double() + e * u, w.double() + ew * uw, 1e-5)[1] * dy.double()).sum()
    want = (loss(1e-5, 0) - loss(-1e-5, 0)) / 2e-5
    assert abs((dx.double() * u).sum() - want) <= H * (dx.double() * u).abs().sum() + 1e-5
    want = (loss(0, 1e-5) - loss(0, -1e-5)) / 2e-5
    assert abs((dw.double() * uw).sum() - want) <= 1e-5 * (1 + (dw.double() * uw).abs().sum())


def test_strides_alignment_broadcast_and_shapes(native_lib):
    from pipelink_b200 import mok, norm
    rows, width = 37, 512
    x, r, w, dy = make(rows, width, seed=4)
    want = norm.rmsnorm_fwd(x, w, r, out="both")
    wide = torch.zeros(rows, 2 * width + 8, dtype=torch.bfloat16, device="cuda")
    for first, spread in ((0, width + 8), (3, width + 5)):       # rows on and off 16-byte boundaries
        wide[:, first:first + width] = x
        wide[:, spread:spread + width] = r
        xs, rs = wide[:, first:first + width], wide[:, spread:spread + width]
        got = norm.rmsnorm_fwd(xs, w, rs, out="both")
        # off 16-byte boundaries other threads hold other columns, so the squares are summed in another order: two fp32
        # sums of `width` positive terms differ by at most 2 (width + 8) 2^-24 of their value, rstd by half of that and
        # its own rounding, and y by as much before both are rounded to bf16, half a step each
        assert torch.equal(got.hidden, want.hidden)
        assert ((got.rstd - want.rstd).abs() <= 2 * (width + 8) * F * want.rstd).all()
        assert ((got.y.double() - want.y.double()).abs() <= 2 * (H + (width + 8) * F) * want.y.double().abs()).all()
        padded = torch.zeros(128, width, dtype=torch.bfloat16, device="cuda")
        padded[:rows] = got.y
        q, sc, _, _ = mok.mxfp8_quantize(padded)
        assert torch.equal(got.fp8, q) and torch.equal(got.sc, sc)
        a, b = norm.rmsnorm_bwd(xs, rs, want.rstd, w, xs), norm.rmsnorm_bwd(x, r, want.rstd, w, x)
        assert torch.allclose(a[1], b[1], rtol=0, atol=float(1e-4 * b[1].abs().max())) and \
            ((a[0].double() - b[0].double()).abs() <= 2 * H * b[0].double().abs() + 1e-6).all()
    # one row for all, columns in front, batch dimensions, an odd weight slice
    row = x[:1].expand(rows, width)
    assert torch.equal(norm.rmsnorm_fwd(row, w).y, norm.rmsnorm_fwd(row.contiguous(), w).y)
    assert torch.equal(norm.rmsnorm_fwd(x.T.contiguous().T, w).y, norm.rmsnorm_fwd(x, w).y)
    assert norm.rmsnorm_fwd(x.view(1, 37, 512), w).y.shape == (1, 37, 512)
    shifted = torch.cat([w[:1], w])[1:]
    assert torch.equal(norm.rmsnorm_fwd(x, shifted).y, norm.rmsnorm_fwd(x, w).y)
    # in place on the residual stream
    stream = r.clone()
    into = norm.Normed(stream, torch.empty(rows, device="cuda"), torch.empty_like(x), None, None)
    norm.rmsnorm_fwd(x, w, stream, into=into)
    assert torch.equal(stream, want.hidden) and torch.equal(into.y, want.y)


def test_reused_outputs(native_lib):
    """`into` of an earlier call: the result names this call's stream."""
    from pipelink_b200 import norm
    x, r, w, _ = make(9, 256, seed=11)
    first = norm.rmsnorm_fwd(x, w)
    n = norm.rmsnorm_fwd(r, w, into=first)
    assert n.hidden is r and n.y is first.y and torch.equal(n.y, norm.rmsnorm_fwd(r, w).y)


def test_extremes(native_lib):
    """Rows of zeros, of the largest and the smallest numbers, and rows that hold infinities or NaN."""
    from pipelink_b200 import norm
    width = 256
    x = torch.zeros(6, width, dtype=torch.bfloat16, device="cuda")
    x[1] = 1e18
    x[2] = 1e-20
    x[3, 5], x[4, 7] = float("inf"), float("nan")
    x[5] = torch.arange(width, device="cuda").bfloat16()
    w = torch.ones(width, dtype=torch.bfloat16, device="cuda")
    n = norm.rmsnorm_fwd(x, w, out="both")
    assert (n.y[0] == 0).all() and (n.fp8[0] == 0).all()
    assert ((n.y[1].double() - 1).abs() <= H).all() and ((n.y[2].double() - 1e-20 / 1e-5 ** 0.5).abs() <= 2 * H * 1e-17).all()
    assert torch.isnan(n.y[3, 5]) and (n.y[3, 6:] == 0).all() and torch.isnan(n.y[4]).all()
    assert torch.isfinite(n.y[5]).all() and (n.fp8[6:] == 0).all()


def test_streams_and_graphs(native_lib):
    from pipelink_b200 import norm
    x, r, w, dy = make(513, 1024, seed=6)
    want = norm.rmsnorm_fwd(x, w, r, out="both")
    want_b = norm.rmsnorm_bwd(dy, want.hidden, want.rstd, w, dy)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            n = norm.rmsnorm_fwd(x, w, r, out="both")
            got.append((n, norm.rmsnorm_bwd(dy, n.hidden, n.rstd, w, dy)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = norm.rmsnorm_fwd(x, w, r, out="both")
        got.append((n, norm.rmsnorm_bwd(dy, n.hidden, n.rstd, w, dy)))
    graph.replay()
    graph.replay()
    for n, b in got:
        assert torch.equal(n.y, want.y) and torch.equal(n.fp8, want.fp8) and torch.equal(n.sc, want.sc)
        assert torch.equal(b[0], want_b[0]) and torch.equal(b[1], want_b[1])


def test_no_rows(native_lib):
    from pipelink_b200 import norm
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    x = torch.empty(0, 128, dtype=torch.bfloat16, device="cuda")
    n = norm.rmsnorm_fwd(x, w, x, out="both")
    assert n.y.shape == (0, 128) and n.fp8.shape == (0, 128)
    dx, dw = norm.rmsnorm_bwd(x, x, n.rstd, w)
    assert dx.shape == (0, 128) and (dw == 0).all()
