"""Attention's backward pass against the formula in 64 bits.

Tolerance, element by element, from the roundings the kernel makes (half a bf16 step is 2^-8 of the value): the operands
P and dX of the three accumulating products, the saved output inside delta, the stored gradient, and fp32 arithmetic
(a sum of 128 products is off by at most 128 * 2^-24 = 2^-17 of the sum of their magnitudes)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -8       # half a step of bf16, relative
A = 2.0 ** -17      # fp32 sum of 128 products, relative to the sum of magnitudes


def make(B, S, Hq, Hkv, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: (scale * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16)
    return draw(B, S, Hq, 128), draw(B, S, Hkv, 128), draw(B, S, Hkv, 128), draw(B, S, Hq, 128)


def formula(q, k, v, do, window=0, softcap=0.0):
    """One head in 64 bits: out, lse, the gradients and a bound on the kernel's error of each."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    S, scale = q.shape[0], 1 / math.sqrt(128)
    i = torch.arange(S, device=q.device)
    seen = i[:, None] >= i[None, :]
    if window:
        seen &= i[:, None] - i[None, :] < window
    x = q @ k.T * scale
    y = softcap * torch.tanh(x / softcap) if softcap else x
    y = y.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(y, 1)
    p = torch.exp(y - lse[:, None])
    out = p @ v
    dp = do @ v.T
    delta = (do * out).sum(1, keepdim=True)
    slope = (1 - torch.tanh(x / softcap) ** 2) if softcap else torch.ones_like(x)
    ds = p * (dp - delta) * slope
    # exponent: the score's fp32 sum, its scaling, the log-sum-exp in fp32, exp2 and the cap's tanh
    e = A * scale * (q.abs() @ k.abs().T) + 2.0 ** -21 * (1 + x.abs() + lse.abs()[:, None] + softcap)
    d_delta = H * (do * out).abs().sum(1, keepdim=True) + A * (do * out).abs().sum(1, keepdim=True)
    d_ds = p * (e * (dp.abs() + delta.abs()) + A * (do.abs() @ v.abs().T) + d_delta) + H * ds.abs()
    d_ds += p * (dp - delta).abs() * 2.0 ** -19 * (softcap > 0)       # the cap's slope
    d_p = p * (e + H)
    sums = 2.0 ** -24 * (S + 2)                                       # fp32 accumulation over S rows
    grads = dict(dq=scale * ds @ k, dk=scale * ds.T @ q, dv=p.T @ do)
    tol = dict(dq=scale * (d_ds + sums * ds.abs()) @ k.abs(), dk=scale * (d_ds + sums * ds.abs()).T @ q.abs(),
               dv=(d_p + sums * p).T @ do.abs())
    return out, lse, grads, tol


def reference(q, k, v, do, window=0, softcap=0.0):
    B, S, Hq, _ = q.shape
    group = Hq // k.shape[2]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty((B, Hq, S), dtype=torch.float64, device=q.device)
    grads = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in grads.items()}
    for b in range(B):
        for h in range(Hq):
            out[b, :, h], lse[b, h], g, t = formula(q[b, :, h], k[b, :, h // group], v[b, :, h // group], do[b, :, h], window, softcap)
            grads["dq"][b, :, h], tol["dq"][b, :, h] = g["dq"], t["dq"]
            for n in ("dk", "dv"):
                grads[n][b, :, h // group] += g[n]
                tol[n][b, :, h // group] += t[n]
    for n in grads:
        tol[n] = tol[n] + H * (grads[n].abs() + tol[n]) + 1e-30
    return out.to(torch.bfloat16), lse.reshape(B * Hq, S).float(), grads, tol


def check(got, grads, tol):
    for (name, want), have in zip(grads.items(), got):
        assert have.dtype == torch.bfloat16 and have.shape == want.shape and torch.isfinite(have).all()
        over = (have.double() - want).abs() / tol[name]
        assert over.max() <= 1, (name, float(over.max()), [int(i) for i in (over == over.max()).nonzero()[0]])


CASES = [
    (1, 1, 1, 1, 0, 0.0), (3, 2, 2, 1, 0, 0.0), (1, 77, 4, 4, 0, 0.0), (2, 127, 4, 2, 0, 0.0), (1, 128, 2, 1, 0, 0.0),
    (2, 129, 6, 2, 0, 0.0), (1, 513, 8, 1, 0, 0.0), (2, 700, 3, 3, 0, 0.0), (1, 1536, 4, 2, 0, 0.0),
    (2, 129, 2, 2, 1, 0.0), (1, 400, 4, 2, 5, 0.0), (1, 640, 2, 1, 128, 0.0), (1, 641, 2, 1, 129, 0.0), (1, 900, 4, 2, 300, 0.0),
    (1, 300, 2, 1, 300, 0.0), (1, 300, 2, 1, 5000, 0.0),
    (2, 200, 4, 2, 0, 30.0), (1, 515, 2, 1, 70, 4.0),
]


@pytest.mark.parametrize("B,S,Hq,Hkv,window,softcap", CASES)
def test_gradients_against_the_formula(native_lib, B, S, Hq, Hkv, window, softcap):
    from pipelink_b200 import attention as att
    q, k, v, do = make(B, S, Hq, Hkv, seed=S + Hq)
    out, lse, grads, tol = reference(q, k, v, do, window, softcap)
    check(att.attention_bwd(do, q, k, v, out, lse, window=window, softcap=softcap), grads, tol)


@pytest.mark.parametrize("S,window", [(900, 300), (385, 0), (200, 0)])
def test_same_bits_in_every_call(native_lib, S, window):
    """Warps of a tile with and without masked pairs take different times; the gradients do not depend on it. Copies of the
    inputs change the times of the first loads."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(1, S, 4, 2, seed=S)
    out, lse, _, _ = reference(q, k, v, do, window)
    first = att.attention_bwd(do, q, k, v, out, lse, window=window)
    for i in range(600):
        args = [t.clone() for t in (do, q, k, v, out, lse)]
        got = att.attention_bwd(*args, window=window, check=i % 2 == 0)
        assert all(torch.equal(a, b) for a, b in zip(got, first)), i


def test_large_scores(native_lib):
    """Probabilities from 1 down to underflow, and masked scores far above the row's log-sum-exp."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(1, 333, 2, 1, seed=5, scale=4.0)
    out, lse, grads, tol = reference(q, k, v, do)
    check(att.attention_bwd(do, q, k, v, out, lse), grads, tol)


@pytest.mark.parametrize("S,window", [(1, 0), (100, 0), (256, 0), (391, 100)])
def test_forward_and_backward_together(native_lib, S, window):
    """The saved output and log-sum-exp come from the forward pass: its own rounding of P enters delta once more."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(2, S, 4, 2, seed=S)
    _, _, grads, tol = reference(q, k, v, do, window)
    out, lse = att.attention_fwd(q, k, v, window=window)
    assert out.shape == q.shape and lse.shape == (8, S)
    want_out, want_lse, _, _ = reference(q, k, v, do, window)
    assert (out.double() - want_out.double()).abs().max() <= 3 * H * v.abs().max().double()
    assert (lse - want_lse).abs().max() <= 1e-3
    check(att.attention_bwd(do, q, k, v, out, lse, window=window), grads, {n: 3 * t for n, t in tol.items()})


def test_directional_difference(native_lib):
    """<gradient, direction> against central differences of the 64-bit forward pass."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(1, 150, 2, 1, seed=9)
    out, lse, _, tol = reference(q, k, v, do)
    got = att.attention_bwd(do, q, k, v, out, lse)
    for i, name in enumerate(("dq", "dk", "dv")):
        u = torch.randn(got[i].shape, device="cuda", dtype=torch.float64)
        loss = []
        for eps in (1e-4, -1e-4):
            ops = [t.double() for t in (q, k, v)]
            ops[i] = ops[i] + eps * u
            total = 0.0
            for h in range(2):
                x = ops[0][0, :, h] @ ops[1][0, :, 0].T / math.sqrt(128)
                x = x.masked_fill(torch.ones_like(x).triu(1).bool(), -math.inf)
                total = total + (torch.softmax(x, 1) @ ops[2][0, :, 0] * do[0, :, h].double()).sum()
            loss.append(total)
        want = float((loss[0] - loss[1]) / 2e-4)
        # rounding errors of the elements, and the difference's own error (third derivatives, 1e-8 of the scale)
        assert abs(float((got[i].double() * u).sum()) - want) <= float((tol[name] * u.abs()).sum()) + 1e-5 * abs(want) + 1e-3


def test_sequences_do_not_see_each_other(native_lib):
    """A tile that ends past its sequence reads zeros, not the next sequence, whatever that holds."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(2, 200, 4, 2, seed=3)
    out, lse, _, _ = reference(q, k, v, do)
    alone = att.attention_bwd(do[:1], q[:1], k[:1], v[:1], out[:1], lse[:4])
    for t in (q, k, v, do, out):
        t[1] = float("nan")
    lse[4:] = float("nan")
    both = att.attention_bwd(do, q, k, v, out, lse)
    for a, b in zip(alone, both):
        assert torch.equal(a.view(torch.int16), b[:1].view(torch.int16))


def test_same_bits_strides_streams_and_graphs(native_lib):
    from pipelink_b200 import attention as att
    from pipelink_b200.mok import DeviceStatus
    B, S, Hq, Hkv = 2, 333, 4, 2
    q, k, v, do = make(B, S, Hq, Hkv, seed=1)
    out, lse, _, _ = reference(q, k, v, do)
    want = att.attention_bwd(do, q, k, v, out, lse)
    same = lambda got: all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(want, got))
    assert same(att.attention_bwd(do, q, k, v, out, lse))
    # slices of a fused projection, and a buffer that starts off a 16-byte boundary
    fused = torch.cat([q, k, v], dim=2)
    shifted = torch.empty(do.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(do.shape).copy_(do)
    assert same(att.attention_bwd(shifted, fused[:, :, :Hq], fused[:, :, Hq:Hq + Hkv], fused[:, :, Hq + Hkv:], out, lse))
    # heads in front of positions, seen through a transpose
    assert same(att.attention_bwd(do.transpose(1, 2).contiguous().transpose(1, 2), q, k, v, out, lse))
    # two calls in flight on two streams
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got.append(att.attention_bwd(do, q, k, v, out, lse, check=False))
    torch.cuda.synchronize()
    assert same(got[0]) and same(got[1])
    # captured, then replayed on new contents of the same tensors
    status, static = DeviceStatus("cuda"), [t.clone() for t in (do, q, k, v, out, lse)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = att.attention_bwd(*static, check=False, status=status)
    graph.replay()
    assert same(captured)
    static[0].mul_(2)
    graph.replay()
    status.check("replay")
    assert torch.equal(captured[0].view(torch.int16), (want[0] * 2).view(torch.int16))


def test_broadcast_gradient(native_lib):
    """The gradient of a sum: one value broadcast over the output."""
    from pipelink_b200 import attention as att
    q, k, v, _ = make(1, 140, 2, 2, seed=2)
    do = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(q.shape)
    out, lse, grads, tol = reference(q, k, v, do)
    check(att.attention_bwd(do, q, k, v, out, lse), grads, tol)


def test_long_sequence_spot_columns(native_lib):
    """Offsets past 32 bits of bytes and a long accumulation: the batch's last rows against a short problem. With a
    window of 64 the last 256 positions depend on the last 320 alone."""
    from pipelink_b200 import attention as att
    B, S, Hq, Hkv, w = 9, 32768, 64, 8, 64
    q, k, v, do = make(1, S, Hq, Hkv, seed=4)
    tail = S - 384
    out, lse, grads, tol = reference(q[:, tail:, :8], k[:, tail:, :1], v[:, tail:, :1], do[:, tail:, :8], w)
    big = [t.expand(B, -1, -1, -1).contiguous() for t in (q, k, v, do)]
    assert big[0].numel() * 2 > 2 ** 32
    o, l = att.attention_fwd(*big[:3], window=w)
    got = att.attention_bwd(big[3], *big[:3], o, l, window=w)
    for have, name, heads in zip(got, ("dq", "dk", "dv"), (8, 1, 1)):
        over = (have[-1, tail + 128:, :heads].double() - grads[name][0, 128:]).abs() / (3 * tol[name][0, 128:])
        assert over.max() <= 1, (name, float(over.max()))
