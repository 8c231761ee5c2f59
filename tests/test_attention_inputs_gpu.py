"""Inputs of attention as programs have them: slices of a fused projection, heads in front of positions, one KV head
broadcast to all, storage off a 16-byte boundary. Every one gives the bits of its dense copy, forward and backward."""
import pytest
import torch

from .test_attention_bwd_gpu import make

pytestmark = pytest.mark.gpu


def bits(ts):
    return [t.contiguous().view(torch.int16) if t.dtype is torch.bfloat16 else t for t in ts]


def both(q, k, v, do, **kw):
    from pipelink_b200 import attention as att
    out, lse = att.attention_fwd(q, k, v, **kw)
    assert out.shape == q.shape
    return bits([out, lse, *att.attention_bwd(do, q, k, v, out, lse, **kw)])


def same(got, want):
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("B,S", [(1, 256), (2, 128), (2, 200)])
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (3, 3)])
def test_strides_and_alignment(native_lib, B, S, Hq, Hkv):
    q, k, v, do = make(B, S, Hq, Hkv, seed=S)
    want = both(q, k, v, do)
    fused = torch.cat([q, k, v], dim=2)
    same(both(fused[:, :, :Hq], fused[:, :, Hq:Hq + Hkv], fused[:, :, Hq + Hkv:], do), want)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    same(both(heads_first(q), heads_first(k), heads_first(v), heads_first(do)), want)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(t.shape).copy_(t)
    same(both(shifted(q), shifted(k), shifted(v), shifted(do)), want)


@pytest.mark.parametrize("S", [128, 150])
def test_broadcast_heads(native_lib, S):
    q, k, v, do = make(2, S, 4, 1, seed=S)
    wide = lambda t: t.expand(-1, -1, 4, -1)
    same(both(q, wide(k), wide(v), do), both(q, wide(k).contiguous(), wide(v).contiguous(), do))
    one = q[:, :, :1].expand(-1, -1, 4, -1)
    same(both(one, k, v, do), both(one.contiguous(), k, v, do))


@pytest.mark.parametrize("window", [256, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5])
def test_windows_that_hide_nothing(native_lib, window):
    """However long: a window that does not fit in 32 bits is not cut down to what is left of it."""
    q, k, v, do = make(1, 256, 2, 1, seed=9)
    same(both(q, k, v, do, window=window), both(q, k, v, do))
