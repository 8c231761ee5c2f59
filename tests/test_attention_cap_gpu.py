"""A soft cap from end to end: attention_fwd's output and log-sum-exp as a user hands them to attention_bwd, with scores
that reach the cap, where a probability depends on the cap's tanh the most."""
import math

import pytest
import torch

from .test_attention_bwd_gpu import A, H, check, reference

pytestmark = pytest.mark.gpu

# batch, sequence, heads, KV heads, window, cap, standard deviation of q and k (of the scores: its square)
CASES = [(1, 300, 4, 2, 0, 30.0, 4.0), (2, 77, 4, 2, 0, 50.0, 4.0), (1, 700, 2, 1, 200, 30.0, 3.0), (1, 515, 6, 2, 70, 4.0, 2.0),
         (2, 256, 4, 2, 0, 15.0, 1.0), (1, 200, 8, 2, 0, 50.0, 7.0)]


def make(B, S, Hq, Hkv, size, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda scale, *shape: (scale * torch.randn(*shape, generator=g, device="cuda")).to(torch.bfloat16)
    return draw(size, B, S, Hq, 128), draw(size, B, S, Hkv, 128), draw(1.0, B, S, Hkv, 128), draw(1.0, B, S, Hq, 128)


@pytest.mark.parametrize("B,S,Hq,Hkv,window,cap,size", CASES)
def test_log_sum_exp_of_capped_scores(native_lib, B, S, Hq, Hkv, window, cap, size):
    """A log-sum-exp is off by at most what the scores are: their fp32 sums, and 2^-16 of the cap by tanh.approx (2^-16.4
    of its value over all of its range as measured on a B200); and by its own logarithm. Query heads that share no KV head
    in pairs run a kernel that adds up P as it is rounded to bf16."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(B, S, Hq, Hkv, size, S)
    _, want, _, _ = reference(q, k, v, do, window, cap)
    _, lse = att.attention_fwd(q, k, v, window=window, softcap=cap)
    rows = lambda t: t.double().abs().transpose(1, 2).repeat_interleave(Hq // t.shape[2], 1)      # [B, Hq, S, 128]
    sums = A / math.sqrt(128) * (rows(q) @ rows(k).transpose(-1, -2)).amax(-1).reshape(B * Hq, S)
    tol = sums + 2.0 ** -16 * cap + 2.0 ** -21 * (want.double().abs() + 4) + (H if (Hq // Hkv) % 2 else 0.0)
    assert ((lse.double() - want.double()).abs() <= tol).all(), float(((lse.double() - want.double()).abs() / tol).max())


@pytest.mark.parametrize("B,S,Hq,Hkv,window,cap,size", CASES)
def test_forward_and_backward_together(native_lib, B, S, Hq, Hkv, window, cap, size):
    from pipelink_b200 import attention as att
    q, k, v, do = make(B, S, Hq, Hkv, size, S)
    _, _, grads, tol = reference(q, k, v, do, window, cap)
    out, lse = att.attention_fwd(q, k, v, window=window, softcap=cap)
    # the forward pass rounds P, O and its log-sum-exp as the backward pass does
    check(att.attention_bwd(do, q, k, v, out, lse, window=window, softcap=cap), grads, {n: 3 * t for n, t in tol.items()})
