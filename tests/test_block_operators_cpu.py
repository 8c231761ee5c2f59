"""Refusals of attention's backward pass, the norm and the router: arguments are checked before anything touches a GPU."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
OK, CAPACITY, ARGUMENT = 0, 2, 3


def bwd(lib, *, batch=1, seq=256, q_heads=4, kv_heads=2, window=0, softcap=0.0, nbytes=None, ptr=4096, last=4096):
    n = lib.plb_attention_bwd_workspace_bytes(batch, seq, q_heads, kv_heads, max(window, 0)) if nbytes is None else nbytes
    return lib.plb_attention_bwd(*[P(ptr)] * 9, P(last), n, batch, seq, q_heads, kv_heads, 1.0, window, softcap, P(ptr), None)


def test_attention_bwd_refusals(native_lib):
    need = native_lib.plb_attention_bwd_workspace_bytes
    assert need(2, 129, 3, 1, 0) >= 2 * 2 * 3 * 256 * 4 and need(1, 8192, 32, 8, 0) >= 2 * 32 * 8192 * 4
    assert need(0, 129, 3, 1, 0) == 0 and need(2, 129, 3, 2, 0) == 0 and need(1, 128, 1, 1, -1) == 0
    for bad in (dict(batch=-1), dict(seq=-1), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=5), dict(window=-1), dict(softcap=-1.0),
                dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=1e-40), dict(ptr=None), dict(ptr=4104), dict(last=None), dict(seq=2 ** 30 + 1), dict(batch=2 ** 23, seq=2 ** 20)):
        assert bwd(native_lib, **bad) in (ARGUMENT, CAPACITY), bad
    assert bwd(native_lib, nbytes=100) == CAPACITY
    assert bwd(native_lib, batch=0) == OK and bwd(native_lib, seq=0) == OK


def norm_fwd(lib, *, ptr=4096, ld=128, res=None, rows=4, width=128, eps=1e-5, hidden=None, rstd=4096, y=4096, fp8=None, sc=None):
    return lib.plb_rmsnorm_fwd(P(ptr), ld, P(res), ld, P(ptr), rows, width, eps, P(hidden), P(rstd), P(y), P(fp8), P(sc), None)


def test_norm_refusals(native_lib):
    for bad in (dict(rows=-1), dict(width=0), dict(eps=-1.0), dict(eps=float("nan")), dict(ld=-1), dict(ptr=None), dict(res=4096),
                dict(hidden=4096), dict(rstd=None), dict(y=None), dict(fp8=4096), dict(sc=4096), dict(fp8=4096, sc=4096, width=96),
                dict(fp8=4097, sc=4096), dict(rows=2 ** 31)):
        assert norm_fwd(native_lib, **bad) == ARGUMENT, bad
    assert norm_fwd(native_lib, rows=0) == OK
    n = native_lib.plb_rmsnorm_bwd_workspace_bytes(300, 256)
    call = lambda ptr=4096, ws=4096, nbytes=n, rows=300, width=256, ld=256: native_lib.plb_rmsnorm_bwd(
        P(ptr), ld, P(ptr), ld, P(ptr), P(ptr), None, 0, rows, width, P(ptr), P(ptr), P(ws), nbytes, None)
    assert call(nbytes=n - 1) == CAPACITY
    for bad in (dict(ptr=None), dict(ws=None), dict(rows=-1), dict(width=0), dict(ld=-1)):
        assert call(**bad) == ARGUMENT, bad


def test_router_refusals(native_lib):
    fwd = lambda ptr=4096, ld=64, tokens=8, experts=64, topk=8, score=0, groups=1, topk_groups=1, scale=1.0: native_lib.plb_route_topk(
        P(ptr), ld, 0, None, tokens, experts, topk, score, groups, topk_groups, 1, 1, scale, P(ptr), P(ptr), None)
    bwd_ = lambda ptr=4096, ld=64, tokens=8, experts=64, topk=8, score=0, scale=1.0: native_lib.plb_route_topk_bwd(
        P(ptr), P(ptr), ld, 0, P(ptr), tokens, experts, topk, score, 1, scale, P(ptr), None)
    both = (dict(ptr=None), dict(ld=-1), dict(tokens=-1), dict(experts=0), dict(experts=1025), dict(topk=0), dict(topk=33),
            dict(experts=4), dict(score=2), dict(scale=float("nan")))
    for bad in both:
        assert fwd(**bad) == ARGUMENT and bwd_(**bad) == ARGUMENT, bad
    for bad in (dict(groups=0), dict(groups=33), dict(groups=7), dict(groups=8, topk_groups=9), dict(groups=8, topk_groups=0),
                dict(groups=16, topk_groups=1)):
        assert fwd(**bad) == ARGUMENT, bad
    assert fwd(tokens=0) == OK and bwd_(tokens=0) == OK


def test_python_refusals(native_lib):
    """CPU tensors, wrong types and shapes are a ValueError, not a launch."""
    from pipelink_b200 import attention, norm, router
    q = torch.zeros(1, 128, 4, 128, dtype=torch.bfloat16)
    k = torch.zeros(1, 128, 2, 128, dtype=torch.bfloat16)
    lse = torch.zeros(4, 128)
    for a in ((q, q, k, k, q, lse), (q[0], q, k, k, q, lse), (q, q[..., :64], k, k, q, lse), (q, q, k[:, :64], k, q, lse),
              (q, q, k, k, q, lse[:2]), (q, q, k, k, q, lse.double()), (q.float(), q, k, k, q, lse), (q, q, k[0], k, q, lse)):
        with pytest.raises(ValueError):
            attention.attention_bwd(*a)
    x, w = torch.zeros(4, 128, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    for call in (lambda: norm.rmsnorm_fwd(x, w), lambda: norm.rmsnorm_fwd(x, w, out="fp8"), lambda: norm.rmsnorm_fwd(x.float(), w),
                 lambda: norm.rmsnorm_bwd(x, x, torch.zeros(4), w), lambda: norm.rmsnorm_fwd(x[0, 0], w)):
        with pytest.raises(ValueError):
            call()
    logits = torch.zeros(4, 64)
    for call in (lambda: router.route_topk(logits, 8), lambda: router.route_topk(logits[0], 8), lambda: router.route_topk(logits.half(), 8),
                 lambda: router.route_topk_bwd(torch.zeros(4, 8), logits, torch.zeros(4, 8, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call()
