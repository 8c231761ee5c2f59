"""A block's branch in an MXFP8 session, both directions, for every dispatch: the same bits as its parts called one after
another."""
import pytest
import torch

from .test_block_gpu import session

pytestmark = pytest.mark.gpu


def parts(host, w, x, res, d_out, d_hidden, topk, **routing):
    """norm, router and ``forward`` / ``backward`` by hand, and the library products between them."""
    from pipelink_b200 import mok, norm, router
    n = norm.rmsnorm_fwd(x, w["norm"], res)
    logits = torch.mm(n.y, w["router"].T, out_dtype=torch.float32)
    experts, weights = router.route_topk(logits, topk, bias=host.block["bias"], **routing)
    out = host.forward(mok.Inputs(n.y, experts, weights), train=True)["output"].clone()
    g = {k: v.clone() for k, v in host.backward(d_out).items()}
    kw = {k: v for k, v in routing.items() if k in ("score", "renormalize", "scale")}
    d_logits = router.route_topk_bwd(g["d_router_weights"], logits, experts, **kw)
    d_y = torch.addmm(g["d_x"].float(), d_logits, w["router"].float()).to(torch.bfloat16)
    d_x, d_norm = norm.rmsnorm_bwd(d_y, n.hidden, n.rstd, w["norm"], d_hidden)
    return out, {**g, "d_x": d_x, "d_norm_weight": d_norm, "d_gate_weight": d_logits.T @ n.y.float()}


@pytest.mark.parametrize("dispatch", ["loads", "bulk", "fused"])
@pytest.mark.parametrize("tokens", [333, 512])
def test_branch_gradients_are_their_parts(native_lib, dispatch, tokens):
    routing = dict(score="sigmoid", groups=4, topk_groups=2, scale=2.5)
    host, w, x, res, d_out = session(("mx", 8, 512, 256, 2, tokens), "mxfp8", train=True, seed=tokens, **routing,
                                     gate_bias=0.1 * torch.randn(8, device="cuda"))
    host.pull_variant, host.fused_dispatch = ("bulk" if dispatch == "bulk" else "loads"), dispatch == "fused"
    d_hidden = 0.5 * d_out.flip(0).contiguous()
    want_out, want = parts(host, w, x, res, d_out, d_hidden, 2, **routing)
    assert all(torch.isfinite(v.float()).all() and (v != 0).any() for v in want.values())
    for train in (True, False, True):                # kept by the forward pass, or taken again from the routed rows
        assert torch.equal(host.forward_block(x, res, train=train)["output"], want_out)
        got = host.backward_block(d_out, d_hidden, recompute=not train)
        assert got.keys() == want.keys()
        for name in want:
            assert torch.equal(got[name], want[name]), (train, name)
