"""Norm, router and experts as one branch, and a whole transformer block's step with attention in front of it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def session(shape_args, precision="mxfp8", train=False, seed=0, **routing):
    from pipelink_b200 import mok
    shape = mok.Shape(*shape_args)
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda scale, *s: (scale * torch.randn(*s, generator=g, device="cuda")).to(torch.bfloat16)
    E, H, I = shape.experts, shape.hidden, shape.intermediate
    w = dict(gate=draw(0.05, E, I, H), up=draw(0.05, E, I, H), down=draw(0.05, E, H, I), norm=1 + draw(0.1, H), router=draw(0.05, E, H))
    host = mok.MoKHost(shape, precision=precision)
    host.load_weights(w["gate"], w["up"], w["down"], train=train)
    host.load_block(w["norm"], w["router"], **routing)
    return host, w, draw(1.0, shape.tokens, H), draw(2.0, shape.tokens, H), draw(1.0, shape.tokens, H)


@pytest.mark.parametrize("precision,dispatch", [("mxfp8", "loads"), ("mxfp8", "bulk"), ("mxfp8", "fused"), ("bf16", "loads")])
@pytest.mark.parametrize("with_residual", [False, True])
def test_branch_is_its_parts(native_lib, precision, dispatch, with_residual):
    """The same bits as norm, router and ``forward`` called one after another (a batch that no tile divides)."""
    from pipelink_b200 import mok, norm, router
    routing = dict(score="sigmoid", groups=4, topk_groups=2, scale=2.5)
    host, w, x, res, _ = session(("parts", 8, 256, 256, 2, 333), precision, **routing, gate_bias=0.1 * torch.randn(8, device="cuda"))
    host.pull_variant, host.fused_dispatch = ("bulk" if dispatch == "bulk" else "loads"), dispatch == "fused"
    res = res if with_residual else None
    for _ in range(2):                        # a second call on the same buffers
        got = {k: v.clone() for k, v in host.forward_block(x, res).items()}
        n = norm.rmsnorm_fwd(x, w["norm"], res)
        logits = torch.mm(n.y, w["router"].T, out_dtype=torch.float32)
        experts, weights = router.route_topk(logits, 2, bias=host.block["bias"], **routing)
        assert torch.equal(got["hidden"], n.hidden) and torch.equal(got["experts"], experts) and torch.equal(got["router"], weights)
        assert torch.equal(got["output"], host.forward(mok.Inputs(n.y, experts, weights))["output"])
        x = got["output"]


def reference(x, res, w, experts, scale, eps=1e-5):
    """The branch in 64 bits with autograd, the choice of experts given."""
    leaf = {k: v.double().requires_grad_(True) for k, v in {**w, "x": x, "res": res}.items()}
    h = leaf["x"] + leaf["res"]
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * leaf["norm"]
    p = torch.softmax(n @ leaf["router"].T, 1).gather(1, experts.long())
    weight = scale * p / p.sum(1, keepdim=True)
    out = torch.zeros_like(n)
    for e in range(w["router"].shape[0]):
        t, slot = (experts == e).nonzero(as_tuple=True)
        y = torch.nn.functional.silu(n[t] @ leaf["gate"][e].T) * (n[t] @ leaf["up"][e].T) @ leaf["down"][e].T
        out = out.index_add(0, t, y * weight[t, slot, None])
    return leaf, h, out


def near(got, want, steps, name):
    """`steps` roundings to bf16 on the way, each off by at most 2^-8 of what it rounds, so of its norm."""
    rel = float((got.double() - want).norm() / want.norm())
    assert rel <= steps * 2.0 ** -8, (name, rel)


def test_branch_gradients(native_lib):
    """bf16 session against autograd. Roundings on the way of a gradient: hidden, y, gate, up, hidden rows, each expert's
    row, the output, and as many in the other direction."""
    host, w, x, res, d_out = session(("grad", 8, 512, 256, 2, 384), "bf16", train=True, scale=1.5)
    d_hidden = 0.5 * d_out.flip(0).contiguous()
    got = host.forward_block(x, res, train=True)
    leaf, h, out = reference(x, res, w, got["experts"], 1.5)
    near(got["output"], out.detach(), 7, "output")
    (out * d_out.double()).sum().add((h * d_hidden.double()).sum()).backward()
    grads = host.backward_block(d_out, d_hidden)
    for name, key in (("d_x", "x"), ("d_x", "res"), ("d_norm_weight", "norm"), ("d_gate_weight", "router"), ("d_w_routed_gate", "gate"),
                      ("d_w_routed_up", "up"), ("d_w_routed_down", "down")):
        near(grads[name], leaf[key].grad, 14, name)
    again = {k: v.clone() for k, v in grads.items()}
    host.forward_block(x, res)
    for name, value in host.backward_block(d_out, d_hidden, recompute=True).items():
        assert torch.equal(value, again[name]), name


def test_whole_block(native_lib):
    """Attention with its projections, then the expert branch, one step of both passes: 300 tokens in two sequences. The
    projections are library products. Nine roundings more than the branch alone in each direction."""
    from pipelink_b200 import attention as att, norm
    H, heads, kv, B, S = 256, 2, 1, 2, 150
    host, w, x, _, d_out = session(("block", 8, H, 256, 2, B * S), "bf16", train=True, seed=3)
    g = torch.Generator(device="cuda").manual_seed(7)
    wq, wk, wv = ((torch.randn(H, n * 128, generator=g, device="cuda") / math.sqrt(H)).to(torch.bfloat16) for n in (heads, kv, kv))
    n1 = norm.rmsnorm_fwd(x, w["norm"])
    q, k, v = (n1.y @ p for p in (wq, wk, wv))
    shaped = [q.view(B, S, heads, 128), k.view(B, S, kv, 128), v.view(B, S, kv, 128)]
    o, lse = att.attention_fwd(*shaped)
    got = host.forward_block(o.view(B * S, H), x, train=True)
    grads = host.backward_block(d_out, d_out)
    dq, dk, dv = att.attention_bwd(grads["d_x"].view(o.shape), *shaped, o, lse)
    d_y = dq.view(B * S, -1) @ wq.T + dk.view(B * S, -1) @ wk.T + dv.view(B * S, -1) @ wv.T
    d_x, d_norm = norm.rmsnorm_bwd(d_y, n1.hidden, n1.rstd, w["norm"], grads["d_x"])

    x64 = x.double().requires_grad_(True)
    y = x64 / torch.sqrt((x64 * x64).mean(1, keepdim=True) + 1e-5) * w["norm"].double()
    q64, k64, v64 = ((y @ p.double()).view(B, S, -1, 128).transpose(1, 2) for p in (wq, wk, wv))
    s = (q64 @ k64.transpose(-1, -2) / math.sqrt(128)).masked_fill(torch.ones(S, S, device="cuda").triu(1).bool(), -math.inf)
    o64 = (torch.softmax(s, -1) @ v64).transpose(1, 2).reshape(B * S, H)
    near(o.view(B * S, H), o64.detach(), 5, "attention")
    leaf, h, out = reference(o.view(B * S, H), x, w, got["experts"], 1.0)
    (out * d_out.double() + h * d_out.double()).sum().backward()
    near(grads["d_x"], leaf["x"].grad, 14, "into the attention branch")
    (o64 * leaf["x"].grad).sum().add((x64 * leaf["x"].grad).sum()).backward()
    near(d_x, x64.grad, 23, "d_x")


def test_branch_refusals(native_lib):
    from pipelink_b200 import mok
    host = mok.MoKHost(mok.Shape("refuse", 4, 256, 256, 1, 64))
    x = torch.zeros(64, 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        host.forward_block(x)
    with pytest.raises(ValueError):
        host.load_block(torch.ones(128), torch.zeros(4, 256))
    with pytest.raises(ValueError):
        host.load_block(torch.ones(256), torch.zeros(4, 256), topk=2)
    host.load_block(torch.ones(256), torch.zeros(4, 256))
    with pytest.raises(RuntimeError):
        host.forward_block(x)
    with pytest.raises(RuntimeError):
        host.backward_block(x)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    host.load_weights(z(4, 256, 256), z(4, 256, 256), z(4, 256, 256))
    with pytest.raises(RuntimeError):
        host.forward_block(x, train=True)
    with pytest.raises(ValueError):
        host.forward_block(x[:32])
    assert (host.forward_block(x)["output"] == 0).all()


def test_branch_of_its_own_output(native_lib):
    """x may be the tensor an earlier call returned, and its gradients are still those of the values it had."""
    host, w, x, _, d_out = session(("own", 4, 256, 256, 2, 200), "bf16", train=True, seed=5)
    first = host.forward_block(x, train=True)["output"]
    kept = first.clone()
    host.forward_block(first, train=True)
    got = {k: v.clone() for k, v in host.backward_block(d_out.T.contiguous().T).items()}     # strides other than the tested
    host.forward_block(kept, train=True)
    for name, value in host.backward_block(d_out).items():
        assert torch.equal(value, got[name]), name


def test_branch_order_of_calls(native_lib):
    from pipelink_b200 import mok
    host, _, x, _, d_out = session(("order", 4, 256, 256, 1, 128), "bf16", train=True)
    got = host.forward_block(x)
    with pytest.raises(RuntimeError):                 # kept nothing for the backward pass
        host.backward_block(d_out)
    with pytest.raises(ValueError):
        host.backward_block(d_out[:64], recompute=True)
    with pytest.raises(ValueError):
        host.backward_block(d_out.float(), recompute=True)
    with pytest.raises(ValueError):
        host.forward_block(x.float())
    host.forward_block(x)
    host.backward_block(d_out, recompute=True)
    host.forward(mok.Inputs(x, got["experts"].clone(), got["router"].clone()), train=True)
    with pytest.raises(RuntimeError):                 # another call's routes and rows are in the buffers
        host.backward_block(d_out)
