"""What may come between forward_block and backward_block: nothing that writes the session's routes, rows or weights."""
import pytest
import torch

from .test_block_gpu import session

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("precision", ["bf16", "mxfp8"])
def test_no_backward_of_mixed_calls(native_lib, precision):
    """A step of the host pipeline, a schedule of other routes or other weights in between: refused, and right again after
    the next forward_block."""
    host, w, x, res, d_out = session(("mixed", 4, 256, 256, 2, 160), precision, train=True)
    host.forward_block(x, res, train=True)
    want = {k: v.clone() for k, v in host.backward_block(d_out).items()}
    routes = torch.randint(0, 4, (1, 160, 1)).repeat(1, 1, 2)
    routes[..., 1] = (routes[..., 0] + 1) % 4

    def pipeline():
        pipe = host.host_pipeline()
        pin = lambda t: t.cpu().pin_memory()
        out = torch.empty(160, 256, dtype=torch.bfloat16).pin_memory()
        pipe.submit(pin(x.flip(0)), pin(routes.int()), pin(torch.full((160, 2), 0.5)), out)
        pipe.drain()

    between = [pipeline, lambda: host.schedule_into(routes.cuda().int()),
               lambda: host.load_weights(w["gate"], w["up"], w["down"], train=True)]
    for step in between:
        host.forward_block(x, res, train=True)
        step()
        for recompute in (False, True):
            with pytest.raises(RuntimeError):
                host.backward_block(d_out, recompute=recompute)
        host.forward_block(x, res, train=True)
        for name, value in host.backward_block(d_out).items():
            assert torch.equal(value, want[name]), name


def test_a_groups_session_has_no_block(native_lib):
    """Its epilogue and its dispatch read what the group's ranks pushed."""
    from pipelink_b200 import ep, mok
    shape = mok.Shape("group", 4, 256, 256, 2, 128)
    group = ep.LocalGroup(shape, 1, "cuda")
    try:
        host = ep.EpMoKHost(shape, 0, group)
        with pytest.raises(ValueError):
            host.load_block(torch.ones(256), torch.zeros(4, 256))
    finally:
        group.close()


def test_nothing_is_recorded_for_autograd(native_lib):
    """Inputs that want gradients leave none of autograd's records in the session's buffers: the gradients are
    backward_block's, and a record would grow with every call."""
    host, w, x, res, d_out = session(("leaf", 4, 256, 256, 2, 160), "bf16", train=True)
    want = host.forward_block(x, train=True)["output"].clone()
    leaf = x.clone().requires_grad_(True)
    for residual in (None, res.clone().requires_grad_(True)):
        got = host.forward_block(leaf, residual, train=True)
        assert not any(t.requires_grad for t in got.values()) and not host.block["hidden"].requires_grad
        assert residual is not None or torch.equal(got["output"], want)
        assert not any(t.requires_grad for t in host.backward_block(d_out.clone().requires_grad_(True)).values())
