"""A block's branch captured into a graph, both directions, and replayed on new contents of the same tensors; two calls of
backward_block after one of forward_block; two sessions at once on two streams."""
import pytest
import torch

from .test_block_gpu import session

pytestmark = pytest.mark.gpu


def step(host, x, res, d_out, d_hidden, check=False):
    out = host.forward_block(x, res, check=check, train=True)
    got = {"output": out["output"], "hidden": out["hidden"]}
    return {**got, **host.backward_block(d_out, d_hidden, check=check)}


def copies(d):
    return {k: v.clone() for k, v in d.items()}


def same(got, want):
    for name in want:
        assert torch.equal(got[name], want[name]), name


@pytest.mark.parametrize("precision", ["bf16", "mxfp8"])
def test_captured_and_replayed(native_lib, precision):
    host, _, x, res, d_out = session(("graph", 8, 256, 256, 2, 200), precision, train=True, seed=11)
    inputs = [[x, res, d_out, res.flip(0).contiguous()], [res, x, d_out.flip(0).contiguous(), x]]
    want = [copies(step(host, *i, check=True)) for i in inputs]
    again = host.backward_block(inputs[1][2], inputs[1][3])                       # of the same forward call
    same(again, {k: v for k, v in want[1].items() if k in again})
    static = [t.clone() for t in inputs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(host, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(host, *static)
    for i in (0, 1, 0):
        for t, new in zip(static, inputs[i]):
            t.copy_(new)
        graph.replay()
        same(captured, want[i])
    host.status.check("replays")


def test_two_sessions_at_once(native_lib):
    one, _, x, res, d_out = session(("one", 8, 256, 256, 2, 333), "mxfp8", train=True, seed=1)
    two, _, x2, res2, d_out2 = session(("two", 4, 512, 256, 1, 200), "mxfp8", train=True, seed=2)
    args = [(one, x, res, d_out, x), (two, x2, res2, d_out2, None)]
    want = [copies(step(*a, check=True)) for a in args]
    torch.cuda.synchronize()
    for _ in range(5):
        streams = [torch.cuda.Stream() for _ in args]
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(copies(step(*a)))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            same(g, w)
