"""The error of attention's gradients against the formula in 64 bits, by norm and at lengths around the tiles' size."""
import pytest
import torch

from .test_attention_bwd_gpu import make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,window", [(4, 40, 0), (2, 77, 0), (2, 128, 0), (1, 256, 0), (1, 257, 0), (1, 600, 0), (1, 600, 16), (1, 600, 130)])
def test_two_roundings_at_any_length(native_lib, B, S, window):
    """On the way of a gradient stand two independent roundings to bf16 of about the same relative size, the products'
    operand (dX, or P) and the stored result. Together they are sqrt(2) times what rounding the exact gradient
    leaves, however many terms are added up, since the errors of the terms add up as the terms do. A tenth for chance
    (thousands of roundings to a norm) and for probabilities that have no rounding, as the first row's 1."""
    from pipelink_b200 import attention as att
    q, k, v, do = make(B, S, 4, 2, seed=S + window)
    out, lse, grads, _ = reference(q, k, v, do, window)
    got = att.attention_bwd(do, q, k, v, out, lse, window=window)
    for have, (name, want) in zip(got, grads.items()):
        error = float((have.double() - want).norm())
        rounding = float((want.to(torch.bfloat16).double() - want).norm())
        assert abs(error / (2 ** 0.5 * rounding) - 1) <= 0.1, (name, error / rounding)
