"""RMS norm of the residual stream: the step between two branches of a transformer block, both directions.

``rmsnorm_fwd`` adds the branch's output to the residual stream, normalises the sum and writes it as bf16, as the
MXFP8 rows and scales the experts' dispatch gathers (``mok.mxfp8_quantize``'s format and bytes), or both, in one
launch; ``rmsnorm_bwd`` returns the gradient that both summands share and the weight's.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .mok import _ptr, _stream, dense, device_of, like, rows_of


class Normed(NamedTuple):
    hidden: torch.Tensor        # bf16, x + residual (x itself without a residual): the stream, and what the backward pass reads
    rstd: torch.Tensor          # f32 [rows]
    y: torch.Tensor | None      # bf16, like x
    fp8: torch.Tensor | None    # u8 [rows up to a multiple of 128, width], E4M3; rows past the last are zeros
    sc: torch.Tensor | None     # u8 [that / 128, width / 128, 32, 16]


def _check(weight, *rows):
    """Width and device of the rows, which have one shape [..., width] (None: one that is not given)."""
    shape, device = rows[0].shape, rows[0].device
    width = shape[-1] if shape else 0
    if width < 1:
        raise ValueError("rows are [..., width]")
    for t in rows:
        if t is not None and (t.dtype is not torch.bfloat16 or t.shape != shape or t.device != device or not t.is_cuda):
            raise ValueError(f"the rows are bf16 tensors of one shape, here {tuple(shape)}, on one CUDA device")
    if weight.dtype is not torch.bfloat16 or weight.shape != (width,) or weight.device != device:
        raise ValueError(f"weight is bf16 [{width}] on the rows' device")
    return width, device


def _check_into(into: Normed, residual, out, rows, width, padded, device):
    for name, t, n, dtype in (("hidden", into.hidden if residual is not None else None, rows * width, torch.bfloat16),
                              ("rstd", into.rstd, rows, torch.float32), ("y", into.y, rows * width, torch.bfloat16),
                              ("fp8", into.fp8, padded * width, torch.uint8), ("sc", into.sc, padded * width // 32, torch.uint8)):
        if t is not None and (t.numel() != n or t.dtype != dtype or t.device != device or not t.is_contiguous()):
            raise ValueError(f"into.{name} is a contiguous {dtype} tensor of {n} elements on {device}")
    if into.rstd is None or (into.y is None) != (out == "mxfp8") or (into.fp8 is None) != (out == "bf16") or \
            (into.sc is None) != (out == "bf16") or (residual is not None and into.hidden is None):
        raise ValueError("into holds the outputs that were asked for, and no others")


def rmsnorm_fwd(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-5,
                out: str = "bf16", into: Normed | None = None) -> Normed:
    """x, residual bf16 [..., width], weight bf16 [width]. `out`: "bf16", "mxfp8" (width a multiple of 128) or "both".
    hidden = bf16(x + residual), y = bf16(hidden * rstd * weight). `into` gives the tensors to write (contiguous; those of
    an earlier call of the same shape, or a session's buffers) instead of new ones; its hidden may be the residual itself.
    A row's squares and their sum are fp32: where the sum passes 3.4e38 (numbers of 1e18 and more) y is 0."""
    if out not in ("bf16", "mxfp8", "both"):
        raise ValueError("out is 'bf16', 'mxfp8' or 'both'")
    width, dev = _check(weight, x, residual)
    if not eps >= 0.0:
        raise ValueError("eps is not negative")
    if out != "bf16" and width % 128:
        raise ValueError("MXFP8 output wants a width that is a multiple of 128")
    rows = x.numel() // width
    padded = (rows + 127) // 128 * 128
    with device_of(x):
        x2, ld_x = rows_of(x)
        r2, ld_r = rows_of(residual) if residual is not None else (None, 0)
        weight = dense(weight)
        if into is None:
            fp8 = sc = None
            if out != "bf16":
                fp8 = x.new_empty((padded, width), dtype=torch.uint8)
                sc = x.new_empty((padded // 128, width // 128, 32, 16), dtype=torch.uint8)
            into = Normed(like(x) if residual is not None else x, x.new_empty(rows, dtype=torch.float32),
                          like(x) if out != "mxfp8" else None, fp8, sc)
        else:
            _check_into(into, residual, out, rows, width, padded, dev)
        _lib.call("plb_rmsnorm_fwd", x2.data_ptr(), ld_x, _ptr(r2), ld_r, weight.data_ptr(), rows, width, eps,
                  into.hidden.data_ptr() if residual is not None else 0, into.rstd.data_ptr(), _ptr(into.y), _ptr(into.fp8),
                  _ptr(into.sc), _stream())
    return into if residual is not None else into._replace(hidden=x)


def rmsnorm_bwd(d_y: torch.Tensor, hidden: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                d_hidden: torch.Tensor | None = None):
    """Gradient of ``rmsnorm_fwd``: (d_x, d_weight). d_x (bf16, like hidden) is the gradient of x and of the residual alike,
    d_weight f32 [width]. `d_hidden` is the gradient that reaches the residual stream past the norm. An MXFP8 output has
    its bf16 value's gradient. The same inputs give the same bits."""
    width, dev = _check(weight, hidden, d_y, d_hidden)
    rows = hidden.numel() // width
    if rstd.shape != (rows,) or rstd.dtype is not torch.float32 or rstd.device != dev:
        raise ValueError("rstd is f32 [rows], as rmsnorm_fwd returns it")
    with device_of(hidden):
        g2, ld_g = rows_of(d_y)
        h2, ld_h = rows_of(hidden)
        e2, ld_e = rows_of(d_hidden) if d_hidden is not None else (None, 0)
        rstd, weight = rstd.contiguous(), dense(weight)
        d_x = like(hidden)
        d_weight = hidden.new_empty(width, dtype=torch.float32)
        nbytes = _lib.load().plb_rmsnorm_bwd_workspace_bytes(rows, width)
        workspace = hidden.new_empty(nbytes, dtype=torch.uint8)
        _lib.call("plb_rmsnorm_bwd", g2.data_ptr(), ld_g, h2.data_ptr(), ld_h, rstd.data_ptr(), weight.data_ptr(), _ptr(e2), ld_e,
                  rows, width, d_x.data_ptr(), d_weight.data_ptr(), workspace.data_ptr(), nbytes, _stream())
    return d_x, d_weight
