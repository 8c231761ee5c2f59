"""Routing of tokens to experts: the choice and its weights from router logits, and the weights' gradient.

``route_topk`` gives what a MoE session takes (``mok.Inputs``: experts, router); ``route_topk_bwd`` takes the
``d_router_weights`` its backward pass returns.
"""
from __future__ import annotations

import torch

from . import _lib
from .mok import _ptr, _stream, device_of, like, rows_of

_SCORES = {"softmax": 0, "sigmoid": 1}
_DTYPES = (torch.float32, torch.bfloat16)
MAX_EXPERTS, MAX_TOPK, MAX_GROUPS = 1024, 32, 32


def _check(logits, topk, score):
    if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError("logits are a CUDA f32 or bf16 tensor [tokens, experts]")
    experts = logits.shape[1]
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= topk <= min(MAX_TOPK, experts):
        raise ValueError(f"1 to {MAX_EXPERTS} experts, of which 1 to {MAX_TOPK} are chosen")
    if score not in _SCORES:
        raise ValueError("score is 'softmax' or 'sigmoid'")


def route_topk(logits: torch.Tensor, topk: int, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
               topk_groups: int = 1, group_score: str = "top2", renormalize: bool = True, scale: float = 1.0,
               into: tuple[torch.Tensor, torch.Tensor] | None = None):
    """logits [tokens, experts] -> (experts i32 [tokens, topk], weights f32 [tokens, topk]), best first, ties to the lowest index.

    The choice goes by score + bias (f32 [experts]; a balance bias that the weights do not see). With groups > 1 only the
    `topk_groups` best of `groups` equal runs of experts take part, a run's score being its best ("max") or the sum of its
    two best ("top2"). Weights are the scores of the chosen, divided by their sum with `renormalize`, times `scale`. A logit
    of -inf masks an expert (chosen only where nothing else is left, with weight 0). Choices are exact: scores that fp32
    cannot tell apart are told apart. `into` gives the two contiguous tensors to write (a session's buffers)."""
    _check(logits, topk, score)
    tokens, experts = logits.shape
    dev = logits.device
    if group_score not in ("top2", "max"):
        raise ValueError("group_score is 'top2' or 'max'")
    if not 1 <= groups <= MAX_GROUPS or experts % groups or not 1 <= topk_groups <= groups or topk > topk_groups * (experts // groups):
        raise ValueError(f"groups (at most {MAX_GROUPS}) divide the experts, and the kept ones hold at least topk experts")
    if bias is not None and (bias.shape != (experts,) or bias.dtype != torch.float32 or bias.device != dev):
        raise ValueError("bias is f32 [experts] on the logits' device")
    if scale != scale:
        raise ValueError("scale is a number")
    with device_of(logits):
        x, ld = rows_of(logits)
        bias = bias.contiguous() if bias is not None else None
        if into is None:
            chosen = logits.new_empty((tokens, topk), dtype=torch.int32)
            weights = logits.new_empty((tokens, topk), dtype=torch.float32)
        else:
            chosen, weights = into
            for t, dtype in ((chosen, torch.int32), (weights, torch.float32)):
                if t.numel() != tokens * topk or t.dtype is not dtype or t.device != dev or not t.is_contiguous():
                    raise ValueError("into holds contiguous i32 and f32 tensors of tokens * topk elements on the logits' device")
        _lib.call("plb_route_topk", x.data_ptr(), ld, int(x.dtype == torch.bfloat16), _ptr(bias), tokens, experts, topk,
                  _SCORES[score], groups, topk_groups, int(group_score == "top2"), int(renormalize), float(scale), chosen.data_ptr(),
                  weights.data_ptr(), _stream())
    return chosen, weights


def route_topk_bwd(d_weights: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, *, score: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``route_topk``'s weights: d_logits [tokens, experts] in the logits' type, for the chosen `experts`
    (bias and groups decide the choice alone and have no gradient)."""
    topk = experts.shape[1] if experts.dim() == 2 else 0
    _check(logits, topk, score)
    tokens, dev = logits.shape[0], logits.device
    if experts.shape != (tokens, topk) or experts.dtype is not torch.int32 or experts.device != dev:
        raise ValueError("experts are i32 [tokens, topk] on the logits' device")
    if d_weights.shape != (tokens, topk) or d_weights.dtype is not torch.float32 or d_weights.device != dev:
        raise ValueError("d_weights are f32 [tokens, topk] on the logits' device")
    if scale != scale:
        raise ValueError("scale is a number")
    with device_of(logits):
        x, ld = rows_of(logits)
        d_weights, experts = d_weights.contiguous(), experts.contiguous()
        d_logits = like(logits)
        _lib.call("plb_route_topk_bwd", d_weights.data_ptr(), x.data_ptr(), ld, int(x.dtype == torch.bfloat16), experts.data_ptr(),
                  tokens, logits.shape[1], topk, _SCORES[score], int(renormalize), float(scale), d_logits.data_ptr(), _stream())
    return d_logits
