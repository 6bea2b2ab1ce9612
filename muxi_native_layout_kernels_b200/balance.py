"""Balance loss of the mixture router, per-expert counts, and the gradient with respect to the router logits.

For a token t with logits l: ``p = softmax(l)`` (``score_fun`` 0) or ``sigmoid(l) / sum sigmoid(l)`` (1).  With c[b, e] the
picks of expert e by the counted tokens of sequence b (``experts_ids`` as ``fused_routing_gate`` writes them) and n_b the
number of those tokens,

    loss = coef / B * sum_b  E / (topk * n_b^2) * sum_e c[b, e] * sum_{t in b} p[t, e]

which is coef when every expert gets its share and grows with the imbalance; the counts are constants of the gradient.
The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as _forward

from ._lib import lib
from .ext import _chk, _cuda_contig, _ptr
from .w4 import _LIMIT, _device_of_thread, _fits, _launch, _same_device

__all__ = ["router_balance_loss", "expert_counts"]

_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 3}


def _mask_ptr(mask: Optional[torch.Tensor], T: int):
    if mask is None:
        return None
    _cuda_contig(mask, "token_mask")
    _chk(mask.dtype in (torch.bool, torch.uint8) and mask.dim() == 1 and mask.numel() == T, "token_mask must be bool or uint8 [T]")
    return mask.data_ptr()


def _checked(x, ids, score_fun, mask, cu):
    """Like the other operators' checks: the first test is the whole of it, the rest finds the message."""
    d, xs, s = x.get_device(), x.shape, ids.shape
    if (x.is_cuda and ids.get_device() == d and x.is_contiguous() and ids.is_contiguous() and x.dtype in _CODES
            and ids.dtype is torch.int32 and len(xs) == 2 and len(s) == 2 and xs[1] > 0 and s[0] == xs[0] and s[1] > 0
            and score_fun in (0, 1) and xs[0] < _LIMIT and xs[1] < _LIMIT and s[1] < _LIMIT
            and (mask is None or (mask.get_device() == d and mask.is_contiguous() and mask.shape == xs[:1]
                                  and (mask.dtype is torch.bool or mask.dtype is torch.uint8)))
            and (cu is None or (cu.get_device() == d and cu.is_contiguous() and cu.dtype is torch.int32 and cu.dim() == 1
                                and 2 <= cu.shape[0] <= _LIMIT))):
        return
    _cuda_contig(x, "gating_output")
    _cuda_contig(ids, "experts_ids")
    _chk(x.dtype in _CODES, "gating_output must be bfloat16, float16 or float32")
    _chk(x.dim() == 2 and x.size(1) > 0, "gating_output must be [T, E]")
    T = x.size(0)
    _chk(ids.dtype == torch.int32 and ids.dim() == 2 and ids.size(0) == T and ids.size(1) > 0, "experts_ids must be int32 [T, topk]")
    _chk(score_fun in (0, 1), "score_fun must be 0 (softmax) or 1 (sigmoid)")
    _mask_ptr(mask, T)
    if cu is not None:
        _cuda_contig(cu, "cu_seqlens")
        _chk(cu.dtype == torch.int32 and cu.dim() == 1 and cu.numel() >= 2, "cu_seqlens must be int32 [sequences + 1]")
    _same_device(x, (ids, "experts_ids"), (mask, "token_mask"), (cu, "cu_seqlens"))
    _fits(T, x.size(1), ids.size(1), 0 if cu is None else cu.numel() - 1)
    raise RuntimeError("router_balance_loss: bad arguments")


def _loss(x, ids, score_fun, coef, mask, cu, want_grad: bool):
    """(loss, counts, d loss / d p behind the workspace's start, gradient or None), on the current stream."""
    if _device_of_thread() != x.get_device():             # the size of the workspace is the current device's
        with torch.cuda.device(x.get_device()):
            return _loss(x, ids, score_fun, coef, mask, cu, want_grad)
    T, E = x.shape
    B = 1 if cu is None else cu.shape[0] - 1
    loss = x.new_empty((), dtype=torch.float32)
    counts = x.new_empty((E,), dtype=torch.int32)
    grad = torch.empty_like(x) if want_grad else None
    nbytes = lib.mlk_router_balance_workspace_bytes(T, E, B)
    # d loss / d p [B, E] comes first (the backward pass reads it again); a small batch with its gradient needs neither
    head = 0 if want_grad and nbytes == 0 else (4 * B * E + 255) // 256 * 256
    ws, at = None, None
    if head:
        ws = x.new_empty((head + nbytes,), dtype=torch.uint8)
        at = ws.data_ptr()
    _launch(x.get_device(), lib.mlk_router_balance_loss, x.data_ptr(), ids.data_ptr(), _ptr(mask), _ptr(cu), T, E, ids.shape[1], B,
            score_fun, coef, _CODES[x.dtype], loss.data_ptr(), counts.data_ptr(), at, _ptr(grad), at + head if nbytes else None,
            nbytes)
    return loss, counts, ws, grad


def _grad(grad_loss, x, dprob, mask, cu, score_fun):
    grad = torch.empty_like(x)
    _launch(x.get_device(), lib.mlk_router_balance_grad, x.data_ptr(), _ptr(mask), _ptr(cu), x.shape[0], x.shape[1],
            1 if cu is None else cu.shape[0] - 1, score_fun, _CODES[x.dtype], dprob.data_ptr(), grad_loss.data_ptr(),
            grad.data_ptr())
    return grad


class _BalanceGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad_loss, x, dprob, mask, cu, score_fun):
        return _grad(grad_loss, x, dprob, mask, cu, score_fun)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("router_balance_loss can be differentiated once")


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, score_fun, coef, mask, cu):
        loss, counts, dprob, _ = _loss(x, ids, score_fun, coef, mask, cu, False)
        ctx.save_for_backward(x, dprob, mask, cu)
        ctx.score_fun = score_fun
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)          # else every backward pass fills zeros for the counts
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None, None
        # with create_graph the step is recorded itself, as one that has no derivative
        call = _BalanceGrad.apply if torch.is_grad_enabled() else _grad
        return call(grad_loss, *ctx.saved_tensors, ctx.score_fun), None, None, None, None, None


def router_balance_loss(gating_output: torch.Tensor, experts_ids: torch.Tensor, score_fun: int = 0, coef: float = 1.0, *,
                        token_mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
                        return_grad: bool = False):
    """``(loss, counts)``: fp32 scalar and int32 ``[E]``; ``loss`` can be differentiated with respect to ``gating_output``.

    ``gating_output [T, E]`` bf16, fp16 or fp32 logits (E <= 1024); ``experts_ids`` int32 ``[T, topk]``, ids outside
    ``[0, E)`` count nowhere.  ``token_mask [T]`` (bool or uint8): only tokens with a nonzero entry are counted.
    ``cu_seqlens`` int32 ``[B + 1]``, not decreasing: the loss is the mean over the B sequences (an empty one adds 0); tokens
    behind the last sequence are in none.  What the logits of tokens that are not counted hold (NaN included) has no
    influence, and their gradient is 0; a token whose logits are all -inf has no distribution and adds 0.
    ``return_grad=True``: ``(loss, counts, d loss / d gating_output)`` in one call, for callers that write their backward
    pass by hand and for captured steps (nothing is recorded for autograd).  A recorded call can be captured together with its
    backward pass as long as no graph recorded outside the capture still holds the same leaves.  Forward-mode derivatives (dual
    tensors) and second derivatives are refused.
    Probabilities, sums and the loss are fp32, added in a fixed order; the gradient is rounded once to the logits' type."""
    _checked(gating_output, experts_ids, score_fun, token_mask, cu_seqlens)
    if _forward._current_level >= 0:          # a dual tensor has no requires_grad: its tangent would be lost unseen
        _chk(_forward.unpack_dual(gating_output).tangent is None, "router_balance_loss has no forward-mode derivative")
    if return_grad:
        loss, counts, _, grad = _loss(gating_output.detach(), experts_ids, score_fun, float(coef), token_mask, cu_seqlens, True)
        return loss, counts, grad
    if not (gating_output.requires_grad and torch.is_grad_enabled()):
        return _loss(gating_output, experts_ids, score_fun, float(coef), token_mask, cu_seqlens, False)[:2]
    return _BalanceLoss.apply(gating_output, experts_ids, score_fun, float(coef), token_mask, cu_seqlens)


def expert_counts(experts_ids: torch.Tensor, num_experts: int, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int32 ``[num_experts]``: how often each expert is picked in ``experts_ids`` (int32 ``[T, topk]``) by the tokens whose
    ``token_mask`` entry (bool or uint8 ``[T]``) is not zero.  Ids outside the range count nowhere."""
    _cuda_contig(experts_ids, "experts_ids")
    _chk(experts_ids.dtype == torch.int32 and experts_ids.dim() == 2 and experts_ids.size(1) > 0, "experts_ids must be int32 [T, topk]")
    T, topk = experts_ids.shape
    mask = _mask_ptr(token_mask, T)
    _same_device(experts_ids, (token_mask, "token_mask"))
    _fits(T, topk, num_experts)
    counts = experts_ids.new_empty((num_experts,))
    _launch(experts_ids.get_device(), lib.mlk_expert_counts, experts_ids.data_ptr(), mask, T, topk, num_experts, counts.data_ptr())
    return counts
