"""4-bit weights with group scales: prepack, dense products, and the experts of a mixture layer.

``W[m, k] = (q[m, k] - z[m, k // group]) * s[m, k // group]`` with ``q`` and ``z`` in 0..15 (``z`` = 8 where none is given),
``s`` in the activation's type (bf16 or fp16) and groups of 32, 64 or 128 consecutive k of a row.  Lay the weights out
once at load time:

    A = layoutA_w4(qweight)            # uint8 [m, k/2], low nibble = even k   -> [m/16, ceil(k/64), 32, 16]
    S = layoutA_w4_groups(scales)      # [m, k/group]                           -> [m/16, k/group, 8, 2]
    Z = layoutA_w4_groups(zeros)       # uint8 [m, k/group], optional
    y = gemm_layoutA_w4(A, S, x, zeros=Z)

Every op also takes / keeps a leading expert dimension where it says so.  Like the other operators, each one checks its
tensors (a violated precondition raises ``RuntimeError``), allocates the result with torch and launches on the current
stream of the tensors' device; no op synchronises, and every one can be captured in a CUDA graph.  The reference has no
4-bit operators.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import Optional

import torch

from ._lib import check, lib
from .ext import _act_code, _bias_ptr, _chk, _cuda_contig, _map_args, _ptr, _status_ptr, _stream

__all__ = ["layoutA_w4", "layoutA_w4_inverse", "layoutA_w4_groups", "gemv_layoutA_w4", "gemm_layoutA_w4",
           "fused_experts_compute_w4"]

_GROUPS = (32, 64, 128)


def _on(t: torch.Tensor):
    """The tensors' device current for the launch (a no-op where it already is)."""
    return nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _same_device(like: torch.Tensor, *named) -> None:
    for t, name in named:
        if t is not None:
            _chk(t.device == like.device, f"{name} must be on the same device as the activations")


def layoutA_w4(W: torch.Tensor) -> torch.Tensor:
    """Row-major packed nibbles ``[m, k/2]`` uint8 (low nibble = even k) -> ``[m/16, ceil(k/64), 32, 16]``; a 3-D
    ``[E, m, k/2]`` keeps its leading dimension.  m % 16 == 0, k % 32 == 0."""
    _cuda_contig(W, "W")
    _chk(W.dtype == torch.uint8, "W must be a uint8 tensor of packed nibbles")
    _chk(W.dim() in (2, 3), "W must be a 2D or 3D tensor")
    m, k = W.shape[-2], 2 * W.shape[-1]
    _chk(m % 16 == 0 and k % 32 == 0 and k > 0, "layoutA_w4 needs m % 16 == 0 and k % 32 == 0")
    out = torch.empty(W.shape[:-2] + (m // 16, (k + 63) // 64, 32, 16), dtype=torch.uint8, device=W.device)
    rows = m * (W.shape[0] if W.dim() == 3 else 1)
    with _on(W):
        check(lib.mlk_layoutA_w4(W.data_ptr(), out.data_ptr(), rows, k, 0, _stream(W)))
    return out


def layoutA_w4_inverse(A: torch.Tensor, k: int) -> torch.Tensor:
    """``[m/16, ceil(k/64), 32, 16]`` (or with a leading expert dimension) -> row-major packed nibbles ``[m, k/2]``."""
    _cuda_contig(A, "A")
    R, kc = _packed_dims(A, "A")
    _chk(k > 0 and k % 32 == 0 and (k + 63) // 64 == kc, "k does not match the packed weights")
    out = torch.empty(A.shape[:-4] + (R * 16, k // 2), dtype=torch.uint8, device=A.device)
    with _on(A):
        check(lib.mlk_layoutA_w4(A.data_ptr(), out.data_ptr(), out.numel() // (k // 2), k, 1, _stream(A)))
    return out


def layoutA_w4_groups(values: torch.Tensor) -> torch.Tensor:
    """Scales or zero points ``[m, k/group]`` -> ``[m/16, k/group, 8, 2]`` (entry (r, h) = row r + 8 h of 16); a 3-D input
    keeps its leading dimension.  Scales are bf16 / fp16, zero points uint8."""
    _cuda_contig(values, "values")
    _chk(values.dtype in (torch.bfloat16, torch.float16, torch.uint8), "values must be bfloat16, float16 (scales) or uint8 (zero points)")
    _chk(values.dim() in (2, 3), "values must be a 2D or 3D tensor")
    m, G = values.shape[-2:]
    _chk(m % 16 == 0 and G > 0, "layoutA_w4_groups needs m % 16 == 0 and at least one group")
    out = torch.empty(values.shape[:-2] + (m // 16, G, 8, 2), dtype=values.dtype, device=values.device)
    rows = m * (values.shape[0] if values.dim() == 3 else 1)
    with _on(values):
        check(lib.mlk_layoutA_w4_groups(values.data_ptr(), out.data_ptr(), rows, G, values.element_size(), _stream(values)))
    return out


def _packed_dims(A: torch.Tensor, name: str, lead: int = -1):
    _chk(A.dtype == torch.uint8, f"{name} must be uint8 (packed by layoutA_w4)")
    _chk(A.dim() - 4 in ((0, 1) if lead < 0 else (lead,)), f"{name} must be [{'E, ' if lead == 1 else ''}m/16, ceil(k/64), 32, 16]")
    _chk(A.size(-2) == 32 and A.size(-1) == 16, f"{name}'s trailing dims must be (32, 16)")
    return A.size(-4), A.size(-3)


def _group(A, scales, zeros, x, k: int, name: str) -> int:
    """Group size told by the scales' shape, after checking all that belongs to one weight tensor against it."""
    _cuda_contig(A, name)
    _cuda_contig(scales, f"{name} scales")
    lead = A.shape[:-4]
    R, kc = _packed_dims(A, name, len(lead))
    _chk(scales.dtype == x.dtype, f"{name} scales must have the activation data type")
    _chk(scales.dim() == len(lead) + 4 and tuple(scales.shape[-2:]) == (8, 2) and scales.shape[:len(lead)] == lead and
         scales.size(-4) == R, f"{name} scales must be [{'E, ' if lead else ''}m/16, k/group, 8, 2] (from layoutA_w4_groups)")
    G = scales.size(-3)
    _chk(G > 0 and k % G == 0 and k // G in _GROUPS, f"{name}: k = {k} with {G} groups is not groups of 32, 64 or 128")
    _chk(kc == (k + 63) // 64, f"{name} holds {kc} blocks of 64 k, k = {k} needs {(k + 63) // 64}")
    if zeros is not None:
        _cuda_contig(zeros, f"{name} zeros")
        _chk(zeros.dtype == torch.uint8 and zeros.shape == scales.shape, f"{name} zeros must be uint8 in the shape of the scales")
    _same_device(x, (A, name), (scales, f"{name} scales"), (zeros, f"{name} zeros"))
    return k // G


def gemm_layoutA_w4(A, scales, B, alpha: float = 1, beta: float = 0, zeros=None, bias=None):
    """``C[n,m] = alpha * B W^T (+ bias)`` for any token count n (0 included), W in 4 bits: ``A`` from ``layoutA_w4``,
    ``scales`` / ``zeros`` from ``layoutA_w4_groups``, ``B[n,k]`` and C row-major.  Sums are held in fp32 and rounded once.
    ``beta`` is ignored, as by the other GEMMs.  Up to 16 tokens the weights' value is exact; larger calls multiply
    the value rounded to the activation type (what a dequantised checkpoint holds)."""
    _chk(B.is_cuda, "B must be a CUDA tensor")
    _chk(B.is_contiguous(), "B must be contiguous")
    _chk(B.dim() == 2, "B must be a 2D tensor")
    code = _act_code(B)
    n, k = B.shape
    R, _ = _packed_dims(A, "A", 0)
    group = _group(A, scales, zeros, B, k, "A")
    m = R * 16
    _same_device(B, (bias, "bias"))
    C = torch.empty((n, m), dtype=B.dtype, device=B.device)
    with _on(B):
        check(lib.mlk_gemm_layoutA_w4(A.data_ptr(), scales.data_ptr(), _ptr(zeros), group, B.data_ptr(), C.data_ptr(), m, n, k,
                                      code, alpha, _bias_ptr(bias, B, m), _status_ptr(B), _stream(B)))
    return C


def gemv_layoutA_w4(A, scales, B, alpha: float = 1, beta: float = 0, zeros=None, bias=None):
    """``y[1,m] = alpha * W x (+ bias)``: ``gemm_layoutA_w4`` for one token ``B[1,k]``."""
    _chk(B.dim() == 2 and B.size(0) == 1, "B must be a vector")
    return gemm_layoutA_w4(A, scales, B, alpha, beta, zeros, bias)


def fused_experts_compute_w4(w1, w1_scales, w2, w2_scales, activations, topk_ids, topk_weights, w1_zeros=None, w2_zeros=None,
                             experts_map=None, out: Optional[torch.Tensor] = None,
                             out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y[t] = sum_j topk_weights[t,j] * W2_e (silu(Wgate_e x_t) * (Wup_e x_t))``, ``e = topk_ids[t,j]``, expert weights in
    4 bits: ``w1 [E, 2I/16, ceil(H/64), 32, 16]`` (gate rows, then up rows) and ``w2 [E, H/16, ceil(I/64), 32, 16]`` from
    ``layoutA_w4``, scales and zero points from ``layoutA_w4_groups``; ``activations [T, H]`` bf16 / fp16, ``topk_ids``
    int32 ``[T, topk]``, ``topk_weights`` in the activations' type.  ``experts_map``: global -> local expert or -1, as in
    ``fused_experts_compute``; ids without an expert here contribute nothing.  ``out_dtype=torch.float32`` gives the
    un-rounded sums; ``out`` receives the result (every element is written).  A token's experts are added in
    slot order in fp32 with one rounding."""
    x = activations
    _cuda_contig(x, "activations")
    _chk(x.dim() == 2, "activations must be [T, H]")
    code = _act_code(x)
    T, H = x.shape
    _packed_dims(w1, "w1", 1)
    _packed_dims(w2, "w2", 1)
    E, I = w1.size(0), w1.size(1) * 8
    _chk(w1.size(1) % 2 == 0 and w2.size(0) == E and w2.size(1) * 16 == H and E > 0, "w1 must hold [E, 2I, H] and w2 [E, H, I]")
    g1 = _group(w1, w1_scales, w1_zeros, x, H, "w1")
    g2 = _group(w2, w2_scales, w2_zeros, x, I, "w2")
    _cuda_contig(topk_ids, "topk_ids")
    _cuda_contig(topk_weights, "topk_weights")
    _chk(topk_ids.dtype == torch.int32 and topk_ids.dim() == 2 and topk_ids.size(0) == T and topk_ids.size(1) > 0,
         "topk_ids must be int32 [T, topk]")
    _chk(topk_weights.dtype == x.dtype and topk_weights.shape == topk_ids.shape,
         "topk_weights must be [T, topk] in the activation data type")
    _same_device(x, (topk_ids, "topk_ids"), (topk_weights, "topk_weights"), (experts_map, "experts_map"), (out, "out"))
    mp, ml = _map_args(experts_map)
    dtype = x.dtype if out_dtype is None else out_dtype
    _chk(dtype in (x.dtype, torch.float32), "out_dtype must be the activation data type or torch.float32")
    if out is None:
        out = torch.empty((T, H), dtype=dtype, device=x.device)
    else:
        _cuda_contig(out, "out")
        _chk(out.shape == x.shape and out.dtype == dtype, "out must be [T, H] in the result's data type")
    topk = topk_ids.size(1)
    with _on(x):
        ws = torch.empty(lib.mlk_experts_w4_workspace_bytes(T, E, topk, H, I), dtype=torch.uint8, device=x.device)
        check(lib.mlk_fused_experts_compute_w4(
            w1.data_ptr(), w1_scales.data_ptr(), _ptr(w1_zeros), g1, w2.data_ptr(), w2_scales.data_ptr(), _ptr(w2_zeros), g2,
            x.data_ptr(), T, E, topk, H, I, topk_ids.data_ptr(), topk_weights.data_ptr(), out.data_ptr(), code,
            int(dtype == torch.float32 and x.dtype != torch.float32), mp, ml, ws.data_ptr(), ws.numel(), _status_ptr(x),
            _stream(x)))
    return out
