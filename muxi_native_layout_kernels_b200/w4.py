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

from typing import Optional

import torch

from ._lib import check, lib
from .ext import _SYNC_BUFFERS, _bias_ptr, _chk, _cuda_contig, _map_args, _ptr, _status_ptr

__all__ = ["layoutA_w4", "layoutA_w4_inverse", "layoutA_w4_groups", "gemv_layoutA_w4", "gemm_layoutA_w4",
           "fused_experts_compute_w4"]

_GROUPS = (32, 64, 128)
_EXACT_TOKENS, _EXACT_SLOTS = 16, 4     # tokens of a product, slots per expert, up to which the kernels do not round the weights
_LIMIT = 2 ** 31        # the C interface's sizes are 32-bit integers, and ctypes cuts off what is longer
_CODES = {torch.bfloat16: 0, torch.float16: 1}
_device_of_thread = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream


def _launch(device: int, call, *args) -> None:
    """``call(*args, stream)`` with the tensors' device current and its current stream."""
    if _device_of_thread() == device:
        status = call(*args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            status = call(*args, _stream_of(device))
    if status:
        check(status)


def _status(device: int, like: torch.Tensor) -> int:
    """Device address of the sticky status word of the current stream."""
    bufs = _SYNC_BUFFERS.get((device, _stream_of(device)))
    return _status_ptr(like) if bufs is None else bufs[1].data_ptr()


def _same_device(like: torch.Tensor, *named) -> None:
    for t, name in named:
        if t is not None:
            _chk(t.device == like.device, f"{name} must be on the same device as the activations")


def _fits(*sizes) -> None:
    _chk(max(sizes) < _LIMIT, "sizes of 2^31 and more are not supported")


def _parts(n: int, step: int):
    """(first row, rows) of the launches that take n rows in order, at most `step` at a time."""
    return [(i, min(step, n - i)) for i in range(0, n, step)]


def layoutA_w4(W: torch.Tensor) -> torch.Tensor:
    """Row-major packed nibbles ``[m, k/2]`` uint8 (low nibble = even k) -> ``[m/16, ceil(k/64), 32, 16]``; a 3-D
    ``[E, m, k/2]`` keeps its leading dimension.  m % 16 == 0, k % 32 == 0, k up to 2^28."""
    _cuda_contig(W, "W")
    _chk(W.dtype == torch.uint8, "W must be a uint8 tensor of packed nibbles")
    _chk(W.dim() in (2, 3), "W must be a 2D or 3D tensor")
    m, k = W.shape[-2], 2 * W.shape[-1]
    _chk(m % 16 == 0 and k % 32 == 0 and k > 0, "layoutA_w4 needs m % 16 == 0 and k % 32 == 0")
    _fits(k)
    out = torch.empty(W.shape[:-2] + (m // 16, (k + 63) // 64, 32, 16), dtype=torch.uint8, device=W.device)
    rows = m * (W.shape[0] if W.dim() == 3 else 1)
    _launch(W.get_device(), lib.mlk_layoutA_w4, W.data_ptr(), out.data_ptr(), rows, k, 0)
    return out


def layoutA_w4_inverse(A: torch.Tensor, k: int) -> torch.Tensor:
    """``[m/16, ceil(k/64), 32, 16]`` (or with a leading expert dimension) -> row-major packed nibbles ``[m, k/2]``."""
    _cuda_contig(A, "A")
    R, kc = _packed_dims(A, "A")
    _chk(k > 0 and k % 32 == 0 and (k + 63) // 64 == kc, "k does not match the packed weights")
    _fits(k)
    out = torch.empty(A.shape[:-4] + (R * 16, k // 2), dtype=torch.uint8, device=A.device)
    _launch(A.get_device(), lib.mlk_layoutA_w4, A.data_ptr(), out.data_ptr(), out.numel() // (k // 2), k, 1)
    return out


def layoutA_w4_groups(values: torch.Tensor) -> torch.Tensor:
    """Scales or zero points ``[m, k/group]`` -> ``[m/16, k/group, 8, 2]`` (entry (r, h) = row r + 8 h of 16); a 3-D input
    keeps its leading dimension.  Scales are bf16 / fp16, zero points uint8."""
    _cuda_contig(values, "values")
    _chk(values.dtype in (torch.bfloat16, torch.float16, torch.uint8), "values must be bfloat16, float16 (scales) or uint8 (zero points)")
    _chk(values.dim() in (2, 3), "values must be a 2D or 3D tensor")
    m, G = values.shape[-2:]
    _chk(m % 16 == 0 and G > 0, "layoutA_w4_groups needs m % 16 == 0 and at least one group")
    _fits(G)
    out = torch.empty(values.shape[:-2] + (m // 16, G, 8, 2), dtype=values.dtype, device=values.device)
    rows = m * (values.shape[0] if values.dim() == 3 else 1)
    _launch(values.get_device(), lib.mlk_layoutA_w4_groups, values.data_ptr(), out.data_ptr(), rows, G, values.element_size())
    return out


def _packed_dims(A: torch.Tensor, name: str):
    _chk(A.dtype == torch.uint8, f"{name} must be uint8 (packed by layoutA_w4)")
    _chk(A.dim() in (4, 5), f"{name} must be [m/16, ceil(k/64), 32, 16], or that behind an expert dimension")
    _chk(A.size(-2) == 32 and A.size(-1) == 16, f"{name}'s trailing dims must be (32, 16)")
    return A.size(-4), A.size(-3)


def _group(A, scales, zeros, x, k: int, name: str) -> int:
    """Group size told by the scales' shape, after checking all that belongs to one weight tensor against it.  The first
    test is the whole of it; what follows only finds the message (formatting it costs more than a small launch)."""
    a, s = A.shape, scales.shape
    d = x.get_device()
    lead = len(a) - 4
    if lead in (0, 1) and len(s) == lead + 4:
        G = s[lead + 1]
        if (A.get_device() == d and scales.get_device() == d and A.dtype is torch.uint8 and scales.dtype is x.dtype
                and A.is_contiguous() and scales.is_contiguous() and a[lead + 2] == 32 and a[lead + 3] == 16
                and s[lead + 2] == 8 and s[lead + 3] == 2 and s[:lead + 1] == a[:lead + 1] and a[lead + 1] == (k + 63) // 64
                and G > 0 and k % G == 0 and k // G in _GROUPS
                and (zeros is None or (zeros.get_device() == d and zeros.dtype is torch.uint8 and zeros.shape == s
                                       and zeros.is_contiguous()))):
            return k // G
    _cuda_contig(A, name)
    _cuda_contig(scales, f"{name} scales")
    R, kc = _packed_dims(A, name)
    lead = A.shape[:-4]
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
    raise RuntimeError(f"{name}: weights, scales and zeros do not belong together")


def gemm_layoutA_w4(A, scales, B, alpha: float = 1, beta: float = 0, zeros=None, bias=None, exact_weights: bool = False):
    """``C[n,m] = alpha * B W^T (+ bias)`` for any token count n (0 included), W in 4 bits: ``A`` from ``layoutA_w4``,
    ``scales`` / ``zeros`` from ``layoutA_w4_groups``, ``B[n,k]`` and C row-major.  Sums are held in fp32 and rounded once.
    ``beta`` is ignored, as by the other GEMMs.  Up to 16 tokens the weights' value is exact; larger calls multiply
    the value rounded to the activation type (what a dequantised checkpoint holds), so that a token's result may differ
    with the number of tokens in the call.  ``exact_weights=True`` keeps the value exact for any n, by launches of 16
    tokens, each of which reads the weights."""
    _chk(B.is_cuda, "B must be a CUDA tensor")
    _chk(B.is_contiguous(), "B must be contiguous")
    _chk(B.dim() == 2, "B must be a 2D tensor")
    code = _CODES.get(B.dtype)
    _chk(code is not None, "Unsupported data type")
    _chk(A.dim() == 4, "A must be [m/16, ceil(k/64), 32, 16]")
    n, k = B.shape
    group = _group(A, scales, zeros, B, k, "A")
    m = A.shape[0] * 16
    if m >= _LIMIT or n >= _LIMIT or k >= _LIMIT:
        _fits(m, n, k)
    if bias is not None:
        _same_device(B, (bias, "bias"))
        bias = _bias_ptr(bias, B, m)
    C = B.new_empty((n, m))
    d = B.get_device()
    for i, count in _parts(n, _EXACT_TOKENS) if exact_weights else ((0, n),):
        _launch(d, lib.mlk_gemm_layoutA_w4, A.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), group,
                B.data_ptr() + 2 * i * k, C.data_ptr() + 2 * i * m, m, count, k, code, alpha, bias, _status(d, B))
    return C


def gemv_layoutA_w4(A, scales, B, alpha: float = 1, beta: float = 0, zeros=None, bias=None):
    """``y[1,m] = alpha * W x (+ bias)``: ``gemm_layoutA_w4`` for one token ``B[1,k]``."""
    _chk(B.dim() == 2 and B.size(0) == 1, "B must be a vector")
    return gemm_layoutA_w4(A, scales, B, alpha, beta, zeros, bias)


def fused_experts_compute_w4(w1, w1_scales, w2, w2_scales, activations, topk_ids, topk_weights, w1_zeros=None, w2_zeros=None,
                             experts_map=None, out: Optional[torch.Tensor] = None,
                             out_dtype: Optional[torch.dtype] = None, exact_weights: bool = False) -> torch.Tensor:
    """``y[t] = sum_j topk_weights[t,j] * W2_e (silu(Wgate_e x_t) * (Wup_e x_t))``, ``e = topk_ids[t,j]``, expert weights in
    4 bits: ``w1 [E, 2I/16, ceil(H/64), 32, 16]`` (gate rows, then up rows) and ``w2 [E, H/16, ceil(I/64), 32, 16]`` from
    ``layoutA_w4``, scales and zero points from ``layoutA_w4_groups``; ``activations [T, H]`` bf16 / fp16, ``topk_ids``
    int32 ``[T, topk]``, ``topk_weights`` in the activations' type.  ``experts_map``: global -> local expert or -1, as in
    ``fused_experts_compute``; ids without an expert here contribute nothing.  ``out_dtype=torch.float32`` gives the
    un-rounded sums; ``out`` receives the result (every element is written).  A token's experts are added in
    slot order in fp32 with one rounding.  At most 1024 experts and 8257408 slots (T * topk).  Up to 4 slots (T * topk,
    those without an expert here included) per expert of ``w1`` the weights' value is exact; above that it is rounded to
    the activation type, as the activation between the two products always is, so that a token's result may differ with
    the number of tokens in the call.  ``exact_weights=True`` keeps the value exact for any T, by launches of as many
    tokens as that allows, each of which reads the weights of the experts that they pick."""
    x = activations
    _chk(x.is_cuda and x.is_contiguous(), "activations must be a contiguous CUDA tensor")
    _chk(x.dim() == 2, "activations must be [T, H]")
    code = _CODES.get(x.dtype)
    _chk(code is not None, "Unsupported data type")
    T, H = x.shape
    _chk(w1.dim() == 5 and w2.dim() == 5, "w1 and w2 must be [E, rows/16, ceil(k/64), 32, 16]")
    s1, s2 = w1.shape, w2.shape
    E, I = s1[0], s1[1] * 8
    _chk(s1[1] % 2 == 0 and s2[0] == E and s2[1] * 16 == H and E > 0, "w1 must hold [E, 2I, H] and w2 [E, H, I]")
    g1 = _group(w1, w1_scales, w1_zeros, x, H, "w1")
    g2 = _group(w2, w2_scales, w2_zeros, x, I, "w2")
    d = x.get_device()
    ids = topk_ids.shape
    _chk(topk_ids.get_device() == d and topk_ids.is_contiguous() and topk_ids.dtype is torch.int32 and len(ids) == 2 and
         ids[0] == T and ids[1] > 0, "topk_ids must be a contiguous int32 [T, topk] on the activations' device")
    _chk(topk_weights.get_device() == d and topk_weights.is_contiguous() and topk_weights.dtype is x.dtype and
         topk_weights.shape == ids, "topk_weights must be a contiguous [T, topk] in the activation data type and on its device")
    mp, ml = None, 0
    if experts_map is not None:
        _same_device(x, (experts_map, "experts_map"))
        mp, ml = _map_args(experts_map)
    topk = ids[1]
    if T >= _LIMIT or E >= _LIMIT or topk >= _LIMIT or H >= _LIMIT or I >= _LIMIT or ml >= _LIMIT:
        _fits(T, E, topk, H, I, ml)
    dtype = x.dtype if out_dtype is None else out_dtype
    _chk(dtype is x.dtype or dtype is torch.float32, "out_dtype must be the activation data type or torch.float32")
    if out is None:
        out = torch.empty_like(x) if dtype is x.dtype else x.new_empty((T, H), dtype=dtype)
    else:
        _chk(out.get_device() == d and out.is_contiguous() and out.shape == x.shape and out.dtype is dtype,
             "out must be a contiguous [T, H] in the result's data type on the activations' device")
    parts, most = ((0, T),), T
    if exact_weights:
        # a single token of up to 8 picks takes a path of its own, which does not round either
        _chk(topk <= max(_EXACT_SLOTS * E, 8), f"exact_weights: {topk} picks of {E} experts are more than {_EXACT_SLOTS} per expert")
        most = max(_EXACT_SLOTS * E // topk, 1)
        parts = _parts(T, most)
    nbytes = lib.mlk_experts_w4_workspace_bytes(min(T, most), E, topk, H, I)
    ws = x.new_empty((nbytes,), dtype=torch.uint8)
    for i, count in parts:
        _launch(d, lib.mlk_fused_experts_compute_w4, w1.data_ptr(), w1_scales.data_ptr(), _ptr(w1_zeros), g1, w2.data_ptr(),
                w2_scales.data_ptr(), _ptr(w2_zeros), g2, x.data_ptr() + 2 * i * H, count, E, topk, H, I,
                topk_ids.data_ptr() + 4 * i * topk, topk_weights.data_ptr() + 2 * i * topk,
                out.data_ptr() + out.element_size() * i * H, code, int(dtype is torch.float32), mp, ml, ws.data_ptr(), nbytes,
                _status(d, x))
    return out
