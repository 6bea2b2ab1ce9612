"""Torch-level helpers the reference package exposes next to its kernels (muxi_layout_kernels/utils.py).

``fused_moe`` is the dense, per-expert torch formulation of the MoE layer that the reference's tests compare the
fused kernels with (utils.py:131-244); ``scale_tensor`` / ``scale_whole_tensor`` expand 128x128 block scales
(utils.py:7-25).  ``quantize_w4`` / ``dequantize_w4`` make and undo 4-bit weights with group scales (no counterpart in the
reference).  None of this is used by the CUDA path of this package; it exists so that code written against
the reference package (its tests, its benchmarks) keeps importing and running.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F

_BLOCK = 128


def scale_tensor(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """``weight[m,k]`` times the per-128x128-block factor ``scale[ceil(m/128), ceil(k/128)]``, in weight's dtype."""
    m, k = weight.shape
    full = scale.repeat_interleave(_BLOCK, dim=0)[:m].repeat_interleave(_BLOCK, dim=1)[:, :k]
    # the reference multiplies block by block with a 0-dim fp32 factor: fp32 product, one rounding
    return (weight.to(torch.float32) * full.to(torch.float32)).to(weight.dtype)


def scale_whole_tensor(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Per-expert ``scale_tensor`` of ``weight[E,m,k]`` after converting it to bf16."""
    w = weight.to(torch.bfloat16)
    return torch.stack([scale_tensor(w[e], scale[e]) for e in range(w.shape[0])])


def quantize_w4(weight: torch.Tensor, group_size: int = 128, zero_points: bool = False):
    """``weight[..., m, k]`` to 4 bits with group scales, round to nearest: ``(qweight, scales, zeros)`` with ``qweight``
    uint8 ``[..., m, k/2]`` (low nibble = even k), ``scales [..., m, k/group_size]`` in weight's dtype and ``zeros`` uint8 or
    None.  Without zero points the values are symmetric around 8 (scale = largest magnitude / 7); with them the range of the
    group, widened to hold 0, is mapped to 0..15.  A group of zeros gets the scale 1."""
    *lead, m, k = weight.shape
    if k % group_size != 0 or group_size not in (32, 64, 128):
        raise ValueError("groups of 32, 64 or 128 that divide k")
    w = weight.to(torch.float32).reshape(*lead, m, k // group_size, group_size)
    if zero_points:
        lo, hi = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
        s = (hi - lo) / 15
    else:
        s = w.abs().amax(-1) / 7
    s = s.to(weight.dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    f = s.to(torch.float32)
    z = torch.round(-lo / f).clamp(0, 15) if zero_points else torch.full_like(f, 8.0)
    q = torch.round(w / f.unsqueeze(-1) + z.unsqueeze(-1)).clamp(0, 15).to(torch.uint8).reshape(*lead, m, k)
    return q[..., 0::2] | (q[..., 1::2] << 4), s, z.to(torch.uint8) if zero_points else None


def dequantize_w4(qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[..., m, k]`` in fp32 from what ``quantize_w4`` returns: ``(q - z) * s``, z = 8 without zero points."""
    q = torch.stack((qweight & 15, qweight >> 4), -1).flatten(-2).to(torch.float32)
    group = q.shape[-1] // scales.shape[-1]
    z = 8.0 if zeros is None else zeros.to(torch.float32).repeat_interleave(group, -1)
    return (q - z) * scales.to(torch.float32).repeat_interleave(group, -1)


def _route(gating_output, topk, num_expert_group, topk_group, renormalize, bias, score_func, dtype):
    if score_func == "softmax":
        scores = torch.softmax(gating_output, dim=-1, dtype=dtype)
    elif score_func == "sigmoid":
        scores = torch.sigmoid(gating_output)
    else:
        raise ValueError("Unsupported scoring function")
    sel = scores if bias is None else scores + bias.unsqueeze(0)
    T = sel.shape[0]
    grouped = sel.view(T, num_expert_group, -1)
    group_scores = grouped.max(dim=-1).values if bias is None else grouped.topk(2, dim=-1)[0].sum(dim=-1)
    keep = torch.topk(group_scores, k=topk_group, dim=-1, sorted=False)[1]
    gmask = torch.zeros_like(group_scores).scatter_(1, keep, 1)
    emask = gmask.unsqueeze(-1).expand(T, num_expert_group, sel.shape[-1] // num_expert_group).reshape(T, -1)
    masked = sel.masked_fill(~emask.bool(), 0.0)
    ids = torch.topk(masked, k=topk, dim=-1, sorted=False)[1]
    weights = scores.gather(1, ids)     # un-biased scores are the routing weights
    if renormalize:
        weights = weights / weights.sum(dim=-1, keepdim=True)
    return ids, weights.to(dtype)


def fused_moe(
    hidden_states: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    gating_output: torch.Tensor,
    topk: int,
    num_expert_group: int = 0,
    topk_group: int = 1,
    global_num_experts: int = 1,
    expert_map: Optional[torch.Tensor] = None,
    renormalize: bool = False,
    e_score_correction_bias: Optional[torch.Tensor] = None,
    score_func: str = "softmax",
) -> torch.Tensor:
    """Dense-loop MoE on *un-permuted* weights ``w1 [E,2I,H]`` (gate rows then up rows) and ``w2 [E,H,I]``.
    Every expert processes every token; tokens not routed to it get weight 0.  All arithmetic runs in the dtype
    of ``hidden_states``, as in the reference."""
    orig_shape = hidden_states.shape
    H = hidden_states.shape[-1]
    dtype = hidden_states.dtype
    x = hidden_states.reshape(-1, H)
    logits = gating_output.reshape(x.shape[0], global_num_experts)
    groups = num_expert_group if num_expert_group else 1
    ids, weights = _route(logits, topk, groups, topk_group, renormalize, e_score_correction_bias, score_func, dtype)
    if expert_map is not None:
        ids = expert_map[ids]
    I = w2.shape[-1]
    out = None
    for e in range(w1.shape[0]):
        w_e = (weights * (ids == e)).sum(dim=-1, keepdim=True)
        h = F.linear(x, w1[e])
        h = h[:, I:] * F.silu(h[:, :I])
        contrib = F.linear(h, w2[e]) * w_e
        out = contrib if out is None else out + contrib
    return out.view(orig_shape)
