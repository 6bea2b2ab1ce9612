"""4-bit weights with group scales, restated on the CPU in 64 bits: quantised values, packed layouts, dense products and
the experts of a mixture layer, each with a bound on what 32-bit sums and 16-bit roundings may cost."""
from __future__ import annotations

import torch

U32 = 2.0 ** -22        # one fp32 addition, a truncating one (tensor cores) included, with a factor of two to spare


def random_weights(m, k, group, dtype, seed, zeros=False, lead=(), scale=0.05):
    """q [.., m, k] in 0..15, s [.., m, k/group] in `dtype`, z like s in uint8 or None."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, lead + (m, k), generator=g, dtype=torch.uint8)
    s = (scale * (0.25 + torch.rand(lead + (m, k // group), generator=g))).to(dtype)
    z = torch.randint(0, 16, lead + (m, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


def pack_rows(q):
    """Row-major nibbles, low nibble = even k."""
    return q[..., 0::2] | (q[..., 1::2] << 4)


def pack_blocks(q):
    """[m/16, ceil(k/64), 32, 16] by the definition, one nibble at a time in numpy-sized steps."""
    *lead, m, k = q.shape
    kc = -(-k // 64)
    out = torch.zeros(*lead, m // 16, kc, 32, 4, dtype=torch.int64)
    full = torch.zeros(*lead, m, kc * 64, dtype=torch.int64)
    full[..., :k] = q
    for lane in range(32):
        r, t = lane // 4, lane % 4
        for j in range(4):
            for p in range(4):
                for odd in range(2):
                    row, kk = r + 8 * (p & 1), 16 * j + 4 * t + 2 * (p >> 1) + odd
                    out[..., lane, j] |= full[..., row::16, kk::64] << (4 * p + 16 * odd)
    b = torch.stack([(out >> (8 * i)) & 255 for i in range(4)], -1)
    return b.to(torch.uint8).flatten(-2)


def pair_order(v):
    """[.., m, G] -> [.., m/16, G, 8, 2], entry (r, h) = row r + 8 h of 16."""
    *lead, m, G = v.shape
    out = torch.empty(*lead, m // 16, G, 8, 2, dtype=v.dtype)
    for r in range(8):
        for h in range(2):
            out[..., r, h] = v[..., r + 8 * h::16, :]
    return out


def dequant(q, s, z, group):
    zz = torch.full_like(s, 8.0, dtype=torch.float64) if z is None else z.double()
    return (q.double() - zz.repeat_interleave(group, -1)) * s.double().repeat_interleave(group, -1)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def dense(q, s, z, group, x, alpha=1.0, bias=None, rounded_weights=False):
    """(y, bound): the product in 64 bits and how far a kernel may be from it.

    The bound: fp32 sums of k products taken 16 at a time, at most k/64/8 blocks per warp and 16 more partial sums; each
    weight off by half a step of the activation type where it is rounded; the result off by half a step (and by half of
    the type's smallest number where it is subnormal)."""
    w = dequant(q, s, z, group)
    y = alpha * (x.double() @ w.t())
    mag = abs(alpha) * (x.double().abs() @ w.abs().t())
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    u = half_step(x.dtype)
    steps = w.shape[1] // 16 + 32 if rounded_weights else 8 + w.shape[1] // 512 + 16
    off = mag * (steps * U32 + (u if rounded_weights else 0.0))
    return y, off + (y.abs() + off) * u + torch.finfo(x.dtype).smallest_normal * u


def experts(w1, w2, group1, group2, x, ids, p, experts_map=None, rounded_weights=False, out_fp32=False):
    """(y, bound) for the experts' sum; w1 / w2 = (q, s, z) with a leading expert dimension."""
    u = half_step(x.dtype)
    uw = u if rounded_weights else 0.0
    E, H = w1[0].shape[0], x.shape[1]
    I = w2[0].shape[-1]
    y = torch.zeros(x.shape[0], H, dtype=torch.float64)
    off = torch.zeros_like(y)
    one = lambda w, e, g: dequant(w[0][e], w[1][e], None if w[2] is None else w[2][e], g)  # noqa: E731
    acc1, acc2 = (H // 16 + 32) * U32, (I // 16 + 32) * U32
    for e in range(E):
        a, b = one(w1, e, group1), one(w2, e, group2)
        for t in range(x.shape[0]):
            for j in range(ids.shape[1]):
                i = int(ids[t, j])
                if experts_map is not None:
                    i = int(experts_map[i]) if 0 <= i < experts_map.numel() else -1
                if i != e:
                    continue
                xt, pt = x[t].double(), float(p[t, j])
                gu = a @ xt
                d = (a.abs() @ xt.abs()) * (uw + acc1)
                gate, up, dg, du = gu[:I], gu[I:], d[:I], d[I:]
                silu = gate * torch.sigmoid(gate)
                h = silu * up
                # |silu'| <= 1.1; the exponential and the division of the kernel: 2^-20 of the value
                dh = 1.1 * dg * (up.abs() + du) + silu.abs() * du + h.abs() * 2.0 ** -20
                dh = dh + (h.abs() + dh) * u + torch.finfo(x.dtype).smallest_normal * u
                y[t] += pt * (b @ h)
                off[t] += abs(pt) * (b.abs() @ dh + (b.abs() @ (h.abs() + dh)) * (uw + acc2))
    off = off + y.abs() * (64 * U32)
    return y, off if out_fp32 else off + (y.abs() + off) * u + torch.finfo(x.dtype).smallest_normal * u
