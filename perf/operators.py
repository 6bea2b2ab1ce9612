"""Cases for timing and checking three operators: products with 4-bit weights (one matrix, and the experts of a
mixture layer) and the balance loss of a mixture layer's router.

`run` computes a case in plain torch operations in 32 bits, or with `own = True` through
``muxi_native_layout_kernels_b200``; `exact` is the definition in 64 bits.

4-bit weights: W[m, k] = (q[m, k] - z[m, k // group]) * s[m, k // group], q and z in 0..15 (z = 8 where none is given),
s in the activation's type.  A program that serves such a model holds the weights as the library lays them out once at
load time; `prepare` makes that form and the row-major one from the same numbers.
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one token against an attention-sized square matrix: the latency end of decoding
        _dense("w4 4096x4096 n1", 4096, 4096, 1, 128, "bf16"),
        # the widest matrix of the soft-FP8 grid at a small decode batch: the streaming end
        _dense("w4 28672x8192 n8", 28672, 8192, 8, 128, "bf16"),
        # a down projection with zero points and finer groups, fp16, a full decode tile
        _dense("w4 4096x14336 n16 fp16 z", 4096, 14336, 16, 64, "fp16", zeros=True),
        # a ragged row shard: rows and k that no 128-wide tile divides, bias, the finest groups
        _dense("w4 1040x2080 n5 odd", 1040, 2080, 5, 32, "bf16", bias=True),
        # the upper end of a decode batch
        _dense("w4 14336x4096 n61 z", 14336, 4096, 61, 32, "bf16", zeros=True),
        # a prompt chunk, compute bound
        _dense("w4 8192x8192 n500", 8192, 8192, 500, 128, "bf16"),
        # fine-grained experts at one token, a decode batch, and a prompt chunk with zero points
        _experts("experts fine T1", 128, 8, 2048, 768, 1, 128, "bf16"),
        _experts("experts fine T33", 128, 8, 2048, 768, 33, 128, "bf16"),
        _experts("experts fine T512 fp16 z", 128, 8, 2048, 768, 512, 64, "fp16", zeros=True),
        # eight large experts, a small decode batch
        _experts("experts wide T5", 8, 2, 4096, 14336, 5, 128, "bf16"),
        # router of eight experts on a short batch, logits as a 16-bit layer hands them over
        _balance("balance E8 T192", 192, 8, 2, "bf16", 0, 1, False, "direct"),
        # a training micro-batch of packed sequences with padding, fp32 router, gradients through autograd
        _balance("balance E128 T16384 seqs", 16384, 128, 8, "fp32", 1, 12, True, "autograd"),
    ]


def _dense(name, m, k, n, group, dtype, zeros=False, bias=False):
    return {"name": name, "op": "dense", "m": m, "k": k, "n": n, "group": group, "dtype": dtype, "zeros": zeros,
            "bias": bias}


def _experts(name, E, topk, H, I, T, group, dtype, zeros=False, ep=1):
    return {"name": name, "op": "experts", "E": E, "topk": topk, "H": H, "I": I, "T": T, "group": group,
            "dtype": dtype, "zeros": zeros, "ep": ep}


def _balance(name, T, E, topk, dtype, score_fun, seqs, padded, grad):
    return {"name": name, "op": "balance", "T": T, "E": E, "topk": topk, "dtype": dtype, "score_fun": score_fun,
            "seqs": seqs, "padded": padded, "grad": grad}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["dense", "dense", "experts", "experts", "balance"])
    if kind == "dense":
        group = rng.choice([32, 64, 128])
        n = _log(rng, 1, 512)
        m = 16 * _log(rng, 16, 1792)
        k = group * max(1, _log(rng, 512, 14336) // group)
        while m * k > 28672 * 8192 or m * k * n > 500 * 8192 * 8192:
            m = max(16, m // 32 * 16)
        c = _dense("", m, k, n, group, rng.choice(["bf16", "fp16"]), rng.random() < 0.5, rng.random() < 0.3)
    elif kind == "experts":
        group = rng.choice([32, 64, 128])
        E = rng.choice([4, 8, 16, 60, 64, 128])
        topk = min(E, rng.choice([1, 2, 4, 6, 8]))
        H = 128 * rng.randint(4, 32)
        I = 128 * rng.randint(2, 24)
        T = _log(rng, 1, 512)
        while E * H * I > 128 * 2048 * 1024:
            I = max(128, I // 256 * 128)
            H = max(512, H // 256 * 128)
        c = _experts("", E, topk, H, I, T, group, rng.choice(["bf16", "fp16"]), rng.random() < 0.5,
                     rng.choice([1, 1, 2]))
    else:
        T = _log(rng, 1, 16384)
        E = rng.choice([4, 8, 16, 60, 64, 128, 160, 256])
        c = _balance("", T, E, min(E, rng.choice([1, 2, 4, 6, 8])), rng.choice(["bf16", "fp16", "fp32"]),
                     rng.choice([0, 1]), min(T, rng.choice([1, 1, 3, 16])), rng.random() < 0.5,
                     rng.choice(["direct", "autograd", "none"]))
    del c["name"]
    return c


def work(case):
    if case["op"] == "dense":
        m, k, n = case["m"], case["k"], case["n"]
        groups = m * (k // case["group"])
        b = m * k // 2 + groups * (3 if case["zeros"] else 2) + 2 * n * (m + k) + (2 * m if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * m * k * n}
    if case["op"] == "experts":
        E, H, I, T = case["E"], case["H"], case["I"], case["T"]
        topk, local = case["topk"], case["T"] * case["topk"] / case["ep"]
        live = E * (1 - (1 - topk / (E * case["ep"])) ** T)          # experts that some token picks, on average
        groups = 3 * H * I / case["group"]
        per = 3 * H * I / 2 + groups * (3 if case["zeros"] else 2)
        return {"bytes": live * per + 4 * T * H + 6 * T * topk, "flops": 6 * local * H * I}
    T, E, size = case["T"], case["E"], 4 if case["dtype"] == "fp32" else 2
    passes = 1 if case["grad"] == "none" else 2                       # logits in, gradient out
    return {"bytes": T * E * size * passes + 4 * T * case["topk"] + T + 4 * E,
            "flops": T * E * (6 if case["grad"] == "none" else 12)}


# ------------------------------------------------------------------------------------------------- inputs

class State(dict):
    __getattr__ = dict.__getitem__


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weights(rows, k, group, dtype, zeros, g, experts=None):
    """Quantised weights of about N(0, 0.02): packed row-major nibbles (low nibble = even k), scales, zero points, and
    the same three as the library lays them out."""
    lead = () if experts is None else (experts,)
    G = k // group
    q = torch.empty(lead + (rows, k), dtype=torch.uint8, device="cuda")
    flat = q.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        part = flat[i:i + (1 << 27)]
        part.copy_(torch.empty(part.numel(), device="cuda").normal_(7.6, 2.6, generator=g).round_().clamp_(0, 15))
    s = (0.02 / 2.6 * (0.5 + torch.rand(lead + (rows, G), generator=g, device="cuda"))).to(dtype)
    z = torch.randint(5, 12, lead + (rows, G), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    packed = q[..., 0::2] | (q[..., 1::2] << 4)
    # library form: 16-row groups x 64 k, lane (r, t) holds rows r and r + 8; of its word j the nibble pair p
    # (bits 4p and 16 + 4p) is row r + 8 * (p % 2), k = 16 j + 4 t + 2 * (p // 2) and the next
    kc = -(-k // 64)
    pad = torch.nn.functional.pad(q, (0, kc * 64 - k)) if kc * 64 != k else q
    v = pad.view(-1, rows // 16, 2, 8, kc, 4, 4, 2, 2)                 # e, R, half, r, C, j, t, p//2, parity
    a = None
    for half in range(2):
        for hi in range(2):
            for odd in range(2):
                w = v[:, :, half, :, :, :, :, hi, odd].permute(0, 1, 3, 2, 5, 4).to(torch.int32)  # e, R, C, r, t, j
                w = w << (4 * (2 * hi + half) + 16 * odd)
                a = w if a is None else a | w
    a = a.contiguous().view(torch.uint8).view(lead + (rows // 16, kc, 32, 16))

    def pairs(x):
        return None if x is None else \
            x.view(lead + (rows // 16, 2, 8, G)).permute(*range(len(lead) + 1), -1, -2, -3).contiguous()

    return packed, s, z, a, pairs(s), pairs(z)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    if case["op"] == "dense":
        q, s, z, A, S, Z = _weights(case["m"], case["k"], case["group"], dt, case["zeros"], g)
        x = torch.randn(case["n"], case["k"], generator=g, device="cuda").to(dt)
        b = torch.randn(case["m"], generator=g, device="cuda").to(dt) if case["bias"] else None
        return State(op="dense", q=q, s=s, z=z, A=A, S=S, Z=Z, x=x, bias=b, group=case["group"], dt=dt)
    if case["op"] == "experts":
        E, H, I, T, topk = case["E"], case["H"], case["I"], case["T"], case["topk"]
        w1 = _weights(2 * I, H, case["group"], dt, case["zeros"], g, E)
        w2 = _weights(H, I, case["group"], dt, case["zeros"], g, E)
        x = torch.randn(T, H, generator=g, device="cuda").to(dt)
        total = E * case["ep"]
        # some experts are more popular than others
        logits = torch.randn(T, total, generator=g, device="cuda") + 0.5 * torch.randn(total, generator=g, device="cuda")
        p, ids = torch.softmax(logits, -1).topk(topk, -1)
        p = (p / p.sum(-1, keepdim=True)).to(dt)
        emap = None
        if case["ep"] > 1:           # this rank holds every ep-th expert
            emap = torch.full((total,), -1, dtype=torch.int32, device="cuda")
            emap[::case["ep"]] = torch.arange(E, dtype=torch.int32, device="cuda")
        local = ids if emap is None else emap[ids].long()
        load = torch.bincount(local[local >= 0].view(-1), minlength=E)
        return State(op="experts", w1=w1, w2=w2, x=x, ids=ids.to(torch.int32), p=p, emap=emap, E=E, H=H, I=I,
                     group=case["group"], most=max(1, int(load.max())), dt=dt)
    T, E, topk = case["T"], case["E"], case["topk"]
    logits = (1.5 * torch.randn(T, E, generator=g, device="cuda") + 0.7 * torch.randn(E, generator=g, device="cuda")).to(dt)
    ids = logits.float().topk(topk, -1)[1].to(torch.int32)
    r = random.Random(seed)
    cuts = sorted(r.randint(0, T) for _ in range(case["seqs"] - 1))
    cu = None
    if case["seqs"] > 1 or case["padded"]:
        # padded: the batch's last rows are behind the last sequence
        end = T - T // 16 if case["padded"] else T
        cu = torch.tensor([0] + [min(c, end) for c in cuts] + [end], dtype=torch.int32, device="cuda")
    mask = (torch.rand(T, generator=g, device="cuda") < 0.9) if case["padded"] else None
    return State(op="balance", logits=logits, ids=ids, mask=mask, cu=cu, E=E, score_fun=case["score_fun"],
                 grad=case["grad"], coef=0.01)


# ------------------------------------------------------------------------------------------------- one pass

def run(state):
    return _own(state) if own else _PLAIN[state.op](state)


def _own(st):
    import muxi_native_layout_kernels_b200 as mlk
    if st.op == "dense":
        if st.x.shape[0] == 1:
            return mlk.gemv_layoutA_w4(st.A, st.S, st.x, zeros=st.Z, bias=st.bias)
        return mlk.gemm_layoutA_w4(st.A, st.S, st.x, zeros=st.Z, bias=st.bias)
    if st.op == "experts":
        return mlk.fused_experts_compute_w4(st.w1[3], st.w1[4], st.w2[3], st.w2[4], st.x, st.ids, st.p,
                                            w1_zeros=st.w1[5], w2_zeros=st.w2[5], experts_map=st.emap)
    if st.grad == "autograd":
        x = st.logits.detach().requires_grad_()
        loss, counts = mlk.router_balance_loss(x, st.ids, st.score_fun, st.coef, token_mask=st.mask, cu_seqlens=st.cu)
        return loss.detach(), counts, torch.autograd.grad(loss, x)[0]
    if st.grad == "direct":
        return mlk.router_balance_loss(st.logits, st.ids, st.score_fun, st.coef, token_mask=st.mask, cu_seqlens=st.cu,
                                       return_grad=True)
    return mlk.router_balance_loss(st.logits, st.ids, st.score_fun, st.coef, token_mask=st.mask, cu_seqlens=st.cu)


def _dequant(packed, s, z, group):
    q = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float()
    q = q.unflatten(-1, (-1, group))
    q = q - (8.0 if z is None else z.float().unsqueeze(-1))
    return (q * s.float().unsqueeze(-1)).flatten(-2)


def _plain_dense(st):
    y = st.x.float() @ _dequant(st.q, st.s, st.z, st.group).t()
    if st.bias is not None:
        y = y + st.bias.float()
    return y.to(st.dt)


def _plain_experts(st):
    T, topk = st.ids.shape
    ids = st.ids.long() if st.emap is None else st.emap[st.ids.long()].long()
    if 2 * T * topk <= st.E:                                           # few slots: the weights of each slot's own expert
        e = ids.clamp_min(0).view(-1)
        pick = lambda w: [None if v is None else v[e] for v in w[:3]]  # noqa: E731
        x = st.x.float().repeat_interleave(topk, 0).unsqueeze(-1)
        h = (_dequant(*pick(st.w1), st.group) @ x).squeeze(-1)
        gate, up = h[:, :st.I], h[:, st.I:]
        y = (_dequant(*pick(st.w2), st.group) @ (gate / (1 + torch.exp(-gate)) * up).unsqueeze(-1)).squeeze(-1)
        y = y.view(T, topk, st.H) * (st.p.float() * (ids >= 0)).unsqueeze(-1)
        return y.sum(1).to(st.dt)
    flat = torch.where(ids < 0, st.E, ids).view(-1)                    # slots of other ranks sort behind the last expert
    order = flat.argsort(stable=True)
    load = torch.zeros(st.E + 1, dtype=torch.long, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    first = load.cumsum(0) - load
    e = flat[order]
    rank = torch.arange(flat.numel(), device=flat.device) - first[e]
    rows = st.E * st.most
    place = torch.where(e < st.E, e * st.most + rank, rows)            # one spare row takes what is not computed here
    x = torch.zeros(rows + 1, st.H, device=flat.device)
    x[place] = st.x.float()[order // topk]
    h = torch.bmm(x[:rows].view(st.E, st.most, st.H), _dequant(*st.w1[:3], st.group).transpose(1, 2))
    gate, up = h[..., :st.I], h[..., st.I:]
    y = torch.bmm(gate / (1 + torch.exp(-gate)) * up, _dequant(*st.w2[:3], st.group).transpose(1, 2))
    y = torch.cat((y.reshape(rows, st.H), torch.zeros(1, st.H, device=y.device)))
    back = torch.empty_like(place)
    back[order] = place
    return (y[back].view(T, topk, st.H) * st.p.float().unsqueeze(-1)).sum(1).to(st.dt)


def _segments(st):
    """Sequence of every token (-1: in none, or masked out) and the number of sequences."""
    T = st.logits.shape[0]
    at = torch.arange(T, device=st.logits.device)
    if st.cu is None:
        seq, B = torch.zeros_like(at), 1
    else:
        B = st.cu.numel() - 1
        seq = torch.searchsorted(st.cu[1:].long().contiguous(), at, right=True)
        seq = torch.where((at >= st.cu[0]) & (seq < B), seq, -1)
    return (seq if st.mask is None else torch.where(st.mask, seq, -1)), B


def _plain_balance(st):
    T, E = st.logits.shape
    topk = st.ids.shape[1]
    seq, B = _segments(st)
    live = (seq >= 0).float()
    row = torch.where(seq >= 0, seq, B)                                # row B takes what no sequence counts
    x = st.logits.float()
    if st.score_fun == 0:
        a = torch.exp(x - x.max(-1, keepdim=True)[0])
        p = a / a.sum(-1, keepdim=True)
    else:
        a = 1 / (1 + torch.exp(-x))
        p = a / a.sum(-1, keepdim=True)
    n = torch.zeros(B + 1, device=x.device).index_add_(0, row, live)[:B]
    counts = torch.zeros((B + 1) * E, dtype=torch.int32, device=x.device)
    counts.scatter_add_(0, (row.unsqueeze(1) * E + st.ids.long()).view(-1), torch.ones_like(st.ids).view(-1))
    counts = counts.view(B + 1, E)[:B]
    P = torch.zeros(B + 1, E, dtype=torch.float64, device=x.device).index_add_(0, row, p.double())[:B].float()
    scale = (st.coef * E / (topk * B)) / (n * n).clamp_min(1)          # a mean over the sequences given
    loss = (scale.unsqueeze(1) * counts.float() * P).sum()
    total = counts.sum(0, dtype=torch.int32)
    if st.grad == "none":
        return loss, total
    c = torch.cat((scale.unsqueeze(1) * counts.float(), torch.zeros(1, E, device=x.device)))[row]
    d = p * (c - (p * c).sum(-1, keepdim=True))
    if st.score_fun == 1:
        d = d * (1 - a)
    return loss, total, d.to(st.logits.dtype)


_PLAIN = {"dense": _plain_dense, "experts": _plain_experts, "balance": _plain_balance}


# ------------------------------------------------------------------------------------------------- 64 bits

def _w64(packed, s, z, group):
    """Rows of one weight matrix in 64 bits."""
    w = torch.empty(packed.shape[0], packed.shape[1] * 2, dtype=torch.float64, device=packed.device)
    w[:, 0::2] = (packed & 15).double()
    w[:, 1::2] = (packed >> 4).double()
    z = torch.full_like(s, 8.0).double() if z is None else z.double()
    return (w - z.repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dense":
        y = torch.empty(st.x.shape[0], case["m"], dtype=torch.float64, device="cuda")
        for i in range(0, case["m"], 2048):
            rows = slice(i, i + 2048)
            y[:, rows] = st.x.double() @ _w64(st.q[rows], st.s[rows], None if st.z is None else st.z[rows], st.group).t()
        return y if st.bias is None else y + st.bias.double()
    if case["op"] == "experts":
        y = torch.zeros(case["T"], st.H, dtype=torch.float64, device="cuda")
        one = lambda w, e: _w64(w[0][e], w[1][e], None if w[2] is None else w[2][e], st.group)  # noqa: E731
        for e in range(st.E):
            t, j = torch.nonzero(st.ids == e * case["ep"], as_tuple=True)
            if t.numel():
                h = st.x[t].double() @ one(st.w1, e).t()
                h = torch.nn.functional.silu(h[:, :st.I]) * h[:, st.I:]
                y.index_add_(0, t, (h @ one(st.w2, e).t()) * st.p[t, j].double().unsqueeze(1))
        return y
    x = st.logits.double().requires_grad_()
    p = torch.softmax(x, 1) if case["score_fun"] == 0 else torch.sigmoid(x) / torch.sigmoid(x).sum(1, keepdim=True)
    cu = [0, case["T"]] if st.cu is None else st.cu.tolist()
    mask = torch.ones(case["T"], dtype=torch.bool, device="cuda") if st.mask is None else st.mask
    parts, total = [], torch.zeros(case["E"], dtype=torch.int64, device="cuda")
    for a, b in zip(cu, cu[1:]):
        keep = mask[a:b]
        n = int(keep.sum())
        if n:
            counts = torch.bincount(st.ids[a:b][keep].long().view(-1), minlength=case["E"])
            total += counts
            parts.append(case["E"] / (case["topk"] * n) * (counts.double() * p[a:b][keep].mean(0)).sum())
    loss = st.coef / (len(cu) - 1) * torch.stack(parts).sum() if parts else x.sum() * 0
    out = (loss.detach(), None)
    return out if case["grad"] == "none" else out + (torch.autograd.grad(loss, x)[0],)
