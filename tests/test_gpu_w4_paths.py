"""4-bit weights on the GPU: long k, many rows, kernel choices at their borders, layers as they are used, refusals."""
import pytest
import torch

from oracle import w4 as ow4
from tests.gpu_util import DT, randn, require_gpu
from tests.test_gpu_w4 import check, laid_out, mlk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [(16, 40960, 128, 16, "bf16"), (32, 65600, 32, 3, "fp16"), (16, 131072, 64, 1, "bf16"),
                                  (48, 40992, 32, 9, "bf16"), (128, 40960, 64, 20, "fp16")])
def test_long_k(case):
    """k that does not fit a CTA's shared memory at once (and the tcgen05 form of it)."""
    dev = require_gpu()
    m, k, group, n, dtype = case
    w = ow4.random_weights(m, k, group, DT[dtype], 1, True, scale=0.01)
    A, S, Z = laid_out(w, dev)
    x = randn((n, k), 2, 1.0, DT[dtype])
    want, bound = ow4.dense(*w, group, x, rounded_weights=n > 16)
    check(mlk().gemm_layoutA_w4(A, S, x.to(dev), zeros=Z), want, bound, case)


def test_weights_beyond_2_to_31_bytes():
    dev = require_gpu()
    m, k, group = 65568, 65536, 128
    g = torch.Generator(device=dev).manual_seed(1)
    rows = torch.randint(0, 256, (m, k // 2), generator=g, device=dev, dtype=torch.uint8)
    s = (0.01 * (0.5 + torch.rand(m, k // group, generator=g, device=dev))).to(torch.bfloat16)
    A, S = mlk().layoutA_w4(rows), mlk().layoutA_w4_groups(s)
    pick = torch.cat((torch.arange(0, 16), torch.arange(m // 2, m // 2 + 16), torch.arange(m - 16, m)))
    part = rows[pick.to(dev)].cpu()
    q = torch.stack((part & 15, part >> 4), -1).flatten(-2)
    del rows
    for n in (1, 20):
        x = randn((n, k), n, 1.0, torch.bfloat16)
        want, bound = ow4.dense(q, s[pick.to(dev)].cpu(), None, group, x, rounded_weights=n > 16)
        got = mlk().gemm_layoutA_w4(A, S, x.to(dev))
        check(got[:, pick.to(dev)], want, bound, n)


@pytest.mark.parametrize("case", [(2, 2, 128, 64, 100, 64, 32), (80, 8, 2048, 32, 50, 128, 32), (4, 1, 96, 160, 33, 32, 32),
                                  (3, 2, 256, 2176, 30, 64, 128), (5, 5, 64, 32, 4, 32, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_experts_at_the_borders_of_the_kernel_choice(case, dtype):
    """128-slot tiles, several row tiles per CTA, items of one slot more than a tile, rows that no 128-row tile divides."""
    dev = require_gpu()
    E, topk, H, I, T, g1, g2 = case
    dt = DT[dtype]
    w1 = ow4.random_weights(2 * I, H, g1, dt, 1, True, (E,))
    w2 = ow4.random_weights(H, I, g2, dt, 2, False, (E,))
    x = randn((T, H), 3, 1.0, dt)
    g = torch.Generator().manual_seed(4)
    ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32)
    p = torch.rand(T, topk, generator=g).to(dt)
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    want, bound = ow4.experts(w1, w2, g1, g2, x, ids, p, rounded_weights=True)
    got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), w1_zeros=a[2])
    check(got, want, bound, (case, dtype))


def test_all_tokens_on_one_expert():
    dev = require_gpu()
    E, H, I, T = 6, 128, 96, 150
    w1 = ow4.random_weights(2 * I, H, 128, torch.bfloat16, 1, False, (E,))
    w2 = ow4.random_weights(H, I, 32, torch.bfloat16, 2, True, (E,))
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    for n in (9, T):        # 1.5 slots per expert on average, all on one; and 25
        x = randn((n, H), 3, 1.0, torch.bfloat16)
        ids, p = torch.full((n, 1), 4, dtype=torch.int32), torch.ones(n, 1, dtype=torch.bfloat16)
        want, bound = ow4.experts(w1, w2, 128, 32, x, ids, p, rounded_weights=True)
        got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), w2_zeros=b[2])
        check(got, want, bound, n)


@pytest.mark.parametrize("n", [1, 8, 16, 40, 200])
def test_static_weights_option(n):
    dev = require_gpu()
    w = ow4.random_weights(272, 1152, 128, torch.bfloat16, 3, True)
    A, S, Z = laid_out(w, dev)
    x = randn((n, 1152), 1, 1.0, torch.bfloat16).to(dev)
    want = mlk().gemm_layoutA_w4(A, S, x, zeros=Z)
    torch.cuda.synchronize()
    mlk().set_static_weights(True)
    try:
        for _ in range(3):
            y = x * 2                      # the kernel in front writes what this one reads
            assert torch.equal(mlk().gemm_layoutA_w4(A, S, y, alpha=0.5, zeros=Z), want)
    finally:
        mlk().set_static_weights(False)
    mlk().set_pdl(False)
    try:
        assert torch.equal(mlk().gemm_layoutA_w4(A, S, x, zeros=Z), want)
    finally:
        mlk().set_pdl(True)
    assert mlk().kernel_status() == 0


@pytest.mark.parametrize("captured", [False, True])
def test_static_weights_in_a_chain(captured):
    """Experts, then products of every kind, each the input of the next, with the weights fetched ahead."""
    dev = require_gpu()
    E, topk, H, I, T = 8, 2, 256, 128, 300
    w1 = laid_out(ow4.random_weights(2 * I, H, 128, torch.bfloat16, 1, False, (E,)), dev)
    w2 = laid_out(ow4.random_weights(H, I, 64, torch.bfloat16, 2, True, (E,)), dev)
    d = laid_out(ow4.random_weights(H, H, 32, torch.bfloat16, 3, False), dev)
    g = torch.Generator().manual_seed(5)
    x = randn((T, H), 6, 1.0, torch.bfloat16).to(dev)
    ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32).to(dev)
    p = torch.rand(T, topk, generator=g).to(torch.bfloat16).to(dev)

    def chain():
        y = mlk().fused_experts_compute_w4(w1[0], w1[1], w2[0], w2[1], x, ids, p, w2_zeros=w2[2])
        for n in (T, 250, 100, 60, 20, 16, 8, 1):
            y = mlk().gemm_layoutA_w4(d[0], d[1], y[:n].contiguous(), alpha=0.25)
            y = mlk().gemm_layoutA_w4(d[0], d[1], y, alpha=0.25)
        return y

    want = chain()
    torch.cuda.synchronize()
    mlk().set_static_weights(True)
    try:
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = chain()
            for _ in range(5):
                graph.replay()
        else:
            for _ in range(5):
                got = chain()
        assert torch.equal(got, want) and mlk().kernel_status() == 0
    finally:
        mlk().set_static_weights(False)


@pytest.mark.parametrize("T", [1, 7, 90])
def test_two_graphs_at_once(T):
    """Two captured layers, replayed on two streams at the same time with inputs of their own."""
    dev = require_gpu()
    E, topk, H, I = 8, 2, 256, 128
    w1 = laid_out(ow4.random_weights(2 * I, H, 128, torch.bfloat16, 1, False, (E,)), dev)
    w2 = laid_out(ow4.random_weights(H, I, 64, torch.bfloat16, 2, True, (E,)), dev)
    g = torch.Generator().manual_seed(4)
    hold = []
    for k in range(2):
        x = randn((T, H), 3 + k, 1.0, torch.bfloat16).to(dev)
        ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32).to(dev)
        p = torch.rand(T, topk, generator=g).to(torch.bfloat16).to(dev)
        call = lambda x=x, ids=ids, p=p: mlk().fused_experts_compute_w4(w1[0], w1[1], w2[0], w2[1], x, ids, p, w2_zeros=w2[2])  # noqa: E731
        want = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
        hold.append((graph, y, want, torch.cuda.Stream(), call))       # call keeps the captured inputs alive
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, s, _ in hold:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, y, want, _, _ in hold:
        assert torch.equal(y, want)


@pytest.mark.parametrize("T", [1, 6, 48])
@pytest.mark.parametrize("score_func", ["softmax", "sigmoid"])
def test_a_layer_as_it_is_used(T, score_func):
    """Dense product -> router and 4-bit experts -> counts -> balance loss, weights quantised by the package's helper."""
    dev = require_gpu()
    m = mlk()
    from muxi_native_layout_kernels_b200 import utils
    from muxi_native_layout_kernels_b200.muxi_moe_planC import fused_moe_w4
    E, topk, H, I, K = 16, 4, 256, 128, 192
    g = torch.Generator().manual_seed(T)
    wd = (0.05 * torch.randn(H, K, generator=g)).to(torch.bfloat16)
    w1 = (0.05 * torch.randn(E, 2 * I, H, generator=g)).to(torch.bfloat16)
    w2 = (0.05 * torch.randn(E, H, I, generator=g)).to(torch.bfloat16)
    qd, q1, q2 = utils.quantize_w4(wd, 64, True), utils.quantize_w4(w1, 128), utils.quantize_w4(w2, 32, True)
    put = lambda q: (m.layoutA_w4(q[0].to(dev)), m.layoutA_w4_groups(q[1].to(dev)),  # noqa: E731
                     None if q[2] is None else m.layoutA_w4_groups(q[2].to(dev)))
    D, P, Q = put(qd), put(q1), put(q2)
    x = randn((T, K), 1, 1.0, torch.bfloat16)
    h = m.gemm_layoutA_w4(D[0], D[1], x.to(dev), zeros=D[2])
    unpack = lambda q: torch.stack((q & 15, q >> 4), -1).flatten(-2)  # noqa: E731
    want, bound = ow4.dense(unpack(qd[0]), qd[1], qd[2], 64, x, rounded_weights=T > 16)
    check(h, want, bound, T)
    logits = randn((T, E), 2, 1.0, torch.bfloat16).to(dev)
    y, ids, p = fused_moe_w4(h, P[0], Q[0], logits, topk, True, w1_scale=P[1], w2_scale=Q[1], w2_zeros=Q[2],
                             score_func=score_func, return_routing=True)
    want, bound = ow4.experts((unpack(q1[0]), q1[1], None), (unpack(q2[0]), q2[1], q2[2]), 128, 32, h.cpu(), ids.cpu(), p.cpu(),
                              rounded_weights=True)
    check(y, want, bound, (T, score_func))
    top = logits.float().topk(topk, -1)[0].sort(-1)[0]
    assert torch.equal(logits.float().gather(1, ids.long()).sort(-1)[0], top)
    loss, counts = m.router_balance_loss(logits, ids, int(score_func == "sigmoid"), 0.01)
    assert torch.equal(counts, m.expert_counts(ids, E)) and int(counts.sum()) == T * topk and float(loss) > 0
    again = fused_moe_w4(h, P[0], Q[0], logits, topk, True, w1_scale=P[1], w2_scale=Q[1], w2_zeros=Q[2], score_func=score_func)
    assert torch.equal(again, y)


def test_fused_moe_w4_refusals_and_empty_batch():
    dev = require_gpu()
    from muxi_native_layout_kernels_b200.muxi_moe_planC import fused_moe_w4
    w1 = laid_out(ow4.random_weights(64, 64, 32, torch.bfloat16, 1, lead=(4,)), dev)
    w2 = laid_out(ow4.random_weights(64, 32, 32, torch.bfloat16, 2, lead=(4,)), dev)
    x, l = torch.zeros(3, 64, dtype=torch.bfloat16, device=dev), torch.zeros(3, 4, dtype=torch.bfloat16, device=dev)
    kw = dict(w1_scale=w1[1], w2_scale=w2[1])
    with pytest.raises(ValueError):
        fused_moe_w4(x, w1[0], w2[0], l, 2, True)
    with pytest.raises(ValueError):
        fused_moe_w4(x, w1[0], w2[0], l, 2, True, score_func="relu", **kw)
    with pytest.raises(ValueError):
        fused_moe_w4(x, w1[0], w2[0], l, 2, True, num_expert_group=2, **kw)
    assert fused_moe_w4(x[:0], w1[0], w2[0], l[:0], 2, True, **kw).shape == (0, 64)


def test_refusals_on_the_device():
    dev = require_gpu()
    m = mlk()
    w = ow4.random_weights(32, 128, 64, torch.bfloat16, 1, True)
    A, S, Z = laid_out(w, dev)
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device=dev)
    ragged = torch.zeros(4 * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(4, 128)
    for a, kw in [((A, S, x.float()), {}), ((A, S, x.to(torch.float16)), {}), ((A, S.to(torch.float16), x), {}),
                  ((A, S, x[:, ::2]), {}), ((A, S, x[:, :64].contiguous()), {}), ((A[:1], S, x), {}), ((A, S[:, :1].contiguous(), x), dict(zeros=Z)),
                  ((A.to(torch.int8), S, x), {}), ((A, S, x), dict(zeros=Z.to(torch.int32))), ((A, S, x), dict(zeros=Z[:1])),
                  ((A, S, x), dict(bias=torch.zeros(31, dtype=torch.bfloat16, device=dev))),
                  ((A, S, x), dict(bias=torch.zeros(32, device=dev))), ((A, S, x.cpu()), {}), ((A.cpu(), S, x), {}), ((A, S, ragged), {}),
                  ((A, S, x[0]), {}), ((A, torch.zeros(2, 4, 8, 2, dtype=torch.bfloat16, device=dev), x), dict(zeros=Z))]:
        with pytest.raises(RuntimeError):
            m.gemm_layoutA_w4(*a, **kw)
    with pytest.raises(RuntimeError):
        m.gemv_layoutA_w4(A, S, x)
    with pytest.raises(RuntimeError):
        m.layoutA_w4(torch.zeros(24, 32, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError):
        m.layoutA_w4(torch.zeros(16, 24, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError):
        m.layoutA_w4_inverse(A, 192)
    with pytest.raises(RuntimeError):
        m.layoutA_w4_groups(torch.zeros(16, 2, device=dev))
    w1 = laid_out(ow4.random_weights(64, 64, 32, torch.bfloat16, 1, lead=(4,)), dev)
    w2 = laid_out(ow4.random_weights(64, 32, 32, torch.bfloat16, 2, lead=(4,)), dev)
    x = torch.zeros(3, 64, dtype=torch.bfloat16, device=dev)
    ids, p = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.zeros(3, 2, dtype=torch.bfloat16, device=dev)
    good = [w1[0], w1[1], w2[0], w2[1], x, ids, p]
    m.fused_experts_compute_w4(*good)
    for i, bad in [(0, w1[0][:2]), (0, w1[0][..., :8].contiguous()), (1, w1[1][:, :1].contiguous()), (2, w2[0][:, :2]), (4, x[:, :32].contiguous()), (4, x.float()), (5, ids.long()),
                   (5, ids[:2]), (6, p.float()), (6, p[:, :1]), (5, ids.cpu())]:
        with pytest.raises(RuntimeError):
            m.fused_experts_compute_w4(*(good[:i] + [bad] + good[i + 1:]))
    for kw in (dict(out=torch.zeros(3, 32, dtype=torch.bfloat16, device=dev)), dict(out=torch.zeros(3, 64, device=dev)),
               dict(out_dtype=torch.float16), dict(experts_map=torch.zeros(4, device=dev)), dict(w1_zeros=torch.zeros(1, device=dev)),
               dict(experts_map=torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            m.fused_experts_compute_w4(*good, **kw)
