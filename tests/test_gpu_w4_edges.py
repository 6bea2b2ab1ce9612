"""4-bit weights: a single token with any number of picks, weights that stay exact, the layer's other arguments, first calls
inside a capture."""
import pytest
import torch

from oracle import w4 as ow4
from tests.gpu_util import DT, randn, require_gpu
from tests.test_gpu_w4 import check, laid_out, mlk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("foreign", [False, True])
@pytest.mark.parametrize("topk", [1, 2, 5, 6, 7, 8, 9, 10, 12])
def test_single_token_with_any_number_of_picks(topk, foreign, dtype):
    """Clusters of every size up to 8, no cluster at 1, and the general path above 8; with `foreign` the first pick has no
    expert here, and at one pick nothing is left."""
    dev = require_gpu()
    E, H, I, dt = 12, 160, 96, DT[dtype]
    w1 = ow4.random_weights(2 * I, H, 32, dt, 1, True, (E,))
    w2 = ow4.random_weights(H, I, 32, dt, 2, False, (E,))
    x = randn((1, H), 3, 1.0, dt)
    g = torch.Generator().manual_seed(topk)
    ids = torch.rand(1, E, generator=g).topk(topk, -1)[1].to(torch.int32)
    if foreign:
        ids[0, 0] = E + 3
    p = torch.rand(1, topk, generator=g).to(dt)
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    for f32 in (False, True):
        want, bound = ow4.experts(w1, w2, 32, 32, x, ids, p, out_fp32=f32)
        out = torch.full((1, H), float("nan"), dtype=torch.float32 if f32 else dt, device=dev)
        got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), w1_zeros=a[2], out=out,
                                             out_dtype=torch.float32 if f32 else None)
        assert got is out
        check(got, want, bound + 1e-30, (topk, foreign, dtype, f32))
        again = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), w1_zeros=a[2],
                                               out_dtype=torch.float32 if f32 else None)
        assert torch.equal(got, again)


def worst_rounded(dtype):
    """(d, s): the weight d * s, d in 1..7, that a rounding to `dtype` moves most, relative to itself."""
    best = (0.0, 1, 1.0)
    steps = round(1 / torch.finfo(dtype).eps)
    for d in range(1, 8):
        for i in range(steps):
            s = 1.0 + i / steps
            w = torch.tensor(d * s, dtype=torch.float64)
            off = float((w.to(dtype).double() - w) / w)
            if abs(off) > abs(best[0]):
                best = (off, d, s)
    return best


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [(8, 2, 1), (8, 8, 1), (8, 2, 9), (8, 2, 16), (16, 12, 1)])
def test_weights_are_exact_up_to_four_slots_per_expert(case, dtype):
    """Every weight is the same number, one that a rounding to 16 bits would move far, always the same way: the sums of
    the exact weights are told from those of rounded ones, which lie outside the bound."""
    dev = require_gpu()
    E, topk, T = case
    H, I, dt = 128, 64, DT[dtype]
    off, d, s = worst_rounded(dt)
    full = lambda m, k, scale: (torch.full((E, m, k), 8 + d, dtype=torch.uint8),  # noqa: E731
                                torch.full((E, m, k // 32), s * scale, dtype=dt), None)
    w1, w2 = full(2 * I, H, 2.0 ** -6), full(H, I, 2.0 ** -6)
    x = torch.ones(T, H, dtype=dt)
    g = torch.Generator().manual_seed(1)
    ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32)
    p = torch.ones(T, topk, dtype=dt)
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    want, bound = ow4.experts(w1, w2, 32, 32, x, ids, p, out_fp32=True)
    gate = H * d * s / 64
    h = lambda e: (gate * (1 + e)) ** 2 / (1 + torch.exp(torch.tensor(-gate * (1 + e), dtype=torch.float64)))  # noqa: E731
    rounded = topk * I * d * s / 64 * (1 + off) * float(h(off))
    assert abs(rounded - float(want[0, 0])) > 1.5 * float(bound[0, 0])       # a kernel that rounds would be seen
    got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), out_dtype=torch.float32)
    check(got, want, bound, (case, dtype))


ROUTES = [dict(), dict(use_grouped_topk=True, num_expert_group=4, topk_group=2), dict(score_func="sigmoid", bias=True),
          dict(score_func="sigmoid", bias=True, use_grouped_topk=True, num_expert_group=4, topk_group=2), dict(gate=True),
          dict(gate=True, score_func="sigmoid", bias=True, use_grouped_topk=True, num_expert_group=2, topk_group=1)]


@pytest.mark.parametrize("T", [1, 5, 60])
@pytest.mark.parametrize("mapped", [False, True])
@pytest.mark.parametrize("route", range(len(ROUTES)))
def test_layer_arguments(route, mapped, T):
    """Grouped picks, a bias, the fused gate product, an experts map in 64 bits, a given result tensor, fp32 sums."""
    dev = require_gpu()
    m = mlk()
    from muxi_native_layout_kernels_b200.muxi_moe_planC import fused_moe_w4
    kw = dict(ROUTES[route])
    bias, gate = kw.pop("bias", False), kw.pop("gate", False)
    total, topk, H, I, dt = 16, 4, 128, 64, torch.bfloat16
    E = 8 if mapped else total
    w1, w2 = ow4.random_weights(2 * I, H, 64, dt, 1, False, (E,)), ow4.random_weights(H, I, 64, dt, 2, True, (E,))
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    x = randn((T, H), 3, 1.0, dt).to(dev)
    logits = randn((T, total), 4, 1.0, dt).to(dev)
    G = randn((total, H), 5, 0.2, dt).to(dev) if gate else None
    B = randn((total,), 6, 0.1, dt).to(dev) if bias else None
    emap = None
    if mapped:
        emap = torch.full((total,), -1, dtype=torch.int64)
        emap[::2] = torch.arange(E)
    ids, p = torch.empty(T, topk, dtype=torch.int32, device=dev), torch.empty(T, topk, dtype=dt, device=dev)
    fun, ng, kg = int(kw.get("score_func") == "sigmoid"), kw.get("num_expert_group") or 1, kw.get("topk_group") or 1
    if gate:
        m.fused_router_gemm_gate(x, G, fun, ng, kg, ids, p, topk, B, renormalize=True)
    else:
        m.fused_routing_gate(logits, fun, T, H, ng, kg, ids, p, topk, B, renormalize=True)
    for f32 in (False, True):
        out = torch.full((T, H), float("nan"), dtype=torch.float32 if f32 else dt, device=dev)
        y, got_ids, got_p = fused_moe_w4(x, a[0], b[0], None if gate else logits, topk, True, w1_scale=a[1], w2_scale=b[1],
                                         w2_zeros=b[2], gating_bias=B, experts_map=None if emap is None else emap.to(dev),
                                         gate_weight=G, out=out, out_dtype=torch.float32 if f32 else None, return_routing=True,
                                         **kw)
        assert y is out and torch.equal(got_ids, ids) and torch.equal(got_p, p)
        want, bound = ow4.experts(w1, w2, 64, 64, x.cpu(), ids.cpu(), p.cpu(), emap, rounded_weights=T * topk > 4 * E, out_fp32=f32)
        check(y, want, bound + 1e-30, (route, mapped, T, f32))


@pytest.mark.parametrize("n", [1, 11, 23, 70, 300])
def test_first_call_of_a_shape_inside_a_capture(n):
    """Nothing of the shape has run before: choosing a kernel and preparing it needs nothing that a capture forbids."""
    dev = require_gpu()
    m, k, E, topk, I = 16 * (31 + n % 7), 32 * (11 + n % 5), 7, 3, 32 * (1 + n % 3)
    w = laid_out(ow4.random_weights(m, k, 32, torch.float16, n, True), dev)
    w1 = laid_out(ow4.random_weights(2 * I, k, 32, torch.float16, 1, True, (E,)), dev)
    w2 = laid_out(ow4.random_weights(k, I, 32, torch.float16, 2, True, (E,)), dev)
    x = randn((n, k), 3, 1.0, torch.float16).to(dev)
    ids = torch.rand(n, E, generator=torch.Generator().manual_seed(n)).topk(topk, -1)[1].to(torch.int32).to(dev)
    p = torch.full((n, topk), 0.25, dtype=torch.float16, device=dev)

    def both():
        return (mlk().gemm_layoutA_w4(w[0], w[1], x, zeros=w[2]),
                mlk().fused_experts_compute_w4(w1[0], w1[1], w2[0], w2[1], x, ids, p, w1_zeros=w1[2], w2_zeros=w2[2]))

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(2):
        graph.replay()
    want = both()
    assert all(torch.equal(u, v) for u, v in zip(got, want))


@pytest.mark.parametrize("n", [1, 9, 61, 300])
def test_result_over_its_own_input(n):
    """`out` may be the activations: they are read before the result is written."""
    dev = require_gpu()
    E, topk, H, I = 8, 2, 128, 96
    a = laid_out(ow4.random_weights(2 * I, H, 128, torch.bfloat16, 1, False, (E,)), dev)
    b = laid_out(ow4.random_weights(H, I, 32, torch.bfloat16, 2, False, (E,)), dev)
    x = randn((n, H), 3, 1.0, torch.bfloat16).to(dev)
    ids = torch.rand(n, E, generator=torch.Generator().manual_seed(n)).topk(topk, -1)[1].to(torch.int32).to(dev)
    p = torch.full((n, topk), 0.5, dtype=torch.bfloat16, device=dev)
    want = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x, ids, p)
    got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x, ids, p, out=x)
    assert got is x and torch.equal(got, want)


def test_largest_number_of_slots():
    """The most slots there are, over the most experts: every work item of a launch is used.  A token's result does not depend
    on its place, so a part of the tokens alone, in tiles of the same size, gives the same bits."""
    dev = require_gpu()
    E, topk, H, I = 1024, 8, 32, 32
    T = (65535 - 1024) * 128 // topk
    a = laid_out(ow4.random_weights(2 * I, H, 32, torch.bfloat16, 1, False, (E,)), dev)
    b = laid_out(ow4.random_weights(H, I, 32, torch.bfloat16, 2, True, (E,)), dev)
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(T, H, generator=g, device=dev).to(torch.bfloat16)
    ids = torch.randint(0, E, (T, topk), generator=g, device=dev, dtype=torch.int32)
    p = torch.rand(T, topk, generator=g, device=dev).to(torch.bfloat16)
    call = lambda rows: mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x[rows].contiguous(), ids[rows].contiguous(),  # noqa: E731
                                                       p[rows].contiguous(), w2_zeros=b[2])
    got = call(slice(0, T))
    for first in (0, T // 2, T - 20000):
        rows = slice(first, first + 20000)
        assert torch.equal(got[rows], call(rows))
    one_more = torch.zeros(T + 1, H, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="slots"):
        mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], one_more, torch.zeros(T + 1, topk, dtype=torch.int32, device=dev),
                                       torch.zeros(T + 1, topk, dtype=torch.bfloat16, device=dev), w2_zeros=b[2])
    assert mlk().kernel_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [0, 1, 16, 17, 32, 45, 130])
def test_products_with_exact_weights_of_any_token_count(n, dtype):
    """The weights of the test above: the rounded product lies outside the bound of the exact one, as the default shows."""
    dev = require_gpu()
    m, k, dt = 48, 160, DT[dtype]
    off, d, s = worst_rounded(dt)
    w = (torch.full((m, k), 8 + d, dtype=torch.uint8), torch.full((m, k // 32), s / 64, dtype=dt), None)
    A, S, _ = laid_out(w, dev)
    x, b = torch.ones(n, k, dtype=dt), randn((m,), 2, 1.0, dt)
    x[:, 1:] = randn((n, k - 1), 3, 1.0, dt).abs()
    want, bound = ow4.dense(*w, 32, x, alpha=0.5, bias=b)
    got = mlk().gemm_layoutA_w4(A, S, x.to(dev), alpha=0.5, bias=b.to(dev), exact_weights=True)
    check(got, want, bound, (n, dtype))
    plain = mlk().gemm_layoutA_w4(A, S, x.to(dev), alpha=0.5, bias=b.to(dev))
    if n <= 16:
        assert torch.equal(got, plain)
    else:
        # the same bits whatever shares the call, 16 tokens at a time
        assert torch.equal(got[16:32], mlk().gemm_layoutA_w4(A, S, x[16:32].to(dev), alpha=0.5, bias=b.to(dev)))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [(2, 2, 1), (2, 2, 40), (8, 2, 50), (2, 5, 9), (3, 8, 4), (1, 1, 300)])
def test_experts_with_exact_weights_of_any_token_count(case, dtype):
    dev = require_gpu()
    E, topk, T = case
    H, I, dt = 128, 64, DT[dtype]
    off, d, s = worst_rounded(dt)
    full = lambda m, k, scale: (torch.full((E, m, k), 8 + d, dtype=torch.uint8),  # noqa: E731
                                torch.full((E, m, k // 32), s * scale, dtype=dt), None)
    w1, w2 = full(2 * I, H, 2.0 ** -6), full(H, I, 2.0 ** -6)
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    x = torch.ones(T, H, dtype=dt) * (1 + torch.arange(T).remainder(3).to(dt).unsqueeze(1) / 4)
    ids = torch.randint(0, E + 1, (T, topk), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    p = torch.ones(T, topk, dtype=dt)
    args = [t.to(dev) for t in (x, ids, p)]
    for f32 in (False, True):
        want, bound = ow4.experts(w1, w2, 32, 32, x, ids, p, out_fp32=f32)
        out = torch.full((T, H), float("nan"), dtype=torch.float32 if f32 else dt, device=dev)
        got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], *args, out=out, exact_weights=True,
                                             out_dtype=torch.float32 if f32 else None)
        assert got is out
        check(got, want, bound + 1e-30, (case, dtype, f32))
    if T * topk > 4 * E and T > 1:      # the default rounds here, and the bound tells
        rough = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], *args, out_dtype=torch.float32)
        assert ((rough.cpu().double() - want).abs() > bound).any()


def test_exact_weights_refusals_and_layer():
    dev = require_gpu()
    from muxi_native_layout_kernels_b200.muxi_moe_planC import fused_moe_w4
    E, topk, H, I, T = 4, 2, 64, 32, 30
    w1, w2 = ow4.random_weights(2 * I, H, 32, torch.bfloat16, 1, True, (E,)), ow4.random_weights(H, I, 32, torch.bfloat16, 2, False, (E,))
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    x, logits = randn((T, H), 3, 1.0, torch.bfloat16).to(dev), randn((T, E), 4, 1.0, torch.bfloat16).to(dev)
    y, ids, p = fused_moe_w4(x, a[0], b[0], logits, topk, True, w1_scale=a[1], w2_scale=b[1], w1_zeros=a[2], exact_weights=True,
                             return_routing=True)
    want, bound = ow4.experts(w1, w2, 32, 32, x.cpu(), ids.cpu(), p.cpu())
    check(y, want, bound, "layer")
    assert fused_moe_w4(x[:0], a[0], b[0], logits[:0], topk, True, w1_scale=a[1], w2_scale=b[1], exact_weights=True).shape == (0, H)
    many = torch.zeros(2, 17, dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="exact_weights"):
        mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x[:2], many, many.to(torch.bfloat16), exact_weights=True)


@pytest.mark.parametrize("static", [False, True])
def test_exact_weights_in_parts_share_their_workspace_in_order(static):
    """The launches of one call follow one another closely, over one workspace: the same bits eager, captured and replayed, and
    with the weights fetched ahead."""
    dev = require_gpu()
    E, topk, H, I, T = 4, 2, 256, 96, 150
    w = laid_out(ow4.random_weights(H, H, 128, torch.bfloat16, 5, True), dev)
    a = laid_out(ow4.random_weights(2 * I, H, 128, torch.bfloat16, 1, False, (E,)), dev)
    b = laid_out(ow4.random_weights(H, I, 32, torch.bfloat16, 2, True, (E,)), dev)
    x = randn((T, H), 3, 1.0, torch.bfloat16).to(dev)
    ids = torch.rand(T, E, generator=torch.Generator().manual_seed(6)).topk(topk, -1)[1].to(torch.int32).to(dev)
    p = torch.full((T, topk), 0.5, dtype=torch.bfloat16, device=dev)

    def chain():
        y = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x, ids, p, w2_zeros=b[2], exact_weights=True)
        return mlk().gemm_layoutA_w4(w[0], w[1], y, alpha=0.25, zeros=w[2], exact_weights=True)

    alone = []
    for i in range(0, T, 8):        # the parts one at a time, each with a workspace of its own
        rows = slice(i, i + 8)
        alone.append(mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x[rows].contiguous(), ids[rows].contiguous(),
                                                    p[rows].contiguous(), w2_zeros=b[2]))
        torch.cuda.synchronize()
    y = torch.cat(alone)
    want = torch.cat([mlk().gemm_layoutA_w4(w[0], w[1], y[i:i + 16].contiguous(), alpha=0.25, zeros=w[2]) for i in range(0, T, 16)])
    torch.cuda.synchronize()
    mlk().set_static_weights(static)
    try:
        assert torch.equal(chain(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = chain()
        for _ in range(5):
            graph.replay()
        assert torch.equal(got, want) and mlk().kernel_status() == 0
    finally:
        mlk().set_static_weights(False)
