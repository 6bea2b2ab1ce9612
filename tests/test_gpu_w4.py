"""4-bit weights on the GPU: prepack, dense products and the experts of a mixture layer, against the 64-bit oracle.

Every comparison is elementwise against a bound that the oracle derives for the same inputs (fp32 sums, one rounding of
the result, and, where the weights are rounded to 16 bits, half a step of each weight)."""
import pytest
import torch

from oracle import w4 as ow4
from tests.gpu_util import DT, randn, require_gpu

pytestmark = pytest.mark.gpu


def mlk():
    import muxi_native_layout_kernels_b200 as m
    return m


def laid_out(w, dev):
    q, s, z = w
    m = mlk()
    return (m.layoutA_w4(ow4.pack_rows(q).to(dev)), m.layoutA_w4_groups(s.to(dev)),
            None if z is None else m.layoutA_w4_groups(z.to(dev)))


def check(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    worst = ((got - want).abs() / bound).max().item() if want.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"
    assert not torch.isnan(got).any(), what


@pytest.mark.parametrize("shape", [(16, 32), (48, 64), (160, 96), (32, 2080), (1040, 256)])
def test_prepack_matches_the_definition_and_inverts(shape):
    dev = require_gpu()
    m = mlk()
    q, s, z = ow4.random_weights(*shape, 32, torch.bfloat16, 1, zeros=True)
    rows = ow4.pack_rows(q)
    A = m.layoutA_w4(rows.to(dev))
    assert torch.equal(A.cpu(), ow4.pack_blocks(q))
    assert torch.equal(m.layoutA_w4_inverse(A, shape[1]).cpu(), rows)
    for v in (s, z, s.to(torch.float16)):
        assert torch.equal(m.layoutA_w4_groups(v.to(dev)).cpu(), ow4.pair_order(v))


def test_prepack_of_experts_keeps_the_leading_dimension():
    dev = require_gpu()
    m = mlk()
    q, s, z = ow4.random_weights(48, 96, 32, torch.float16, 2, zeros=True, lead=(3,))
    A = m.layoutA_w4(ow4.pack_rows(q).to(dev))
    assert torch.equal(A.cpu(), ow4.pack_blocks(q))
    assert torch.equal(m.layoutA_w4_inverse(A, 96).cpu(), ow4.pack_rows(q))
    assert torch.equal(m.layoutA_w4_groups(s.to(dev)).cpu(), ow4.pair_order(s))


DENSE = [  # m, k, group
    (16, 32, 32), (16, 64, 64), (16, 128, 128), (48, 96, 32), (32, 160, 32), (272, 192, 64), (128, 2080, 32), (144, 1152, 128),
    (1040, 544, 32), (2064, 640, 128),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("mkg", DENSE)
def test_dense_against_oracle(mkg, zeros, dtype):
    dev = require_gpu()
    m, k, group = mkg
    w = ow4.random_weights(m, k, group, DT[dtype], m + k, zeros)
    A, S, Z = laid_out(w, dev)
    for n in (1, 2, 7, 8, 9, 16):
        x = randn((n, k), n, 1.0, DT[dtype])
        want, bound = ow4.dense(*w, group, x)
        got = mlk().gemm_layoutA_w4(A, S, x.to(dev), zeros=Z)
        check(got, want, bound, (mkg, zeros, dtype, n))
        if n == 1:
            assert torch.equal(mlk().gemv_layoutA_w4(A, S, x.to(dev), zeros=Z), got)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [17, 31, 32, 33, 63, 64, 65, 127, 130, 200, 257, 520])
def test_many_tokens_against_oracle(n, dtype):
    dev = require_gpu()
    for i, (m, k, group) in enumerate([(16, 32, 32), (144, 160, 32), (272, 384, 128), (400, 192, 64)]):
        w = ow4.random_weights(m, k, group, DT[dtype], m + k, i % 2 == 1)
        A, S, Z = laid_out(w, dev)
        x = randn((n, k), n, 1.0, DT[dtype])
        want, bound = ow4.dense(*w, group, x, rounded_weights=True)
        got = mlk().gemm_layoutA_w4(A, S, x.to(dev), zeros=Z)
        check(got, want, bound, (m, k, group, n, dtype))
        # the roundings of weights and result are independent: in the 2-norm a step of the type covers both
        rel = ((got.cpu().double() - want).norm() / want.norm()).item()
        assert rel <= torch.finfo(DT[dtype]).eps, (m, k, group, n, dtype, rel)


@pytest.mark.parametrize("n", [1, 12, 40, 150])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_alpha_and_bias(n, dtype):
    dev = require_gpu()
    m, k, group = 208, 256, 64
    w = ow4.random_weights(m, k, group, DT[dtype], 5, True)
    A, S, Z = laid_out(w, dev)
    x, b = randn((n, k), 3, 1.0, DT[dtype]), randn((m,), 4, 1.0, DT[dtype])
    want, bound = ow4.dense(*w, group, x, alpha=-0.37, bias=b, rounded_weights=n > 16)
    got = mlk().gemm_layoutA_w4(A, S, x.to(dev), alpha=-0.37, beta=2.0, zeros=Z, bias=b.to(dev))
    check(got, want, bound, (n, dtype))


@pytest.mark.parametrize("n", [1, 8, 16, 40, 130])
def test_extreme_scales_and_activations(n):
    """Scales and activations near the ends of the types: exact powers of two, so that the products stay in range."""
    dev = require_gpu()
    m, k, group = 32, 128, 32
    for dtype, lo, hi in ((torch.bfloat16, 2.0 ** -100, 2.0 ** 96), (torch.float16, 2.0 ** -14, 2.0 ** 3)):
        q, _, z = ow4.random_weights(m, k, group, dtype, 6, True)
        for sv, xv in ((lo, hi), (hi, lo)):
            s = torch.full((m, k // group), sv, dtype=dtype)
            x = (randn((n, k), 7, 1.0, torch.float32).sign() * xv).to(dtype)
            want, bound = ow4.dense(q, s, z, group, x, rounded_weights=n > 16)
            got = mlk().gemm_layoutA_w4(*laid_out((q, s, None), dev)[:2], x.to(dev), zeros=laid_out((q, s, z), dev)[2])
            check(got, want, bound, (n, dtype, sv))


@pytest.mark.parametrize("n", [1, 9, 40])
def test_infinite_and_nan_tokens_stay_in_their_rows(n):
    dev = require_gpu()
    m, k, group = 64, 160, 32
    w = ow4.random_weights(m, k, group, torch.bfloat16, 8, True)
    A, S, Z = laid_out(w, dev)
    x = randn((n + 1, k), 9, 1.0, torch.bfloat16)
    x[0, 5] = float("inf")
    if n > 1:
        x[1, 7] = float("nan")
    bad = 2 if n > 1 else 1
    want, bound = ow4.dense(*w, group, x[bad:], rounded_weights=n + 1 > 16)
    got = mlk().gemm_layoutA_w4(A, S, x.to(dev), zeros=Z)
    check(got[bad:], want, bound, n)
    assert not torch.isfinite(got[0]).all()
    if n > 1:
        assert torch.isnan(got[1]).all()


def test_no_tokens():
    dev = require_gpu()
    w = ow4.random_weights(32, 64, 32, torch.bfloat16, 1)
    A, S, _ = laid_out(w, dev)
    assert mlk().gemm_layoutA_w4(A, S, torch.empty(0, 64, dtype=torch.bfloat16, device=dev)).shape == (0, 32)


EXPERTS = [  # E, topk, H, I, T, group1, group2
    (4, 2, 64, 32, 1, 32, 32), (8, 2, 128, 96, 3, 64, 32), (16, 4, 256, 128, 9, 128, 64), (3, 1, 96, 160, 5, 32, 32),
    (8, 8, 128, 128, 17, 128, 128), (4, 2, 384, 288, 40, 128, 32), (2, 2, 128, 64, 70, 32, 64),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("case", EXPERTS)
def test_experts_against_oracle(case, zeros, dtype):
    dev = require_gpu()
    E, topk, H, I, T, g1, g2 = case
    dt = DT[dtype]
    w1 = ow4.random_weights(2 * I, H, g1, dt, 1, zeros, (E,))
    w2 = ow4.random_weights(H, I, g2, dt, 2, zeros, (E,))
    x = randn((T, H), 3, 1.0, dt)
    g = torch.Generator().manual_seed(4)
    ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32)
    p = torch.rand(T, topk, generator=g).to(dt)
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    for f32 in (False, True):
        want, bound = ow4.experts(w1, w2, g1, g2, x, ids, p, rounded_weights=True, out_fp32=f32)
        got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), w1_zeros=a[2],
                                             w2_zeros=b[2], out_dtype=torch.float32 if f32 else None)
        assert got.dtype == (torch.float32 if f32 else dt)
        check(got, want, bound, (case, zeros, dtype, f32))
        # four independent roundings at most (both weights, the activation, the result)
        rel = ((got.cpu().double() - want).norm() / want.norm()).item()
        assert rel <= 2 * torch.finfo(dt).eps, (case, zeros, dtype, f32, rel)


@pytest.mark.parametrize("T", [1, 6, 50])
def test_experts_map_repeated_and_foreign_ids(T):
    """Experts of other ranks, ids outside the map, a token with the same expert twice, tokens with no expert here."""
    dev = require_gpu()
    E, topk, H, I = 4, 3, 128, 64
    w1 = ow4.random_weights(2 * I, H, 64, torch.bfloat16, 1, True, (E,))
    w2 = ow4.random_weights(H, I, 32, torch.bfloat16, 2, False, (E,))
    x = randn((T, H), 3, 1.0, torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(-2, 12, (T, topk), generator=g, dtype=torch.int32)
    ids[0] = torch.tensor([3, 3, 5])
    if T > 1:
        ids[1] = torch.tensor([-1, 11, 9])
    emap = torch.full((10,), -1, dtype=torch.int32)
    emap[3], emap[5], emap[0], emap[8] = 2, 0, 1, 3
    p = torch.rand(T, topk, generator=g).to(torch.bfloat16)
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    want, bound = ow4.experts(w1, w2, 64, 32, x, ids, p, emap, rounded_weights=True)
    out = torch.full((T, H), 7.0, dtype=torch.bfloat16, device=dev)
    got = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], x.to(dev), ids.to(dev), p.to(dev), w1_zeros=a[2],
                                         experts_map=emap.to(dev), out=out)
    assert got is out
    check(got, want, bound, T)
    if T > 1:
        assert (got[1] == 0).all()


def test_experts_no_tokens():
    dev = require_gpu()
    w1, w2 = ow4.random_weights(64, 64, 32, torch.bfloat16, 1, lead=(2,)), ow4.random_weights(64, 32, 32, torch.bfloat16, 2, lead=(2,))
    a, b = laid_out(w1, dev), laid_out(w2, dev)
    y = mlk().fused_experts_compute_w4(a[0], a[1], b[0], b[1], torch.empty(0, 64, dtype=torch.bfloat16, device=dev),
                                       torch.empty(0, 2, dtype=torch.int32, device=dev),
                                       torch.empty(0, 2, dtype=torch.bfloat16, device=dev))
    assert y.shape == (0, 64)


@pytest.mark.parametrize("n", [1, 16, 40, 300])
def test_results_do_not_depend_on_the_run(n):
    dev = require_gpu()
    w = ow4.random_weights(528, 1152, 128, torch.bfloat16, 3, True)
    A, S, Z = laid_out(w, dev)
    x = randn((n, 1152), 1, 1.0, torch.bfloat16).to(dev)
    first = mlk().gemm_layoutA_w4(A, S, x, zeros=Z)
    for _ in range(3):
        assert torch.equal(mlk().gemm_layoutA_w4(A, S, x, zeros=Z), first)


@pytest.mark.parametrize("T", [1, 5, 64])
def test_experts_in_a_graph_and_on_another_stream(T):
    dev = require_gpu()
    E, topk, H, I = 8, 2, 256, 128
    w1 = laid_out(ow4.random_weights(2 * I, H, 128, torch.bfloat16, 1, False, (E,)), dev)
    w2 = laid_out(ow4.random_weights(H, I, 64, torch.bfloat16, 2, True, (E,)), dev)
    x = randn((T, H), 3, 1.0, torch.bfloat16).to(dev)
    g = torch.Generator().manual_seed(4)
    draws = [torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32).to(dev) for _ in range(3)]
    p = torch.rand(T, topk, generator=g).to(torch.bfloat16).to(dev)
    call = lambda i: mlk().fused_experts_compute_w4(w1[0], w1[1], w2[0], w2[1], x, i, p, w2_zeros=w2[2])  # noqa: E731
    eager = [call(i) for i in draws]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [call(i) for i in draws]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    ids = draws[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(ids)
    for i, want in zip(draws, eager):
        ids.copy_(i)
        graph.replay()
        assert torch.equal(y, want)
