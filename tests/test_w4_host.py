"""4-bit weights without a GPU: the oracle's own layouts, quantisation helpers, and the refusals of every entry point."""
import pytest
import torch

from oracle import w4 as ow4


def test_oracle_blocks_hold_every_nibble_once():
    q = torch.arange(16 * 64).reshape(16, 64) % 16
    b = ow4.pack_blocks(q.to(torch.uint8))
    assert b.shape == (1, 1, 32, 16)
    low, high = (b & 15).flatten(), (b >> 4).flatten()
    assert torch.equal(torch.bincount(torch.cat((low, high)).long(), minlength=16), torch.full((16,), 64))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_round_trip(dtype, group, zeros):
    from muxi_native_layout_kernels_b200 import utils
    g = torch.Generator().manual_seed(group)
    w = (0.05 * torch.randn(2, 32, 256, generator=g) + (0.02 if zeros else 0)).to(dtype)
    w[0, 3, :group] = 0
    q, s, z = utils.quantize_w4(w, group, zeros)
    assert q.shape == (2, 32, 128) and q.dtype == torch.uint8 and s.shape == (2, 32, 256 // group) and s.dtype == dtype
    assert (z is None) != zeros
    d = utils.dequantize_w4(q, s, z)
    # nearest of 16 values: half a step, and up to half a step more where a rounded scale or zero point clips the ends
    step = s.float().repeat_interleave(group, -1)
    assert ((d - w.float()).abs() <= step * 1.05).all()
    assert (d[0, 3, :group] == 0).all()
    with pytest.raises(ValueError):
        utils.quantize_w4(w, 48)


def test_python_refusals_on_the_cpu():
    import muxi_native_layout_kernels_b200 as m
    from muxi_native_layout_kernels_b200.muxi_moe_planC import fused_moe_w4
    W = torch.zeros(32, 32, dtype=torch.uint8)
    A, S = torch.zeros(2, 1, 32, 16, dtype=torch.uint8), torch.zeros(2, 1, 8, 2, dtype=torch.bfloat16)
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    for call in (lambda: m.layoutA_w4(W), lambda: m.layoutA_w4_groups(S[0, 0]), lambda: m.layoutA_w4_inverse(A, 64),
                 lambda: m.gemm_layoutA_w4(A, S, x), lambda: m.gemv_layoutA_w4(A, S, x)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        fused_moe_w4(x, A, A, x, 1, False)


def test_c_entries_refuse_bad_arguments():
    from muxi_native_layout_kernels_b200._lib import lib
    ok, odd = 1 << 20, (1 << 20) + 2                # addresses that no refused call reads

    def gemm(**kw):
        a = dict(A=ok, s=ok, z=None, group=32, B=ok, C=ok, m=32, n=1, k=64, dtype=0, alpha=1.0, bias=None, status=None)
        a.update(kw)
        return lib.mlk_gemm_layoutA_w4(*a.values(), None)

    for bad in (dict(A=None), dict(s=None), dict(B=None), dict(C=None), dict(group=16), dict(group=48), dict(group=128), dict(m=0),
                dict(m=24), dict(n=-1), dict(k=0), dict(k=48), dict(dtype=2), dict(A=odd), dict(s=odd), dict(z=odd), dict(B=odd),
                dict(C=odd), dict(bias=odd + 1)):
        assert gemm(**bad) == 1, bad
        assert lib.mlk_last_error()
    assert gemm(n=0, B=None, C=None) == 0           # nothing to do

    def experts(**kw):
        a = dict(w1=ok, s1=ok, z1=None, g1=32, w2=ok, s2=ok, z2=None, g2=32, x=ok, T=4, E=2, topk=2, H=64, I=32, ids=ok, p=ok, y=ok,
                 dtype=0, f32=0, map=None, maplen=0, ws=ok, nbytes=1 << 30, status=None)
        a.update(kw)
        return lib.mlk_fused_experts_compute_w4(*a.values(), None)

    for bad in (dict(w1=None), dict(s2=None), dict(g1=40), dict(g2=64), dict(x=None), dict(T=-1), dict(E=0), dict(topk=0), dict(H=48),
                dict(I=16), dict(ids=None), dict(p=None), dict(y=None), dict(dtype=2), dict(ws=None), dict(nbytes=64), dict(x=odd),
                dict(ws=odd), dict(map=ok, maplen=0), dict(w2=odd)):
        assert experts(**bad) == 1, bad
    assert experts(T=1 << 24) == 2
    assert experts(T=0, x=None, ids=None, p=None, y=None, ws=None) == 0
    assert lib.mlk_experts_w4_workspace_bytes(0, 2, 2, 64, 32) == 0
    assert lib.mlk_experts_w4_workspace_bytes(4, 2, 2, 64, 32) > 4 * 2 * (64 * 4 + 32 * 2)

    for bad in ((ok, ok, 8, 64, 0), (ok, ok, 16, 48, 0), (ok, ok, 16, 0, 0), (None, ok, 16, 64, 0), (ok, odd, 16, 64, 1)):
        assert lib.mlk_layoutA_w4(*bad, None) == 1, bad
    for bad in ((ok, ok, 8, 2, 2), (ok, ok, 16, 0, 2), (ok, ok, 16, 2, 4), (ok, None, 16, 2, 2)):
        assert lib.mlk_layoutA_w4_groups(*bad, None) == 1, bad


def test_c_entries_refuse_sizes_and_addresses_out_of_range():
    """Sizes beyond the kernels' 32-bit row arithmetic and addresses that the types' alignment rules out."""
    from muxi_native_layout_kernels_b200._lib import lib
    ok, odd, big = 1 << 20, (1 << 20) + 1, (1 << 28) + 128

    def gemm(m=32, k=64):
        return lib.mlk_gemm_layoutA_w4(ok, ok, None, 32, ok, ok, m, 1, k, 0, 1.0, None, None, None)

    assert gemm(m=big) == 2 and gemm(k=big) == 2 and gemm(m=2 ** 31 - 16) == 2

    def experts(H=64, I=32, ids=ok, p=ok, mp=None):
        return lib.mlk_fused_experts_compute_w4(ok, ok, None, 32, ok, ok, None, 32, ok, 4, 2, 2, H, I, ids, p, ok, 0, 0, mp, 2, ok,
                                                1 << 62, None, None)

    assert experts(H=big) == 2 and experts(I=big // 2) == 2 and experts(I=1 << 30) == 2
    assert experts(ids=ok + 2) == 1 and experts(p=odd) == 1 and experts(mp=ok + 2) == 1
    assert lib.mlk_layoutA_w4_groups(odd, ok, 16, 2, 2, None) == 1
    assert lib.mlk_layoutA_w4_groups(ok, odd, 16, 2, 2, None) == 1
