"""Limits of the 4-bit and balance entry points, each refused on the host before anything is launched (no GPU)."""
import pytest


def experts(T=4, E=2, topk=2, H=64, I=32, status=None):
    from muxi_native_layout_kernels_b200._lib import lib
    ok = 1 << 20                                    # an aligned address that no refused call reads
    return lib.mlk_fused_experts_compute_w4(ok, ok, None, 32, ok, ok, None, 32, ok, T, E, topk, H, I, ok, ok, ok, 0, 0, None, 0,
                                            ok, 1 << 62, status, None)


@pytest.mark.parametrize("T", [1, 2, 5000])
def test_number_of_experts_has_one_limit(T):
    """Whatever the number of tokens: more than 1024 experts are refused, by this operator."""
    from muxi_native_layout_kernels_b200._lib import lib
    for topk in (1, 2, 9):
        assert experts(T=T, E=1025, topk=topk) == 2
        assert b"fused_experts_compute_w4" in lib.mlk_last_error()


def test_number_of_slots_has_one_limit():
    """65535 work items of up to 128 slots are a launch, and every expert may leave one unfilled: (65535 - 1024) * 128
    slots, whatever the number of experts."""
    from muxi_native_layout_kernels_b200._lib import lib
    most = (65535 - 1024) * 128
    for T, topk in ((most // 8 + 1, 8), (most + 1, 1), ((1 << 23), 1), (1 << 21, 8)):
        for E in (2, 128, 1024):
            assert experts(T=T, E=E, topk=topk) == 2, (T, E, topk)
            assert b"slots" in lib.mlk_last_error()


def test_every_address_has_to_be_aligned():
    """What the kernels write or read as 32-bit words, besides the inputs: results, workspace, scalar and status word."""
    from muxi_native_layout_kernels_b200._lib import lib
    ok = 1 << 20

    def loss(T=50000, loss=ok, counts=ok, dprob=ok, ws=ok):
        return lib.mlk_router_balance_loss(ok, ok, None, None, T, 8, 2, 1, 0, 1.0, 0, loss, counts, dprob, None, ws, 1 << 40, None)

    for T in (4, 50000):                            # one launch, three launches
        for off in (1, 2, 3):
            assert loss(T, loss=ok + off) == 1 and loss(T, counts=ok + off) == 1 and loss(T, dprob=ok + off) == 1
    assert loss(ws=ok + 2) == 1
    assert lib.mlk_router_balance_grad(ok, None, None, 4, 8, 1, 0, 0, ok + 2, None, ok, None) == 1
    assert lib.mlk_router_balance_grad(ok, None, None, 4, 8, 1, 0, 0, ok, ok + 2, ok, None) == 1
    assert lib.mlk_expert_counts(ok, None, 4, 2, 8, ok + 2, None) == 1
    assert lib.mlk_gemm_layoutA_w4(ok, ok, None, 32, ok, ok, 32, 20, 64, 0, 1.0, None, ok + 2, None) == 1
    assert experts(status=ok + 2) == 1
