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
