"""Sizes that the C interface's 32-bit integers cannot hold are refused by the Python functions, not cut off (no GPU: stand-ins
that have a tensor's shape and nothing behind it)."""
import pytest
import torch


class Shaped:
    """A contiguous CUDA tensor to look at."""
    is_cuda, device = True, torch.device("cuda", 0)

    def __init__(self, shape, dtype):
        self.shape, self.dtype = torch.Size(shape), dtype

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def dim(self):
        return len(self.shape)

    def size(self, i=None):
        return self.shape if i is None else self.shape[i]

    def numel(self):
        return self.shape.numel()

    def element_size(self):
        return self.dtype.itemsize


BIG = 2 ** 32                    # a multiple that 32 bits lose without a trace


@pytest.fixture
def m(monkeypatch):
    """The package with allocation and launch replaced: whatever gets that far has passed the checks."""
    import muxi_native_layout_kernels_b200 as pkg
    from muxi_native_layout_kernels_b200 import balance, w4

    def reached(*a, **kw):
        pytest.fail("not refused")

    for mod in (balance, w4):
        monkeypatch.setattr(mod, "_launch", reached)
    monkeypatch.setattr(torch, "empty", reached)
    for name in ("new_empty", "detach", "data_ptr", "requires_grad"):
        monkeypatch.setattr(Shaped, name, property(reached), raising=False)
    return pkg


@pytest.mark.parametrize("extra", [4, -4, 2 ** 31 + 8])
def test_balance(m, extra):
    T = BIG + extra if extra < 2 ** 31 else 2 ** 31
    x, ids = Shaped((T, 1), torch.bfloat16), Shaped((T, 1), torch.int32)
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.router_balance_loss(x, ids)
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.router_balance_loss(x, ids, return_grad=True)
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.router_balance_loss(Shaped((4, 8), torch.bfloat16), Shaped((4, BIG + 2), torch.int32))
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.router_balance_loss(Shaped((4, 8), torch.bfloat16), Shaped((4, 2), torch.int32),
                              cu_seqlens=Shaped((T + 1,), torch.int32))
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.router_balance_loss(Shaped((4, BIG + 8), torch.bfloat16), Shaped((4, 2), torch.int32))


def test_expert_counts(m):
    for ids, E in ((Shaped((BIG + 4, 1), torch.int32), 8), (Shaped((4, BIG + 1), torch.int32), 8), (Shaped((4, 2), torch.int32), BIG + 8)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            m.expert_counts(ids, E)


def test_prepack(m):
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.layoutA_w4(Shaped((16, BIG // 2 + 32), torch.uint8))
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.layoutA_w4_inverse(Shaped((1, BIG // 64 + 1, 32, 16), torch.uint8), BIG + 64)
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.layoutA_w4_groups(Shaped((16, BIG + 1), torch.uint8))


def test_products(m):
    def product(rows, k):
        return (Shaped((rows // 16, (k + 63) // 64, 32, 16), torch.uint8), Shaped((rows // 16, k // 32, 8, 2), torch.bfloat16),
                Shaped((1, k), torch.bfloat16))

    for rows, k in ((BIG + 16, 32), (16, BIG + 64), (2 ** 31, 32)):
        for f in (m.gemm_layoutA_w4, m.gemv_layoutA_w4):
            with pytest.raises(RuntimeError, match="2\\^31"):
                f(*product(rows, k))
    with pytest.raises(RuntimeError, match="2\\^31"):
        m.gemm_layoutA_w4(*product(16, 32)[:2], Shaped((BIG + 1, 32), torch.bfloat16))


def test_experts(m):
    def call(T=4, topk=2, H=64, I=32, E=2):
        f, u = torch.bfloat16, torch.uint8
        m.fused_experts_compute_w4(Shaped((E, 2 * I // 16, (H + 63) // 64, 32, 16), u), Shaped((E, 2 * I // 16, H // 32, 8, 2), f),
                                   Shaped((E, H // 16, (I + 63) // 64, 32, 16), u), Shaped((E, H // 16, I // 32, 8, 2), f),
                                   Shaped((T, H), f), Shaped((T, topk), torch.int32), Shaped((T, topk), f))

    for kw in (dict(T=BIG + 4), dict(topk=BIG + 2), dict(H=BIG + 64), dict(I=BIG + 32), dict(E=BIG + 2)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            call(**kw)


def test_prepack_at_the_end_of_32_bits():
    """The C entry's own arithmetic on k near 2^31."""
    from muxi_native_layout_kernels_b200._lib import lib
    ok = 1 << 20
    for inverse in (0, 1):
        assert lib.mlk_layoutA_w4(ok, ok, 16, 2 ** 31 - 32, inverse, None) == 2
        assert lib.mlk_layoutA_w4(ok, ok, 16, 2 ** 28 + 32, inverse, None) == 2
