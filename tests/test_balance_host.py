"""Balance loss: the 64-bit oracle against differences and autograd, and the refusals of the operators (no GPU)."""
import pytest
import torch

from oracle import balance as ob


def case(T, E, topk, seed, seqs=None, masked=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g, dtype=torch.float64)
    ids = torch.randint(-1, E + 1, (T, topk), generator=g, dtype=torch.int32)
    mask = torch.rand(T, generator=g) < 0.7 if masked else None
    cu = None if seqs is None else torch.tensor(seqs, dtype=torch.int32)
    return x, ids, mask, cu


CASES = [(6, 4, 2, 1, None, False), (9, 5, 3, 2, [0, 4, 4, 7], True), (3, 8, 1, 3, [1, 3], False)]


@pytest.mark.parametrize("score_fun", [0, 1])
@pytest.mark.parametrize("c", CASES)
def test_gradient_formula_against_differences(c, score_fun):
    x, ids, mask, cu = case(*c)
    loss, counts, grad = ob.balance(x, ids, score_fun, 0.3, mask, cu)
    h = 1e-6
    for t in range(x.shape[0]):
        for e in range(x.shape[1]):
            up, dn = x.clone(), x.clone()
            up[t, e] += h
            dn[t, e] -= h
            d = (ob.balance(up, ids, score_fun, 0.3, mask, cu)[0] - ob.balance(dn, ids, score_fun, 0.3, mask, cu)[0]) / (2 * h)
            # second differences are of order 1 (coef * E / topk): h^2, plus the rounding of the loss over h
            assert abs(d - float(grad[t, e])) < 1e-8


@pytest.mark.parametrize("score_fun", [0, 1])
def test_balanced_routing_gives_coef(score_fun):
    x = torch.zeros(8, 4, dtype=torch.float64)
    ids = torch.tensor([[i % 4, (i + 1) % 4] for i in range(8)], dtype=torch.int32)
    loss, counts, grad = ob.balance(x, ids, score_fun, 0.25)
    assert abs(loss - 0.25) < 1e-12 and counts.tolist() == [4, 4, 4, 4] and float(grad.abs().max()) < 1e-15


def test_refusals():
    from muxi_native_layout_kernels_b200 import expert_counts, router_balance_loss
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        router_balance_loss(x, ids)
    with pytest.raises(RuntimeError, match="CUDA"):
        expert_counts(ids, 8)


def test_c_entry_refuses_bad_arguments():
    from muxi_native_layout_kernels_b200._lib import lib
    ok = 1 << 20                                  # an aligned address that no refused call reads

    def loss(**kw):
        a = dict(logits=ok, ids=ok, mask=None, cu=None, T=50000, E=8, topk=2, B=1, score=0, coef=1.0, dtype=0, loss=ok, counts=ok,
                 dprob=ok, grad=None, ws=ok, nbytes=1 << 20)
        a.update(kw)
        return lib.mlk_router_balance_loss(*a.values(), None)

    for bad in (dict(logits=None), dict(ids=None), dict(loss=None), dict(counts=None), dict(dprob=None), dict(ws=None),
                dict(nbytes=8), dict(T=-1), dict(E=0), dict(E=1025), dict(topk=0), dict(B=0), dict(B=2), dict(score=2),
                dict(dtype=2), dict(dtype=4)):
        assert loss(**bad) in (1, 2), bad
        assert lib.mlk_last_error()
    assert lib.mlk_expert_counts(ok, None, 4, 2, 0, ok, None) in (1, 2)
    assert lib.mlk_expert_counts(None, None, 4, 2, 8, ok, None) == 1
    assert lib.mlk_expert_counts(ok, None, -1, 2, 8, ok, None) == 1
    assert lib.mlk_router_balance_grad(ok, None, None, 4, 8, 1, 0, 0, None, None, ok, None) == 1
    assert lib.mlk_router_balance_grad(ok, None, None, 4, 8, 2, 0, 0, ok, None, ok, None) == 1


def test_c_entry_refuses_sizes_and_addresses_out_of_range():
    """More picks than a 32-bit count holds, and addresses that the types' alignment rules out."""
    from muxi_native_layout_kernels_b200._lib import lib
    ok = 1 << 20

    def loss(logits=ok, ids=ok, cu=None, grad=None, T=50000, topk=2, dtype=0):
        return lib.mlk_router_balance_loss(logits, ids, None, cu, T, 8, topk, 1, 0, 1.0, dtype, ok, ok, ok, grad, ok, 1 << 40, None)

    assert loss(T=1 << 28, topk=8) == 2
    assert loss(logits=ok + 1) == 1 and loss(logits=ok + 2, dtype=3) == 1
    assert loss(ids=ok + 2) == 1 and loss(cu=ok + 2) == 1 and loss(grad=ok + 1) == 1
    assert lib.mlk_router_balance_grad(ok + 1, None, None, 4, 8, 1, 0, 0, ok, None, ok, None) == 1
    assert lib.mlk_expert_counts(ok, None, 1 << 28, 8, 8, ok, None) == 2
    assert lib.mlk_expert_counts(ok + 1, None, 4, 2, 8, ok, None) == 1
