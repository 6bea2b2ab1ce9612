"""Balance loss at the ends of its range: strongly negative logits under sigmoid scores, derivatives of other kinds,
counts in a captured graph."""
import pytest
import torch

from oracle import balance as ob
from tests.gpu_util import require_gpu
from tests.test_gpu_balance import TYPES, check, dev_of, mlk

pytestmark = pytest.mark.gpu

BASES = [-50.0, -88.0, -90.0, -91.0, -95.0, -100.0, -104.0, -105.0, -200.0, -10000.0]


def negative_rows(T, E, topk, dtype, seed):
    """Row t lies around BASES[t % 10], every eleventh row is ordinary, every thirteenth has one ordinary logit."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g)
    x = x + torch.tensor(BASES)[torch.arange(T) % len(BASES)].unsqueeze(1)
    x[::11] = 1.5 * torch.randn(x[::11].shape, generator=g)
    x[::13, E // 2] = 0.25
    ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32)
    ids[:, 0] = torch.where(torch.arange(T) % 2 == 0, 0, ids[:, 0])          # an imbalance, so that the gradient is not small
    return x.to(TYPES[dtype]), ids


def check_far(got, x, ids, score_fun, coef):
    """`check`, plus what fp32 can hold below 2^-126, where a rounding is off by up to 2^-150 whatever the value.  A score
    exp (2 units of 2^-149) * d * inv, inv <= 2, is off by 2 (2 + 1/2) + 1/2 = 5.5 units; a term p u of the row's sum by
    5.5 U + 1/2, U = the largest u, and the sum of E of them (exact there) by E (5.5 U + 1/2); the gradient p (u - sum)
    (1 - sigma) by 5.5 U, that sum's error and three roundings more: (E + 1) (5.5 U) + E / 2 + 3 / 2 units."""
    T, E = x.shape
    u = coef * E * torch.bincount(ids.flatten().long(), minlength=E).max().item() / (ids.shape[1] * T * T)
    off = ((E + 1) * 5.5 * u + E / 2 + 1.5) * 2.0 ** -149
    _, _, grad = ob.balance(x, ids, score_fun, coef)
    g = got[2].cpu().double()
    far = torch.where((g - grad).abs() <= off, grad, g)          # what is left has to pass as it is
    check((got[0], got[1], far.to(x.dtype).cuda()), x, ids, score_fun, coef, None, None)
    assert got[2].dtype == x.dtype


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 8, 2), (40, 8, 2), (60, 128, 8), (33, 60, 3), (300, 128, 8), (17000, 8, 2), (1200, 128, 8)])
def test_sigmoid_scores_of_strongly_negative_rows(shape, dtype):
    """Ratios of sigmoids that are no fp32 numbers themselves, held to what `check` grants ordinary rows: differences from
    the row's largest logit are at most 16 where they matter (an fp32 rounding of 2^-20), exp and the quotients add 2^-22,
    a row's sum of at most 1 + 32 + 5 terms 2^-19.  Scores that are subnormal: see `check_far`."""
    require_gpu()
    T, E, topk = shape
    x, ids = negative_rows(T, E, topk, dtype, T + E)
    got = mlk().router_balance_loss(*dev_of(x, ids), 1, 0.7, return_grad=True)
    assert torch.isfinite(got[0]) and torch.isfinite(got[2]).all()
    check_far(got, x, ids, 1, 0.7)
    leaf = x.cuda().requires_grad_()
    loss, counts = mlk().router_balance_loss(leaf, ids.cuda(), 1, 0.7)
    loss.backward()
    check_far((loss.detach(), counts, leaf.grad), x, ids, 1, 0.7)


@pytest.mark.parametrize("T", [24, 17000])
def test_sigmoid_rows_without_a_distribution_or_with_nan(T):
    """Rows of -inf stay 0 beside rows of -1e4; infinities count as scores of 1 and 0; NaN reaches the loss."""
    require_gpu()
    x, ids = negative_rows(T, 8, 2, "fp32", 3)
    x[4] = -float("inf")
    x[5, :5] = -float("inf")
    x[6, 1] = float("inf")
    x[7] = torch.finfo(torch.float32).min
    got = mlk().router_balance_loss(*dev_of(x, ids), 1, 1.0, return_grad=True)
    check_far(got, x, ids, 1, 1.0)
    assert (got[2][4] == 0).all()
    x[8, 2] = float("nan")
    got = mlk().router_balance_loss(*dev_of(x, ids), 1, 1.0, return_grad=True)
    assert torch.isnan(got[0]) and torch.isnan(got[2][8]).any() and torch.isfinite(got[2][9]).all()


def test_forward_mode_is_refused():
    """A dual tensor has no requires_grad; its tangent must not be dropped in silence."""
    require_gpu()
    import torch.autograd.forward_ad as fw
    x, ids = torch.randn(6, 8, device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for kw in ({}, {"return_grad": True}):
            with pytest.raises(RuntimeError, match="forward"):
                mlk().router_balance_loss(dual, ids, **kw)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
            mlk().router_balance_loss(dual, ids)
        mlk().router_balance_loss(x, ids)
    mlk().router_balance_loss(x, ids)


@pytest.mark.parametrize("T", [6, 17000])
def test_second_order_of_the_rest(T):
    """create_graph over a loss of which this one is a part: the first derivatives are the usual ones, the other part
    can be differentiated again, and only differentiating this one again is an error."""
    require_gpu()
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 8, generator=g).cuda().requires_grad_()
    w = torch.randn(5, generator=g).cuda().requires_grad_()
    ids = torch.randint(0, 8, (T, 2), generator=g, dtype=torch.int32).cuda()
    want = mlk().router_balance_loss(x.detach(), ids, 0, 0.5, return_grad=True)[2]
    total = mlk().router_balance_loss(x, ids, 0, 0.5)[0] + (w ** 3).sum()
    gx, gw = torch.autograd.grad(total, (x, w), create_graph=True)
    assert (gx.detach() - want).abs().max() <= want.abs().max() * 2.0 ** -15
    (gw ** 2).sum().backward(retain_graph=True)
    assert torch.allclose(w.grad, 36 * w.detach() ** 3, rtol=1e-5) and x.grad is None
    with pytest.raises(RuntimeError, match="once"):
        gx.sum().backward()


@pytest.mark.parametrize("masked", [False, True])
def test_expert_counts_in_a_graph(masked):
    """Captured without a call before it, replayed with other picks: every replay starts from zero."""
    require_gpu()
    g = torch.Generator().manual_seed(1)
    draws = [torch.randint(-1, 20, (700, 3), generator=g, dtype=torch.int32) for _ in range(3)]
    mask = (torch.rand(700, generator=g) < 0.5).cuda() if masked else None
    ids = draws[0].cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        counts = mlk().expert_counts(ids, 16, mask)
    for d in draws + draws[:1]:
        ids.copy_(d)
        graph.replay()
        rows = d if mask is None else d[mask.cpu()]
        want = torch.bincount(rows[(rows >= 0) & (rows < 16)].long(), minlength=16)
        assert torch.equal(counts.cpu().long(), want)


def test_oracle_used_here_holds_far_from_zero():
    """The 64-bit form at -1e4 against the closed form of two experts: p = 1 / (1 + e^d)."""
    x = torch.tensor([[-10000.0, -10001.0]], dtype=torch.float64)
    p = ob.probs(x, 1)
    assert abs(float(p[0, 0]) - 1 / (1 + float(torch.exp(torch.tensor(-1.0, dtype=torch.float64))))) < 1e-12
