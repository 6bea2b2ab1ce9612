"""Balance loss, per-expert counts and gradients on the GPU against the 64-bit oracle."""
import pytest
import torch

from oracle import balance as ob
from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def mlk():
    import muxi_native_layout_kernels_b200 as m
    return m


def inputs(T, E, topk, dtype, seed, seqs=None, masked=False, foreign=False):
    g = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(T, E, generator=g)).to(TYPES[dtype])
    ids = torch.rand(T, E, generator=g).topk(topk, -1)[1].to(torch.int32)
    if foreign:
        ids[::3, 0] = -1
        ids[1::3, -1] = E + 5
    mask = torch.rand(T, generator=g) < 0.6 if masked else None
    cu = None if seqs is None else torch.tensor(seqs, dtype=torch.int32)
    return x, ids, mask, cu


def dev_of(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check(got, x, ids, score_fun, coef, mask, cu):
    """loss and gradient against the oracle: fp32 chains of at most 512 additions (2^-15), p and u within 2^-18 of their
    values, the gradient rounded once."""
    loss, counts, grad = ob.balance(x, ids, score_fun, coef, mask, cu)
    assert got[0].dtype == torch.float32 and got[0].dim() == 0
    assert abs(float(got[0]) - loss) <= abs(loss) * 2.0 ** -15
    assert got[1].dtype == torch.int32 and torch.equal(got[1].cpu().long(), counts)
    if len(got) > 2:
        p = ob.probs(x, score_fun)
        # |d| = p |u - sum p u|: both terms bounded through the largest u of the loss
        u = torch.zeros_like(p)
        bounds = [0, x.shape[0]] if cu is None else cu.tolist()
        for a, z in zip(bounds, bounds[1:]):
            rows = [t for t in range(a, z) if mask is None or bool(mask[t])]
            if rows:
                c = torch.stack([(ids[rows] == e).sum() for e in range(x.shape[1])]).double()
                u[rows] = coef * x.shape[1] * c / ((len(bounds) - 1) * ids.shape[1] * len(rows) ** 2)
        step = torch.finfo(x.dtype).eps / 2
        bound = p * (u + (p * u).sum(-1, keepdim=True)) * 2.0 ** -17
        bound = bound + (grad.abs() + bound) * step + torch.finfo(x.dtype).smallest_normal * step
        g = got[2].cpu().double()
        assert got[2].dtype == x.dtype
        assert ((g - grad).abs() <= bound).all(), float(((g - grad).abs() / bound).max())


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 4, 4), (33, 60, 3), (192, 8, 2), (130, 128, 8), (257, 160, 6), (70, 256, 8), (9, 1024, 8),
          (12, 1000, 2), (6, 1023, 5), (500, 7, 1), (64, 17, 2), (40, 768, 3), (25, 36, 2)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("score_fun", [0, 1])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_sequence(shape, score_fun, dtype):
    require_gpu()
    x, ids, _, _ = inputs(*shape, dtype, sum(shape))
    got = mlk().router_balance_loss(*dev_of(x, ids), score_fun, 0.7, return_grad=True)
    check(got, x, ids, score_fun, 0.7, None, None)
    assert torch.equal(mlk().router_balance_loss(*dev_of(x, ids), score_fun, 0.7)[0], got[0])


SEQS = [(10, [0, 10]), (50, [0, 7, 7, 50]), (64, [3, 20, 21, 40]), (40, [0, 0, 0]), (300, [0, 299, 300]),
        (200, list(range(0, 201, 2))), (90, [90, 90]), (1500, [0, 3, 700, 1300, 1301, 1450]), (700, list(range(0, 701)))]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("score_fun", [0, 1])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("seq", range(len(SEQS)))
def test_sequences_masks_and_foreign_ids(seq, masked, score_fun, dtype):
    require_gpu()
    T, cu = SEQS[seq]
    E, topk = (16, 2) if seq % 2 else (12, 3)
    x, ids, mask, cu = inputs(T, E, topk, dtype, seq, cu, masked, foreign=True)
    got = mlk().router_balance_loss(*dev_of(x, ids), score_fun, 1.3, **dict(zip(("token_mask", "cu_seqlens"), dev_of(mask, cu))),
                                    return_grad=True)
    check(got, x, ids, score_fun, 1.3, mask, cu)


def test_uncounted_tokens_are_not_read():
    """NaN and infinities in masked tokens and behind the last sequence leave no trace; every id outside: loss 0."""
    require_gpu()
    x, ids, mask, cu = inputs(60, 8, 2, "bf16", 3, [0, 20, 48], True)
    want = mlk().router_balance_loss(*dev_of(x, ids), 0, 1.0, token_mask=mask.cuda(), cu_seqlens=cu.cuda(), return_grad=True)
    y = x.clone()
    y[~mask] = float("nan")
    y[48:] = float("inf")
    got = mlk().router_balance_loss(*dev_of(y, ids), 0, 1.0, token_mask=mask.to(torch.uint8).cuda(), cu_seqlens=cu.cuda(), return_grad=True)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    assert (got[2][48:] == 0).all() and (got[2][~mask] == 0).all()
    none = mlk().router_balance_loss(x.cuda(), torch.full_like(ids, -1).cuda(), 0, 1.0, return_grad=True)
    assert float(none[0]) == 0 and int(none[1].sum()) == 0 and (none[2] == 0).all()
    off = mlk().router_balance_loss(*dev_of(x, ids), 0, 1.0, token_mask=torch.zeros(60, dtype=torch.bool).cuda(), return_grad=True)
    assert float(off[0]) == 0 and int(off[1].sum()) == 0 and (off[2] == 0).all()


@pytest.mark.parametrize("score_fun", [0, 1])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_masked_logits(dtype, score_fun):
    """Logits of -inf and of the type's lowest value; a token with nothing but -inf."""
    require_gpu()
    x, ids, _, _ = inputs(40, 16, 2, dtype, 4)
    x[:, 3] = -float("inf")
    x[5:9, :8] = -float("inf")
    x[10] = -float("inf")
    x[11, 4:] = torch.finfo(x.dtype).min
    got = mlk().router_balance_loss(*dev_of(x, ids), score_fun, 1.0, return_grad=True)
    check(got, x, ids, score_fun, 1.0, None, None)
    assert (got[2][10] == 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_autograd_and_upstream_gradient(dtype):
    require_gpu()
    x, ids, mask, cu = inputs(150, 32, 4, dtype, 5, [0, 60, 140], True)
    kw = dict(token_mask=mask.cuda(), cu_seqlens=cu.cuda())
    direct = mlk().router_balance_loss(*dev_of(x, ids), 1, 0.5, return_grad=True, **kw)
    leaf = x.cuda().requires_grad_()
    loss, counts = mlk().router_balance_loss(leaf, ids.cuda(), 1, 0.5, **kw)
    assert torch.equal(loss.detach(), direct[0]) and torch.equal(counts, direct[1]) and not counts.requires_grad
    loss.backward()
    assert torch.equal(leaf.grad, direct[2])
    leaf.grad = None
    (4 * mlk().router_balance_loss(leaf, ids.cuda(), 1, 0.5, **kw)[0]).backward()
    # a factor of four is exact except where the type's smallest numbers begin
    small = direct[2].abs().float() <= 8 * torch.finfo(x.dtype).smallest_normal
    assert torch.equal(leaf.grad[~small], 4 * direct[2][~small])
    with torch.no_grad():
        assert torch.equal(mlk().router_balance_loss(leaf, ids.cuda(), 1, 0.5, **kw)[0], direct[0])


@pytest.mark.parametrize("T", [40, 6000])
def test_backward_pass_in_a_graph(T):
    """Forward and backward captured together, no eager graph of the leaf alive, replayed with other logits."""
    require_gpu()
    (x, ids, _, _), other = inputs(T, 32, 4, "fp32", 5), inputs(T, 32, 4, "fp32", 6)[0]
    leaf, ids = x.cuda().requires_grad_(), ids.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mlk().router_balance_loss(leaf, ids)[0].backward()
    torch.cuda.current_stream().wait_stream(side)
    leaf.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts = mlk().router_balance_loss(leaf, ids)
        loss.backward()
    with torch.no_grad():
        leaf.copy_(other)
    for _ in range(2):
        graph.replay()
    want = mlk().router_balance_loss(leaf.detach(), ids, return_grad=True)
    assert torch.equal(loss.detach(), want[0]) and torch.equal(counts, want[1])
    # both forms sum in fp32 in orders of their own
    assert (leaf.grad - want[2]).abs().max() <= want[2].abs().max() * 2.0 ** -15


def test_unaligned_logits():
    require_gpu()
    x, ids, _, _ = inputs(31, 16, 2, "bf16", 6)
    buf = torch.empty(31 * 16 + 1, dtype=torch.bfloat16, device="cuda")
    view = buf[1:].view(31, 16)
    view.copy_(x)
    got = mlk().router_balance_loss(view, ids.cuda(), 0, 1.0, return_grad=True)
    check(got, x, ids, 0, 1.0, None, None)


def test_no_tokens():
    require_gpu()
    x, ids = torch.empty(0, 8, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda")
    loss, counts, grad = mlk().router_balance_loss(x, ids, return_grad=True)
    assert float(loss) == 0 and int(counts.sum()) == 0 and grad.shape == (0, 8)


@pytest.mark.parametrize("shape", [(1, 8, 2), (5000, 128, 8), (77, 60, 3)])
@pytest.mark.parametrize("masked", [False, True])
def test_expert_counts(shape, masked):
    require_gpu()
    T, E, topk = shape
    _, ids, mask, _ = inputs(T, E, topk, "fp32", 7, None, masked, foreign=True)
    got = mlk().expert_counts(ids.cuda(), E, None if mask is None else mask.cuda())
    rows = ids if mask is None else ids[mask]
    flat = rows[(rows >= 0) & (rows < E)].long()
    assert torch.equal(got.cpu().long(), torch.bincount(flat, minlength=E))
    assert int(mlk().expert_counts(torch.empty(0, 2, dtype=torch.int32, device="cuda"), E).sum()) == 0


@pytest.mark.parametrize("T", [40, 4000])
def test_graph_streams_and_repetition(T):
    """Captured and replayed with new inputs, on two streams at once, and bit for bit the same every time."""
    require_gpu()
    sets = [inputs(T, 64, 4, "fp32", s, [0, T // 3, T]) for s in range(3)]
    sets = [[t.cuda() for t in s if t is not None] for s in sets]
    call = lambda s: mlk().router_balance_loss(s[0], s[1], 0, 1.0, cu_seqlens=s[2], return_grad=True)  # noqa: E731
    want = [call(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append(call(s))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    hold = [t.clone() for t in sets[0]]
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(hold)
        graphs.append((g, out))
    for s, w in zip(sets, want):
        for h, t in zip(hold, s):
            h.copy_(t)
        torch.cuda.synchronize()
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(u, v) for u, v in zip(out, w))


def test_behind_the_router():
    """Used as it is meant to: the router picks, the loss counts what it picked, the gradient flows to the gate weights."""
    require_gpu()
    T, H, E, topk = 96, 64, 16, 2
    g = torch.Generator().manual_seed(1)
    h = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    gate = (0.2 * torch.randn(E, H, generator=g)).to(torch.bfloat16).cuda().requires_grad_()
    logits = h @ gate.t()
    ids = torch.empty(T, topk, dtype=torch.int32, device="cuda")
    w = torch.empty(T, topk, dtype=torch.bfloat16, device="cuda")
    mlk().fused_routing_gate(logits.detach(), 0, T, H, 1, 1, ids, w, topk)
    loss, counts = mlk().router_balance_loss(logits, ids, 0, 0.01)
    loss.backward()
    assert torch.equal(counts, mlk().expert_counts(ids, E))
    want, _, d = ob.balance(logits.detach().cpu(), ids.cpu(), 0, 0.01)
    assert abs(float(loss) - want) <= want * 2.0 ** -15
    ref = d.t() @ h.cpu().double()
    # bf16 gradient of the logits (half a step each) through one bf16 product
    mag = d.abs().t() @ h.cpu().double().abs()
    assert ((gate.grad.cpu().double() - ref).abs() <= mag * 2.0 ** -8 + ref.abs() * 2.0 ** -8).all()


def test_refusals_on_the_device():
    require_gpu()
    f = mlk().router_balance_loss
    x, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for a, kw in [((x.double(), ids), {}), ((x, ids.long()), {}), ((x[:, ::2], ids), {}), ((x, ids[:3]), {}), ((x, ids, 2), {}),
                  ((x, ids), dict(token_mask=torch.ones(5, dtype=torch.bool, device="cuda"))),
                  ((x, ids), dict(token_mask=torch.ones(4, device="cuda"))), ((x, ids), dict(token_mask=torch.ones(4, dtype=torch.bool))),
                  ((x, ids), dict(cu_seqlens=torch.zeros(1, dtype=torch.int32, device="cuda"))),
                  ((x, ids), dict(cu_seqlens=torch.zeros(3, dtype=torch.int64, device="cuda"))),
                  ((torch.zeros(4, 2048, device="cuda"), ids), {})]:
        with pytest.raises(RuntimeError):
            f(*a, **kw)
    with pytest.raises(RuntimeError):
        mlk().expert_counts(ids, 0)
    with pytest.raises(RuntimeError):
        mlk().expert_counts(ids.long(), 8)
