"""Expert router and balance loss against the formulas in 64 bits.

Tolerances.  Choices and counts are equal.  A weight is a quotient of exponentials (2 ulp each) of differences of logits: a difference d
is off by 2^-24 |d|, which the exponential turns into a relative error, and beyond |d| = 30 the weight itself is below 1e-13.  With the
sums (at most 32 + 5 additions) that is at most 96 * 2^-24 relative.  Gradients are products of at most four such factors with a
difference: 256 * 2^-24 of the sum of the absolute parts, plus half a step of their type.
"""
import math

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
REL, GRAD = 96 * 2.0 ** -24, 256 * 2.0 ** -24


def _logits(T, E, dt, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed + 1000 * T + E)
    return (torch.randn(T, E, generator=g) * scale).to(dt).cuda()


def _choice(order, K):
    """Indices of the K largest, ties to the lowest index, -1 where only -inf and NaN are left."""
    order = torch.where(order.isnan(), -math.inf, order)
    top = order.sort(dim=-1, descending=True, stable=True)
    return torch.where(top.values[:, :K] > -math.inf, top.indices[:, :K], -1)


def _reference(l, K, score, bias, renormalize, scale, valid):
    p = torch.softmax(torch.where((l == -math.inf).all(-1, keepdim=True), 0.0, l), -1) if score == "softmax" else torch.sigmoid(l)
    order = l if bias is None else torch.where(l == -math.inf, -math.inf, p + bias.double())
    idx = _choice(order.detach(), K)
    if valid is not None:
        idx = torch.where(valid[:, None], idx, -1)
    live = idx >= 0
    if renormalize:   # over the logarithms (up to a term common to the token), which do not underflow
        logs = l if score == "softmax" else torch.nn.functional.logsigmoid(l)
        c = torch.where(live, logs.gather(-1, idx.clamp(min=0)), -math.inf)
        c = torch.where(live.any(-1, keepdim=True), c, 0.0)
        w = torch.softmax(c, -1)
    else:
        w = p.gather(-1, idx.clamp(min=0))
    return idx, torch.where(live, w * scale, 0.0)


def _check_route(l, K, score="softmax", bias=None, renormalize=True, scale=1.0, valid=None, seed=0):
    from nvshmem_b200.ops import routing
    l = l.detach().requires_grad_(True)
    idx, w = routing.moe_route(l, K, score=score, bias=bias, renormalize=renormalize, scale=scale, valid=valid)
    dw = torch.randn(w.shape, generator=torch.Generator().manual_seed(seed)).cuda()
    (dl,) = torch.autograd.grad(w, l, dw)
    ld = l.detach().double().requires_grad_(True)
    ridx, rw = _reference(ld, K, score, bias, renormalize, scale, valid)
    assert idx.dtype == torch.int32 and torch.equal(idx.long(), ridx)
    assert ((w.double() - rw).abs() <= REL * rw.abs() + 1e-30).all(), (w.double() - rw).abs().max()
    (rdl,) = torch.autograd.grad(rw, ld, dw.double())
    # parts of a gradient: |w| (|dw| + sum |dw| |w|), on the chosen experts; for the full softmax p_e sum |dw| w elsewhere
    s = abs(scale) if scale else 1.0
    g = (dw.double().abs() * rw.detach().abs()).sum(-1, keepdim=True) / s
    part = torch.zeros_like(rdl).scatter_add_(-1, ridx.clamp(min=0), rw.detach().abs() * (dw.double().abs() + g))
    if score == "softmax" and not renormalize:
        part = part + torch.nan_to_num(torch.softmax(ld.detach(), -1)) * g * s
    # half the smallest subnormal step, several times over
    lim = part * GRAD + rdl.abs() * (torch.finfo(l.dtype).eps / 2) + torch.finfo(l.dtype).smallest_normal * torch.finfo(l.dtype).eps
    assert dl.dtype == l.dtype and ((dl.double() - rdl).abs() <= lim).all(), ((dl.double() - rdl).abs() / lim).max()
    again = routing.moe_route(l.detach(), K, score=score, bias=bias, renormalize=renormalize, scale=scale, valid=valid)
    assert torch.equal(again[0], idx) and torch.equal(again[1], w)
    return idx, w


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 2, 2), (5, 7, 3), (9, 31, 16), (8, 32, 4), (33, 33, 1), (64, 100, 8), (17, 128, 6), (100, 255, 9), (61, 256, 8), (7, 300, 10),
                                   (12, 513, 16), (3, 1024, 16), (2050, 64, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_sizes(T, E, K, score, renormalize):
    _check_route(_logits(T, E, F32), K, score, renormalize=renormalize, scale=2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("E", [40, 256, 700])
def test_route_with_bias_mask_and_types(dt, score, renormalize, E):
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E)).cuda() * 0.1
    valid = torch.rand(77, generator=torch.Generator().manual_seed(1)).cuda() > 0.3
    _check_route(_logits(77, E, dt), 5, score, bias, renormalize, 1.0, valid)
    _check_route(_logits(77, E, dt), 5, score, None, renormalize, 1.0, valid)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
def test_ties_go_to_the_lowest_expert(bias):
    from nvshmem_b200.ops import routing
    l = torch.zeros(4, 200, device="cuda")
    l[1, 100:] = 1.0
    l[2] = torch.arange(200, device="cuda") % 3
    l[3, ::2] = -0.0   # equal to 0
    b = torch.zeros(200, device="cuda") if bias else None
    idx, w = routing.moe_route(l, 4, bias=b)
    assert idx.tolist() == [[0, 1, 2, 3], [100, 101, 102, 103], [2, 5, 8, 11], [0, 1, 2, 3]]
    assert torch.equal(w, torch.full_like(w, 0.25))


@pytest.mark.gpu
@pytest.mark.parametrize("E", [24, 256, 1000])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_that_32_bits_do_not_tell_apart(E, score):
    """Score + bias of neighbouring experts differ by 1e-9 to 1e-6, in shuffled order: the choice is that of 64 bits."""
    from nvshmem_b200.ops import routing
    g = torch.Generator().manual_seed(E)
    l = torch.randn(60, E, generator=g)
    p = (torch.softmax(l.double(), -1) if score == "softmax" else torch.sigmoid(l.double()))[0]
    l = l[:1] + torch.zeros(60, 1)
    l[30:] += torch.randn(30, 1, generator=g) if score == "softmax" else 0.0
    gap = torch.rand(E, generator=g).double() * 3 - 9
    bias = (0.9 - p + torch.randperm(E, generator=g).double() * 10 ** gap).float()
    _check_route(l.cuda(), min(E, 16), score, bias.cuda())


@pytest.mark.gpu
def test_biased_softmax_of_bad_logits():
    from nvshmem_b200.ops import routing
    l, b = _logits(3, 20, F32), torch.zeros(20, device="cuda")
    clean = routing.moe_route(l, 3, bias=b)
    l[1, 4], l[2, 6] = float("nan"), math.inf
    idx, w = routing.moe_route(l, 3, bias=b)
    assert torch.equal(idx[0], clean[0][0]) and torch.equal(w[0], clean[1][0]) and w[1:].isnan().all()
    assert not (idx[1] == 4).any()


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renormalize", [True, False])
def test_masked_experts_and_extreme_logits(score, bias, renormalize):
    l = _logits(8, 48, F32)
    inf = math.inf
    l[0, 5:] = -inf                                # five experts left
    l[1] = -inf                                    # none
    l[2, 3:] = -inf                                # fewer than K
    l[3] = torch.finfo(F32).min                    # the lowest value is a number like any other
    l[4] -= 300.0                                  # every sigmoid underflows in 32 bits
    l[5] += 60.0
    l[6, ::2] = torch.finfo(F32).min
    b = torch.linspace(-0.2, 0.2, 48, device="cuda") if bias else None
    rows = [0, 1, 2, 3, 5, 6, 7] if score == "sigmoid" and renormalize else range(8)
    if score == "sigmoid" and renormalize:         # the reference's softmax over log-sigmoids holds for row 3 as well
        rows = range(8)
    idx, w = _check_route(l[list(rows)], 5, score, b, renormalize)
    assert (idx[1] == -1).all() and not w[1].any() and idx[2].tolist().count(-1) == 2


@pytest.mark.gpu
def test_nan_and_infinite_logits():
    from nvshmem_b200.ops import routing
    l = _logits(4, 20, F32)
    clean = routing.moe_route(l, 3)
    l[1, 4], l[2, 6] = float("nan"), math.inf
    x = l.clone().requires_grad_(True)
    idx, w = routing.moe_route(x, 3)
    assert not (idx[1] == 4).any() and w[1].isnan().all()
    assert idx[2, 0] == 6 and w[2].isnan().all()
    (g,) = torch.autograd.grad(w, x, torch.ones_like(w))
    for i in (0, 3):
        assert torch.equal(idx[i], clean[0][i]) and torch.equal(w[i], clean[1][i]) and g[i].isfinite().all()
    assert g[1].isnan().any()
    idx, w = routing.moe_route(l, 3, score="sigmoid")
    assert not (idx[1] == 4).any() and w.isfinite().all() and idx[2, 0] == 6


@pytest.mark.gpu
def test_strided_logits_and_expanded_gradient():
    from nvshmem_b200.ops import routing
    wide = _logits(30, 101, F32).requires_grad_(True)
    idx, w = routing.moe_route(wide[:, 3:99], 4, renormalize=False)
    (g,) = torch.autograd.grad(w.sum(), wide)
    ref = wide.detach().double().requires_grad_(True)
    ridx, rw = _reference(ref[:, 3:99], 4, "softmax", None, False, 1.0, None)
    (rg,) = torch.autograd.grad(rw.sum(), ref)
    assert torch.equal(idx.long(), ridx) and ((g.double() - rg).abs() <= GRAD * 2).all()
    columns = routing.moe_route(wide.detach().t().contiguous().t()[:, 3:99], 4, renormalize=False)   # experts outermost
    assert torch.equal(columns[0], idx) and torch.equal(columns[1], w)


def _balance_reference(l, idx, score, valid):
    T, E = l.shape
    p = torch.softmax(l if score == "softmax" else torch.nn.functional.logsigmoid(l), -1)
    p = torch.where((l == -math.inf).all(-1, keepdim=True), 0.0, p)
    rows = torch.arange(T, device=l.device) if valid is None else valid.nonzero()[:, 0]
    ids = idx[rows].long().flatten()
    counts = torch.bincount(ids[(ids >= 0) & (ids < E)], minlength=E)
    n = max(1, rows.numel())
    return E * (counts.double() / (n * idx.shape[1]) @ p[rows].sum(0)) / n, counts, p


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 8, 2), (5, 7, 3), (61, 40, 3), (100, 256, 8), (3000, 64, 6), (4099, 256, 8), (50, 1000, 16)])
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("mask", [False, True])
def test_balance_loss(T, E, K, dt, score, mask):
    """The loss is a sum of T E positive products, added at most 64 deep per thread, CTA and slice: 128 * 2^-24 relative."""
    from nvshmem_b200.ops import routing
    l = _logits(T, E, dt).requires_grad_(True)
    g = torch.Generator().manual_seed(T)
    idx = torch.rand(T, E, generator=g).argsort(-1)[:, :K].to(torch.int32)
    idx[0, 0] = -1
    idx = idx.cuda()
    valid = torch.rand(T, generator=g).cuda() > 0.25 if mask else None
    loss, counts = routing.balance_loss(l, idx, score=score, valid=valid)
    (dl,) = torch.autograd.grad(loss, l, torch.tensor(0.3, device="cuda"))
    ld = l.detach().double().requires_grad_(True)
    rloss, rcounts, p = _balance_reference(ld, idx, score, valid)
    (rdl,) = torch.autograd.grad(rloss, ld, torch.tensor(0.3, device="cuda").double())
    assert counts.dtype == torch.int32 and torch.equal(counts.long(), rcounts)
    assert abs(loss.double() - rloss) <= 128 * 2.0 ** -24 * rloss
    n = max(1, int(valid.sum()) if mask else T)
    c = 0.3 * E * rcounts.double() / (n * n * K)
    lim = GRAD * p.detach() * (c + (p.detach() * c).sum(-1, keepdim=True)) + rdl.abs() * (torch.finfo(dt).eps / 2) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert dl.dtype == dt and ((dl.double() - rdl).abs() <= lim).all()
    if mask:
        assert not dl[~valid].any()
    with torch.no_grad():
        again = routing.balance_loss(l, idx, score=score, valid=valid)
    assert torch.equal(again[0], loss) and torch.equal(again[1], counts)


@pytest.mark.gpu
def test_balance_of_masked_rows_and_empty_batches():
    from nvshmem_b200.ops import routing
    l = _logits(6, 10, F32)
    l[2] = -math.inf
    l[3, 4:] = -math.inf
    x = l.clone().requires_grad_(True)
    idx = torch.arange(12, dtype=torch.int32, device="cuda").view(6, 2) % 10
    idx[5] = torch.tensor([10, -7])       # outside: skipped
    for score in ("softmax", "sigmoid"):
        loss, counts = routing.balance_loss(x, idx, score=score)
        (g,) = torch.autograd.grad(loss, x)
        want, wcounts, _ = _balance_reference(l.double(), idx, score, None)
        assert torch.equal(counts.long(), wcounts) and abs(loss.double() - want) <= 128 * 2.0 ** -24 * want
        assert g.isfinite().all() and not g[2].any() and not g[3, 4:].any()
    none = torch.zeros(6, dtype=torch.bool, device="cuda")
    loss, counts = routing.balance_loss(x, idx, valid=none)
    (g,) = torch.autograd.grad(loss, x)
    assert loss.item() == 0 and not counts.any() and not g.any()
    e = torch.zeros(0, 10, device="cuda", requires_grad=True)
    loss, counts = routing.balance_loss(e, idx[:0])
    assert loss.item() == 0 and not counts.any() and torch.autograd.grad(loss, e)[0].shape == (0, 10)
    i0, w0 = routing.moe_route(e, 2)
    assert i0.shape == w0.shape == (0, 2) and torch.autograd.grad(w0.sum(), e)[0].shape == (0, 10)


@pytest.mark.gpu
def test_gradients_agree_with_differences():
    """Central differences of the fp32 losses with a step of 2^-5 along a random direction of norm 1: 2^-10 / 6 of the third
    derivative (below 4 for these functions) and 2^-24 * 2^5 * 8 of rounding: below 2^-10."""
    from nvshmem_b200.ops import routing
    l = _logits(5, 12, F32, seed=3)
    idx, _ = routing.moe_route(l, 3)
    dw = torch.randn(5, 3, generator=torch.Generator().manual_seed(2)).cuda()
    losses = [lambda t, s=s, r=r: (routing.moe_route(t, 3, score=s, renormalize=r)[1].double() * dw).sum() for s in ("softmax", "sigmoid") for r in (True, False)]
    losses += [lambda t, s=s: routing.balance_loss(t, idx, score=s)[0].double() for s in ("softmax", "sigmoid")]
    gen = torch.Generator().manual_seed(4)
    for f in losses:
        x = l.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(x), x)
        d = torch.randn(l.shape, generator=gen).cuda()
        d = d / d.norm() * 2.0 ** -5
        assert torch.equal(routing.moe_route(l + d, 3)[0], idx) and torch.equal(routing.moe_route(l - d, 3)[0], idx)
        diff = (f(l + d) - f(l - d)) / 2 * 2.0 ** 5
        assert abs(diff - (g.double() * d.double()).sum() * 2.0 ** 5) <= 2.0 ** -10


def test_refusals():
    from nvshmem_b200.ops import routing
    from nvshmem_b200.ops.routing import RoutingError
    l, idx = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int32)
    bad = [lambda: routing.moe_route(l[0], 2), lambda: routing.moe_route(l.double(), 2), lambda: routing.moe_route(l, 0), lambda: routing.moe_route(l, 17),
           lambda: routing.moe_route(torch.zeros(2, 40), 17), lambda: routing.moe_route(torch.zeros(2, 1025), 2), lambda: routing.moe_route(torch.zeros(2, 0), 1),
           lambda: routing.moe_route(l, 2, score="tanh"), lambda: routing.moe_route(l, 2, bias=torch.zeros(15)), lambda: routing.moe_route(l, 2, bias=torch.zeros(16).half()),
           lambda: routing.moe_route(l, 2, valid=torch.ones(4)), lambda: routing.moe_route(l, 2, valid=torch.ones(3, dtype=torch.bool)),
           lambda: routing.balance_loss(l, idx.long()), lambda: routing.balance_loss(l, idx[:3]), lambda: routing.balance_loss(l, idx[0]),
           lambda: routing.balance_loss(l, idx[:, :0]), lambda: routing.balance_loss(l, idx), lambda: routing.moe_route(l, 2)]  # the last two: not on a GPU
    for call in bad:
        with pytest.raises(RoutingError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E, K", [(100, 8), (256, 8), (256, 16), (384, 8), (512, 1), (1000, 16), (1024, 6)])
def test_where_the_largest_lie(E, K, dt):
    """The largest logits in a few columns modulo 32, in the first and the last columns, few finite ones, many equal ones: the order is that of a stable sort."""
    from nvshmem_b200.ops import moe_route
    g = torch.Generator().manual_seed(E + K)
    e = torch.arange(E)
    rows = [torch.randn(E, generator=g) + 10.0 * (e % 32 < n) for n in (1, 2, 4, 5, 8, 31)]
    rows += [torch.randn(E, generator=g) + 10.0 * (e % 32 == E % 32), torch.randn(E, generator=g) + 10.0 * (e < 40), torch.randn(E, generator=g) + 10.0 * (e >= E - 3)]
    rows += [torch.randn(E, generator=g).masked_fill(e % 32 >= n, -float("inf")) for n in (1, 2, 3, 9)]
    rows += [torch.randn(E, generator=g).masked_fill(torch.randperm(E, generator=g) >= n, -float("inf")) for n in (0, 1, K - 1, K, K + 1, 40)]
    rows += [torch.zeros(E), (e % 2).float(), (e // 32).float(), -(e // 32).float(), torch.randint(0, 3, (E,), generator=g).float(), torch.randint(0, 40, (E,), generator=g).float()]
    logits = torch.stack(rows).to(dt).cuda()
    for bias in (None, torch.zeros(E, device="cuda")):   # a bias orders by the sigmoids, where logits from 37 on are equal
        _check_route(logits, K, score="sigmoid", bias=bias)


def _bad_rows(E, spread):
    """Rows with a NaN or +inf among logits that lie `spread` apart, in shuffled order, and a last row without."""
    g = torch.Generator().manual_seed(E)
    l = torch.stack([torch.randperm(E, generator=g) * spread for _ in range(6)]).float()
    l[0, 3], l[1, E - 1], l[1, 0] = float("nan"), float("nan"), float("nan")
    l[2, 5] = math.inf
    l[3, 7], l[3, 2], l[3, 4] = math.inf, math.inf, float("nan")
    l[4, 6], l[4, ::2] = float("nan"), -math.inf
    return l


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [1e-7, 1e-5, 1e-2, 0.5])   # in 64 bits throughout, in 32 bits throughout, and between
@pytest.mark.parametrize("E,K", [(20, 3), (40, 16), (300, 8), (1000, 16)])
@pytest.mark.parametrize("bias", [0.0, 1e-6, 0.1])
def test_biased_choice_beside_bad_logits(E, K, spread, bias):
    """Softmax + bias orders the logits that are numbers, whatever decides between them: NaN are left out, +inf share the softmax."""
    from nvshmem_b200.ops import routing
    l = _bad_rows(E, spread)
    b = torch.randn(E, generator=torch.Generator().manual_seed(1)) * bias
    d = l.double()
    top = torch.where(d.isnan(), -math.inf, d).amax(-1, keepdim=True)
    e = torch.where(d == top, 1.0, torch.exp(d - top))
    p = torch.where(d.isnan(), 0.0, e)
    p = p / p.sum(-1, keepdim=True)
    order = torch.where(d.isnan() | (d == -math.inf), -math.inf, p + b.double())
    bad = (d.isnan() | (d == math.inf)).any(-1)   # not the last two: the NaN of the fifth row is among those it then sets to -inf
    for renormalize in (True, False):
        idx, w = routing.moe_route(l.cuda(), K, bias=b.cuda(), renormalize=renormalize)
        want = _choice(order, K)
        assert torch.equal(idx.cpu().long(), want)
        w = w.cpu()
        assert w[bad][want[bad] >= 0].isnan().all() and not w[want < 0].any() and w[~bad].isfinite().all()


@pytest.mark.gpu
def test_places_left_over_beside_bad_logits():
    from nvshmem_b200.ops import routing
    l = torch.full((2, 40), -math.inf, device="cuda")
    l[0, 3], l[0, 9], l[1, 2], l[1, 4] = 1.0, float("nan"), math.inf, 0.0
    for renormalize in (True, False):
        idx, w = routing.moe_route(l, 4, renormalize=renormalize)
        assert idx.tolist() == [[3, -1, -1, -1], [2, 4, -1, -1]]
        assert w[0, 0].isnan() and w[1, :2].isnan().all() and not w[idx < 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("E,K", [(24, 8), (64, 6), (256, 8), (256, 16), (1024, 8)])
@pytest.mark.parametrize("std,mean", [(0.02, 0.0), (0.1, 0.0), (1.5, 0.0), (10.0, 0.0), (30.0, 0.0), (1.5, -12.0), (3.0, -80.0)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_biased_choice_of_narrow_and_peaked_scores(E, K, std, mean, score):
    """Scores of any size against a bias of any size, among them biases that bring experts of very different scores together: the choice is
    that of 64 bits.  (Sums of score and bias that 64 bits do not tell apart by 2^-44 are left out.)"""
    from nvshmem_b200.ops import routing
    g = torch.Generator().manual_seed(E + K)
    l = (torch.randn(400, E, generator=g) * std + mean).cuda()
    d = l.double()
    p = torch.softmax(d, -1) if score == "softmax" else torch.sigmoid(d)
    size = p.mean().item()
    meet = (p[0].max() - p[0]).float() + torch.rand(E, generator=g).cuda() * p[0].max().float() * 1e-4
    for b in (torch.zeros(E, device="cuda"), torch.randn(E, generator=g).cuda() * size, torch.randn(E, generator=g).cuda() * size * 1e-4,
              torch.randn(E, generator=g).cuda() * 0.1, meet, -meet):
        order = p + b.double()
        top = order.sort(-1, descending=True).values[:, :K + 1]
        clear = ((top[:, :-1] - top[:, 1:]) > 2.0 ** -44 * top[:, :-1].abs()).all(-1)
        idx, _ = routing.moe_route(l, K, score=score, bias=b)
        assert torch.equal(idx.long()[clear], _choice(order, K)[clear])


@pytest.mark.gpu
def test_narrow_scores_take_no_longer():
    """The choice goes to 64 bits for a few tokens only, however narrow or peaked the softmax is: within twice the time of wide scores (all tokens in
    64 bits take several times as long).  The best of ten runs of twenty calls each."""
    from nvshmem_b200.ops import routing
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(8192, 256, generator=g, device="cuda")
    bias = torch.zeros(256, device="cuda")

    def time():
        best = math.inf
        for _ in range(10):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    x = z.clone()
    routing.moe_route(x, 8, bias=bias)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            routing.moe_route(x, 8, bias=bias)
    times = {}
    for std in (1.5, 0.02, 0.1, 10.0):
        x.copy_(z * std)
        times[std] = time()
    assert max(times.values()) <= 2 * times[1.5], times
