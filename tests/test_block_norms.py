"""The norms around a block against the formulas in 64 bits.

Tolerances.  Every result is a sum of products whose factors carry at most 16 roundings to fp32 and whose sums are at most 48 additions
deep (16 values of a thread, 5 + 5 steps across a group, then rows of one CTA and the CTAs' parts), so it is off by at most
64 * 2^-24 of the sum of the absolute products (`mag` below), plus half a step of its own type relative to the value.
"""
import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEEP = 64 * 2.0 ** -24


def _norm_inputs(T, H, dt, rt, wt, gate, post=True, pre=True, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed + T * 131 + H)
    rn = lambda *s, scale=1.0, shift=0.0: torch.randn(*s, generator=g) * scale + shift
    d = {"h": rn(T, H, scale=0.5).to(dt), "residual": rn(T, H, scale=2.0).to(rt), "dr": rn(T, H).to(rt), "dy": rn(T, H).to(dt)}
    d["post"] = rn(H, scale=0.2, shift=1.0).to(wt) if post else None
    d["pre"] = rn(H, scale=0.2, shift=1.0).to(wt) if pre else None
    shape = {"channel": (H,), "token": (T, 1), "full": (T, H)}.get(gate)
    d["gate"] = rn(*shape, scale=0.3, shift=0.4).to(wt) if shape else None
    return {k: None if v is None else v.to(device) for k, v in d.items()}


def _reference(d, a, b, eps, off, backward=True):
    """Values and sums of absolute products in fp64."""
    v = {k: None if t is None else t.detach().double() for k, t in d.items()}
    H = v["residual"].shape[1]
    one = torch.ones((), dtype=torch.float64, device=v["residual"].device)
    mean = lambda t: t.mean(-1, keepdim=True)
    out, mag = {}, {}
    if v["h"] is not None:
        s1 = torch.rsqrt(mean(v["h"] ** 2) + eps) if v["post"] is not None else one
        w = v["post"] + off if v["post"] is not None else one
        gate = v["gate"] if v["gate"] is not None else one
        z = v["h"] * s1 * w
        branch = b * gate * z
    else:
        branch = torch.zeros_like(v["residual"])
    r = a * v["residual"] + branch
    rm = (a * v["residual"]).abs() + branch.abs()
    out["r"], mag["r"] = r, rm
    if v["pre"] is not None:
        s2, wp = torch.rsqrt(mean(r ** 2) + eps), v["pre"] + off
        out["y"], mag["y"] = r * s2 * wp, rm * s2 * wp.abs() * (1 + mean(rm * r.abs()) * s2 ** 2)
    if not backward:
        return out, mag
    G, Gm = v["dr"], v["dr"].abs()
    if v["pre"] is not None:
        rh, rhm = r * s2, rm * s2 * (1 + mean(rm * r.abs()) * s2 ** 2)
        dyw = v["dy"] * wp
        c1, c1m = mean(dyw * rh), mean(dyw.abs() * rhm)
        A, Am = v["dr"] + s2 * dyw, v["dr"].abs() + s2 * dyw.abs()
        G, Gm = A - s2 * rh * c1, Am + s2 * (rhm * c1m)
        out["d_pre"], mag["d_pre"] = (v["dy"] * rh).sum(0), (v["dy"].abs() * rhm).sum(0)
    else:
        A, Am = G, Gm
    out["d_residual"], mag["d_residual"] = a * G, abs(a) * Gm
    if v["h"] is None:
        return out, mag
    hh = v["h"] * s1
    dz, dzm = b * gate * G, (b * gate).abs() * Gm
    if v["post"] is not None:
        q = (b * gate * z).abs()
        c2m = mean(q * Am) + (c1m * mean(q * s2 * rhm) if v["pre"] is not None else 0.0)
        out["d_h"], mag["d_h"] = s1 * (dz * w - hh * mean(dz * w * hh)), s1 * (dzm * w.abs() + hh.abs() * c2m)
        out["d_post"], mag["d_post"] = (dz * hh).sum(0), (dzm * hh.abs()).sum(0)
    else:
        out["d_h"], mag["d_h"] = dz, dzm
    if v["gate"] is not None:
        dg, dgm = b * G * z, (b * z).abs() * Gm
        if v["gate"].shape == v["h"].shape and v["gate"].shape[1] > 1:
            out["d_gate"], mag["d_gate"] = dg, dgm
        elif v["gate"].dim() == 1:
            out["d_gate"], mag["d_gate"] = dg.sum(0), dgm.sum(0)
        else:
            zq = (b * z).abs()
            out["d_gate"] = dg.sum(1, keepdim=True)
            mag["d_gate"] = (zq * Am).sum(1, keepdim=True) + (H * c1m * mean(zq * s2 * rhm) if v["pre"] is not None else 0.0)
    return out, mag


def _compare(got, want, mag, what):
    t = got.dtype
    lim = want.abs() * (torch.finfo(t).eps / 2) + mag * DEEP + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    bad = (got.double() - want).abs() > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / lim).max().item():.3g} of the tolerance"


def _check(d, a=0.75, b=1.25, eps=1e-6, off=0.0):
    from nvshmem_b200.ops import norms
    names = [n for n in ("h", "residual", "post", "pre", "gate") if d[n] is not None]
    for n in names:
        d[n] = d[n].detach().requires_grad_(True)
    r, y = norms.block_norms(d["h"], d["residual"], post_weight=d["post"], pre_weight=d["pre"], gate=d["gate"], residual_scale=a, branch_scale=b, eps=eps,
                             weight_offset=off)
    outs, grads = ([r], [d["dr"]]) if y is None else ([r, y], [d["dr"], d["dy"]])
    got = dict(zip(("d_" + n for n in names), torch.autograd.grad(outs, [d[n] for n in names], grads)))
    got["r"] = r.detach()
    if y is not None:
        got["y"] = y.detach()
    want, mag = _reference(d, a, b, eps, off)
    assert set(got) == set(want)
    for k in sorted(got):
        assert got[k].dtype == {"d_h": d["h"].dtype, "y": d["h"].dtype, "r": d["residual"].dtype, "d_residual": d["residual"].dtype}.get(k, got[k].dtype)
        _compare(got[k], want[k].reshape(got[k].shape), mag[k].expand_as(want[k]).reshape(got[k].shape), k)
    with torch.no_grad():
        r2, y2 = norms.block_norms(d["h"], d["residual"], post_weight=d["post"], pre_weight=d["pre"], gate=d["gate"], residual_scale=a, branch_scale=b, eps=eps,
                                   weight_offset=off)
    assert torch.equal(r2, r) and (y is None or torch.equal(y2, y))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(1, 1), (1, 8), (3, 7), (5, 64), (9, 255), (33, 256), (130, 520), (7, 1001), (300, 2048), (17, 4104), (40, 8192), (3, 8200),
                                 (2, 16383), (5, 16384)])
@pytest.mark.parametrize("dt,rt,wt", [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F32, F32, F32)])
def test_sizes_and_types(T, H, dt, rt, wt):
    _check(_norm_inputs(T, H, dt, rt, wt, "channel"))


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T,H,dt,rt,wt", [(19, 640, BF16, F32, BF16), (6, 333, F16, F32, F16)])
def test_gates_and_missing_norms(gate, post, pre, T, H, dt, rt, wt):
    _check(_norm_inputs(T, H, dt, rt, wt, gate, post, pre), off=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(700, 1024), (1500, 96), (400, 8192)])
def test_more_rows_than_ctas(T, H):
    _check(_norm_inputs(T, H, BF16, BF16, BF16, "channel"))


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T,H,dt,rt,wt", [(320, 1032, BF16, F32, BF16), (700, 2048, F16, F16, F32), (301, 4104, F32, F32, F32), (1300, 2048, BF16, BF16, BF16),
                                          (420, 8192, BF16, F32, F32), (1250, 1024, F32, F32, F32)])
def test_many_rows(gate, post, pre, T, H, dt, rt, wt):
    """More rows than the SMs take at once, which walk them through a ring in shared memory."""
    _check(_norm_inputs(T, H, dt, rt, wt, gate, post, pre), off=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("gate,post,pre", [("channel", True, True), ("token", True, False), ("full", True, True), ("none", False, True)])
@pytest.mark.parametrize("T,H", [(160, 16384), (300, 8200), (90, 9216)])
def test_many_long_rows(gate, post, pre, T, H):
    """Above 8192 columns a pair of CTAs takes half a row each."""
    _check(_norm_inputs(T, H, BF16, BF16, F32, gate, post, pre))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(900, 1024), (1201, 1536), (640, 3000), (310, 5128), (333, 7168), (2000, 4096), (500, 8184)])
@pytest.mark.parametrize("dt,rt,wt", [(BF16, BF16, BF16), (BF16, F32, F32)])
def test_many_rows_sizes(T, H, dt, rt, wt):
    _check(_norm_inputs(T, H, dt, rt, wt, "channel"))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("T,H", [(1, 128), (77, 1000), (260, 7168), (400, 1024), (1000, 7168), (1400, 1024), (160, 16384), (700, 16384), (3000, 2048)])
def test_rms_norm(T, H, dt, wt):
    from nvshmem_b200.ops import norms
    d = _norm_inputs(T, H, dt, dt, wt, "none")
    x, w = d["residual"].requires_grad_(True), d["pre"].requires_grad_(True)
    y = norms.rms_norm(x, w, eps=1e-5, weight_offset=0.5)
    dx, dw = torch.autograd.grad(y, [x, w], d["dy"])
    ref = {"h": None, "residual": x, "pre": w, "post": None, "gate": None, "dy": d["dy"], "dr": torch.zeros_like(x)}
    want, mag = _reference(ref, 1.0, 1.0, 1e-5, 0.5)
    _compare(y.detach(), want["y"], mag["y"], "y")
    _compare(dx, want["d_residual"], mag["d_residual"], "dx")
    _compare(dw, want["d_pre"], mag["d_pre"], "dw")


@pytest.mark.gpu
def test_strided_rows_and_broadcast_gradients():
    """Rows of a wider buffer at odd offsets, gradients that are expanded, a gate expanded over channels."""
    from nvshmem_b200.ops import norms
    d = _norm_inputs(12, 200, BF16, F32, BF16, "none")
    wide_h, wide_r = torch.zeros(12, 413, dtype=BF16, device="cuda"), torch.zeros(12, 301, device="cuda")
    wide_h[:, 5:205], wide_r[:, 101:301] = d["h"], d["residual"]
    gate = (torch.rand(12, 1, device="cuda") + 0.5).to(BF16).requires_grad_(True)
    h, res = wide_h.requires_grad_(True), wide_r.requires_grad_(True)
    r, y = norms.block_norms(h[:, 5:205], res[:, 101:301], d["post"], d["pre"], gate.expand(12, 200))
    gh, gr, gg = torch.autograd.grad([r.sum() + y.sum()], [h, res, gate])
    ref = {**d, "gate": gate.detach().expand(12, 200), "dr": torch.ones_like(d["dr"]), "dy": torch.ones_like(d["dy"])}
    want, mag = _reference(ref, 1.0, 1.0, 1e-6, 0.0)
    _compare(r.detach(), want["r"], mag["r"], "r")
    _compare(gh[:, 5:205], want["d_h"], mag["d_h"], "d_h")
    _compare(gr[:, 101:301], want["d_residual"], mag["d_residual"], "d_residual")
    assert not gh[:, :5].any() and not gh[:, 205:].any() and not gr[:, :101].any()
    # the gate's gradient: 200 bf16 values, each off by half a step, summed by torch in fp32 and rounded once more
    lim = mag["d_gate"].sum(1, keepdim=True) * (DEEP + 2.0 ** -8) + want["d_gate"].sum(1, keepdim=True).abs() * 2.0 ** -8
    assert ((gg.double() - want["d_gate"].sum(1, keepdim=True)).abs() <= lim).all()


@pytest.mark.gpu
def test_only_some_gradients_are_asked_for():
    from nvshmem_b200.ops import norms
    d = _norm_inputs(50, 512, BF16, BF16, BF16, "channel")
    want, mag = _reference(d, 1.0, 1.0, 1e-6, 0.0)
    for name in ("h", "residual", "post", "pre", "gate"):
        t = {n: d[n].clone() for n in ("h", "residual", "post", "pre", "gate")}
        t[name].requires_grad_(True)
        r, y = norms.block_norms(t["h"], t["residual"], t["post"], t["pre"], t["gate"])
        (g,) = torch.autograd.grad([r, y], [t[name]], [d["dr"], d["dy"]])
        _compare(g, want["d_" + name], mag["d_" + name], name)
    # one of the two outputs unused
    t = {n: d[n].clone().requires_grad_(True) for n in ("h", "residual", "post", "pre", "gate")}
    r, y = norms.block_norms(t["h"], t["residual"], t["post"], t["pre"], t["gate"])
    for out, zero, grad in ((r, "dy", d["dr"]), (y, "dr", d["dy"])):
        grads = torch.autograd.grad(out, list(t.values()), grad, retain_graph=True, allow_unused=True)
        want, mag = _reference({**d, zero: torch.zeros_like(d[zero])}, 1.0, 1.0, 1e-6, 0.0)
        for name, g in zip(t, grads):
            _compare(g, want["d_" + name], mag["d_" + name], name)


@pytest.mark.gpu
def test_gradient_agrees_with_differences():
    """Directional differences of the fp32 forward: f is about 1 a value, so with a step of 2^-6 the rounding adds 2^-24 * 2^6 a
    value, random over 96 values, and the cubic term 2^-12 / 6 of a third derivative of order 1: together below 2^-10 of the sum."""
    from nvshmem_b200.ops import norms
    d = _norm_inputs(3, 32, F32, F32, F32, "full", seed=5)
    names = ("h", "residual", "post", "pre", "gate")
    leaves = [d[n].requires_grad_(True) for n in names]

    def f(h, residual, post, pre, gate):
        r, y = norms.block_norms(h, residual, post, pre, gate, residual_scale=0.5, branch_scale=2.0)
        return (r.double() * d["dr"]).sum() + (y.double() * d["dy"]).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(len(leaves)):
        step = torch.randn(leaves[i].shape, generator=gen, device="cuda")
        step = step / step.norm() * 2.0 ** -6
        with torch.no_grad():
            diff = (f(*[l + (step if j == i else 0) for j, l in enumerate(leaves)]) - f(*[l - (step if j == i else 0) for j, l in enumerate(leaves)])) / 2
        want = (grads[i].double() * step.double()).sum()
        assert abs(diff - want) <= 2.0 ** -10 * (grads[i].double() * step.double()).abs().sum() + 2.0 ** -18, names[i]


@pytest.mark.gpu
def test_rows_of_zeros_and_bad_rows_stay_apart():
    """A row of zeros gives zeros; infinities and NaN stay in their rows."""
    from nvshmem_b200.ops import norms
    d = _norm_inputs(6, 300, BF16, BF16, BF16, "channel")
    good = norms.block_norms(d["h"], d["residual"], d["post"], d["pre"], d["gate"])
    d["h"][1], d["residual"][1] = 0, 0
    d["h"][3, 7], d["residual"][4, 0] = float("nan"), float("inf")
    r, y = norms.block_norms(d["h"], d["residual"], d["post"], d["pre"], d["gate"])
    assert not r[1].any() and not y[1].any()
    assert r[3].isnan().all() and y[4].isnan().any()
    for i in (0, 2, 5):
        assert torch.equal(r[i], good[0][i]) and torch.equal(y[i], good[1][i])


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused():
    """A graph of the gradients may be asked for, but not gone through."""
    from nvshmem_b200.ops import moe_route, rms_norm
    x, w = torch.randn(5, 64, device="cuda", requires_grad=True), torch.ones(64, device="cuda")
    for out in (rms_norm(x, w), moe_route(x, 4)[1]):
        (plain,) = torch.autograd.grad(out.sum(), x, retain_graph=True)
        (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)


@pytest.mark.gpu
def test_tiny_rows_without_eps():
    """Values of 1e-13 with eps = 0: nothing between overflows."""
    d = _norm_inputs(20, 1024, F32, F32, F32, "channel")
    for k in ("h", "residual"):
        d[k] = d[k] * 1e-13
    from nvshmem_b200.ops import norms
    leaves = [d[n].requires_grad_(True) for n in ("h", "residual", "post", "pre", "gate")]
    r, y = norms.block_norms(*leaves, branch_scale=1e-13, eps=0.0)
    grads = torch.autograd.grad([r, y], leaves, [d["dr"] * 1e13, d["dy"]])
    want, mag = _reference({**d, "dr": d["dr"] * 1e13}, 1.0, 1e-13, 0.0, 0.0)
    _compare(y.detach(), want["y"], mag["y"], "y")
    for n, g in zip(("h", "residual", "post", "pre", "gate"), grads):
        assert g.isfinite().all()
        _compare(g, want["d_" + n], mag["d_" + n], n)


@pytest.mark.gpu
def test_no_rows():
    from nvshmem_b200.ops import norms
    d = _norm_inputs(0, 64, BF16, BF16, BF16, "channel")
    leaves = [d[n].requires_grad_(True) for n in ("h", "residual", "post", "pre", "gate")]
    r, y = norms.block_norms(*leaves)
    grads = torch.autograd.grad(r.sum() + y.sum(), leaves)
    assert r.shape == y.shape == (0, 64) and all(not g.any() for g in grads)


def test_refusals():
    from nvshmem_b200.ops import norms
    from nvshmem_b200.ops.norms import NormError
    h, w = torch.zeros(4, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    bad = [lambda: norms.rms_norm(h[0], w), lambda: norms.rms_norm(h.int(), w), lambda: norms.rms_norm(h, w[:32]), lambda: norms.rms_norm(h, w.half()),
           lambda: norms.rms_norm(h, None), lambda: norms.rms_norm(torch.zeros(2, 16385, dtype=BF16), torch.ones(16385, dtype=BF16)),
           lambda: norms.rms_norm(torch.zeros(2, 0, dtype=BF16), torch.ones(0, dtype=BF16)),
           lambda: norms.block_norms(h, h[:3]), lambda: norms.block_norms(h, h.half()), lambda: norms.block_norms(h.float(), h),
           lambda: norms.block_norms(h, h, w, w.float()), lambda: norms.block_norms(h, h, w, gate=torch.ones(4, dtype=BF16)),
           lambda: norms.block_norms(h, h, gate=torch.ones(1, 64, dtype=BF16)), lambda: norms.block_norms(h, h, gate=torch.ones(4, 64, dtype=torch.int32)),
           lambda: norms.block_norms(h, h, w, w), lambda: norms.rms_norm(h, w)]  # the last two: not on a GPU
    for call in bad:
        with pytest.raises(NormError):
            call()


def test_refusals_name_the_argument():
    """Shapes and types are refused for what they are, before the look at the device; a tensor given twice is checked in each place."""
    from nvshmem_b200.ops import norms
    h, w, token = torch.zeros(4, 64, dtype=BF16), torch.ones(64, dtype=BF16), torch.ones(4, 1, dtype=BF16)
    bad = [(lambda: norms.rms_norm(h, w[:32]), "before the block must be of shape"), (lambda: norms.rms_norm(h, w.half()), "must be torch.bfloat16 or float32"),
           (lambda: norms.rms_norm(h, w[None]), "before the block must be of shape"), (lambda: norms.rms_norm(torch.zeros(2, 16385), torch.ones(16385)), "rows of 1 to"),
           (lambda: norms.block_norms(h, h[:3]), "residual"), (lambda: norms.block_norms(h, h.half()), "residual"), (lambda: norms.block_norms(h.float(), h), "residual"),
           (lambda: norms.block_norms(h, h, w[:63]), "after the block must be of shape"), (lambda: norms.block_norms(h, h, w, w.float()), "one type"),
           (lambda: norms.block_norms(h, h, token, gate=token), "after the block must be of shape"),
           (lambda: norms.block_norms(h, h, None, token, gate=token), "before the block must be of shape"),
           (lambda: norms.block_norms(h, h, gate=w[:4]), "gate must be of shape"), (lambda: norms.block_norms(h, h, gate=token.float().double()), "gate must be"),
           (lambda: norms.block_norms(h, h, w, w), "on the GPU")]
    for call, message in bad:
        with pytest.raises(norms.NormError, match=message):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, F32])
def test_a_weight_and_a_gate_in_one_unaligned_place(dt):
    """A gate per token that shares its memory with the weights, which do not start on 16 bytes."""
    from nvshmem_b200.ops import norms
    d = _norm_inputs(64, 64, dt, dt, dt, "token")
    w = torch.cat([d["post"][:1], d["post"]])[1:]
    assert w.data_ptr() % 16
    gate = w.view(64, 1)
    r, y = norms.block_norms(d["h"], d["residual"], w, w, gate)
    want, mag = _reference({**d, "post": w, "pre": w, "gate": gate}, 1.0, 1.0, 1e-6, 0.0, backward=False)
    _compare(r, want["r"], mag["r"], "r")
    _compare(y, want["y"], mag["y"], "y")


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,dt,rt,gate,post", [(1700, 8192, BF16, F32, "channel", True), (1333, 7000, BF16, F32, "full", True), (1700, 8192, BF16, F32, "token", False),
                                                 (2900, 4096, F32, F32, "channel", True), (1024, 8192, F32, F32, "none", True),
                                                 (500, 16384, BF16, F32, "channel", True), (400, 12296, F16, F32, "full", True)])
def test_many_rows_a_cta(T, H, dt, rt, gate, post):
    """The ring goes round several times."""
    _check(_norm_inputs(T, H, dt, rt, F32, gate, post, True))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(40, 1000), (40, 1001), (400, 2048)])
def test_infinities_without_norms(T, H):
    """r = residual + gate h alone: the gradients of h and residual do not depend on either, infinite or not."""
    from nvshmem_b200.ops import norms
    d = _norm_inputs(T, H, BF16, F32, BF16, "token", False, False)
    d["h"][1, 3], d["residual"][2, 5] = float("inf"), -float("inf")
    h, res = d["h"].requires_grad_(True), d["residual"].requires_grad_(True)
    dh, dres = torch.autograd.grad(norms.block_norms(h, res, gate=d["gate"])[0], [h, res], d["dr"])
    assert torch.equal(dres, d["dr"])
    _compare(dh, d["gate"].double() * d["dr"].double(), (d["gate"].double() * d["dr"].double()).abs(), "d_h")


FRESH = """
import sys
import torch
sys.path.insert(0, {root!r})
from tests.test_block_norms import _check, _norm_inputs, BF16, F32
torch.cuda.set_device(0)
for T, H, dt, rt, wt, gate, pre in (
        (400, 4080, BF16, BF16, BF16, "channel", True), (1000, 2040, BF16, BF16, F32, "none", True), (900, 2448, BF16, F32, F32, "channel", False),
        (700, 2720, BF16, F32, BF16, "token", True), (1000, 1632, F32, F32, F32, "full", True), (900, 1528, F32, F32, F32, "channel", True)):
    _check(_norm_inputs(T, H, dt, rt, wt, gate, True, pre))
"""
FRESH_NORM = """
import torch
from nvshmem_b200.ops import rms_norm
torch.cuda.set_device(0)
for T, H, dt in ((200, 8160, torch.bfloat16), (300, 4080, torch.float32), (900, 2040, torch.float16)):
    x = torch.randn(T, H, device="cuda").to(dt).requires_grad_(True)
    y = rms_norm(x, torch.ones(H, device="cuda", dtype=dt))
    want = x.detach().double()
    want = want * torch.rsqrt(want.square().mean(-1, keepdim=True) + 1e-6)
    # half a step of the type (below its smallest normal value the steps stay smallest_normal * eps: a few of a million fp16 values lie
    # there, where half a step is 2^-25 whatever the value is), and the statistics' part of 2^-18
    half = torch.finfo(dt).eps / 2
    assert ((y.detach().double() - want).abs() <= want.abs() * (half + 2.0 ** -18) + torch.finfo(dt).smallest_normal * half).all(), H
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert g.isfinite().all()
"""


@pytest.mark.gpu
@pytest.mark.parametrize("script", [FRESH, FRESH_NORM], ids=["block_norms", "rms_norm"])
def test_stages_that_just_fit_the_default_shared_memory(script):
    """Rows whose stages take just under 48 KB: with the kernel's own arrays that is more than a launch gets unless the limit is raised.  In a
    process of its own, as a limit stays raised once another size has asked for it."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", script.replace("{root!r}", repr(root))], cwd=root, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
