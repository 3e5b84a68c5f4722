"""The operators around a block as they are used together: norm, router, exchange, experts, norm with gate and residual, 4-bit product;
a training step of router, balance loss and norms; all of it captured and replayed, on other streams and side by side."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def nv():
    import nvshmem_b200.core as nv
    torch.cuda.set_device(0)
    nv.init(device=0, uid=nv.get_unique_id(), rank=0, nranks=1)
    yield nv
    nv.finalize()


def _rms(v, w, eps=1e-6):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w


class _Layer:
    """A mixture-of-experts layer between its norms, and a product in 4 bits behind it."""

    def __init__(self, T, H=512, F=256, E=8, K=2, N=384):
        from nvshmem_b200.ops import fused_gemm as fg
        from nvshmem_b200.ops.moe import MoeDispatchCombine
        from nvshmem_b200.ops.mxfp4 import quantize_mxfp4
        g = torch.Generator(device="cuda").manual_seed(T)
        rn = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(BF16)
        self.T, self.H, self.F, self.E, self.K = T, H, F, E, K
        self.pre, self.post, self.nxt = (1 + rn(H, scale=0.1) for _ in range(3))
        self.gate, self.router = 0.5 + rn(H, scale=0.1), rn(E, H, scale=H ** -0.5)
        self.w_in, self.w_out, w = rn(E, 2 * F, H, scale=H ** -0.5), rn(E, H, F, scale=F ** -0.5), rn(N, H, scale=H ** -0.5)
        self.gated, self.w4 = fg.interleave_gate_up(self.w_in), quantize_mxfp4(w)
        self.moe = MoeDispatchCombine(T, H, K, E)
        self.act = torch.empty(self.moe.cap_rows, F, dtype=BF16, device="cuda")

    def __call__(self, x, valid):
        from nvshmem_b200.ops import balance_loss, block_norms, gemm_mxfp4, moe_route, rms_norm
        from nvshmem_b200.ops import fused_gemm as fg
        y = rms_norm(x, self.pre)
        logits = y @ self.router.t()
        idx, weight = moe_route(logits, self.K, valid=valid)
        loss, counts = balance_loss(logits, idx, valid=valid)
        recv, offsets = self.moe.dispatch(y, idx)
        fg.grouped_gemm(recv, self.gated, offsets, out=self.act, act="swiglu")
        fg.grouped_gemm(self.act, self.w_out, offsets, out=self.moe.expert_out)
        h = self.moe.combine(idx, weight)
        r, z = block_norms(h, x, self.post, self.nxt, self.gate, residual_scale=0.5, branch_scale=2.0)
        return {"idx": idx, "weight": weight, "loss": loss, "counts": counts, "r": r, "z": z, "out": gemm_mxfp4(z, self.w4)}


@pytest.mark.parametrize("T", [1, 61, 192])
def test_a_layer_of_them(nv, T):
    """Against plain fp32.  The chain rounds to bf16 at the norm (2^-8 half a step, relative), the experts' activation and output, the
    combine, r and z: six roundings, 6 * 2^-8 of a value's scale, taken at the largest value of the result."""
    from nvshmem_b200.ops import fused_gemm as fg
    layer = _Layer(T)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, layer.H, device="cuda", generator=g).to(BF16)
    valid = torch.arange(T, device="cuda") < max(1, T - 5)
    got = layer(x, valid)
    torch.cuda.synchronize()
    fg.check_errors()
    # the plain form, from the same choice (the logits are a library product in bf16: its borders may fall either way)
    y = _rms(x.float(), layer.pre.float()).to(BF16).float()
    logits = y @ layer.router.float().t()
    idx, w = got["idx"].long(), got["weight"]
    assert (idx[~valid] == -1).all() and not w[~valid].any() and int(got["counts"].sum()) == int(valid.sum()) * layer.K
    chosen = logits.gather(-1, idx.clamp(min=0))
    assert ((chosen.softmax(-1) - w).abs()[valid] <= 0.05).all()
    h = torch.zeros(T, layer.H, device="cuda")
    for e in range(layer.E):
        tok, slot = (idx == e).nonzero(as_tuple=True)
        a = y[tok] @ layer.w_in[e].float().t()
        a = torch.nn.functional.silu(a[:, :layer.F]) * a[:, layer.F:]
        h.index_add_(0, tok, (a @ layer.w_out[e].float().t()) * w[tok, slot].unsqueeze(-1))
    r = 0.5 * x.float() + 2.0 * layer.gate.float() * _rms(h, layer.post.float())
    z = _rms(r, layer.nxt.float())
    for name, want in (("r", r), ("z", z)):
        err = (got[name].float() - want).abs().max()
        assert err <= 6 * 2.0 ** -8 * want.abs().max(), (name, err)
    # the rows behind the valid ones got nothing from the experts
    assert torch.equal(got["r"][~valid].float(), (0.5 * x[~valid].float()).to(BF16).float())
    from nvshmem_b200.ops.mxfp4 import quantize_mxfp4
    want = quantize_mxfp4(got["z"]).dequantize(F32) @ layer.w4.dequantize(F32).t()
    assert (got["out"].float() - want).abs().max() <= 2.0 ** -8 * want.abs().max() + 1e-5
    layer.moe.close()


@pytest.mark.parametrize("T", [61, 192])
def test_a_layer_captured_and_replayed(nv, T):
    from nvshmem_b200.ops import fused_gemm as fg
    layer = _Layer(T)
    x, valid = torch.empty(T, layer.H, dtype=BF16, device="cuda"), torch.empty(T, dtype=torch.bool, device="cuda")

    def fill(seed):
        torch.manual_seed(seed)
        x.copy_(torch.randn(T, layer.H, device="cuda"))
        valid.copy_(torch.rand(T, device="cuda") > 0.2)

    fill(0)
    layer(x, valid)
    graphs = []
    for _ in range(2):   # two graphs of the same calls, replayed in turn
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = layer(x, valid)
        graphs.append((graph, out))
    torch.cuda.synchronize()
    for seed in (1, 2, 3):
        fill(seed)
        want = {k: v.clone() for k, v in layer(x, valid).items()}
        graph, out = graphs[seed % 2]
        for v in out.values():
            v.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        fg.check_errors()
        for k in want:
            assert torch.equal(out[k], want[k]), k
    layer.moe.close()


def _step(d, K):
    """Loss and gradients of a small training step: norm, router, weights, balance loss, norm with gate and residual."""
    from nvshmem_b200.ops import balance_loss, block_norms, moe_route, rms_norm
    y = rms_norm(d["x"], d["pre"])
    logits = y @ d["router"].t()
    idx, weight = moe_route(logits, K, score="sigmoid", renormalize=True, scale=1.5)
    loss, counts = balance_loss(logits, idx)
    r, z = block_norms(y * weight.sum(-1, keepdim=True) * weight[:, :1], d["x"], d["post"], d["nxt"], d["gate"])
    total = loss + (r * d["dr"]).mean() + (z * d["dr"]).mean()
    names = ("x", "pre", "router", "post", "nxt", "gate")
    return (total, counts, idx, *torch.autograd.grad(total, [d[n] for n in names]))


def _training_data(T, H, E, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s, scale=1.0, shift=0.0: torch.randn(*s, device="cuda", generator=g) * scale + shift
    d = {"x": rn(T, H), "pre": rn(H, scale=0.1, shift=1.0), "router": rn(E, H, scale=H ** -0.5), "post": rn(H, scale=0.1, shift=1.0), "nxt": rn(H, scale=0.1, shift=1.0),
         "gate": rn(T, 1, scale=0.1, shift=0.5)}
    return {**{k: v.requires_grad_(True) for k, v in d.items()}, "dr": rn(T, H)}


@pytest.mark.parametrize("T,H,E,K", [(37, 96, 12, 3), (700, 1024, 64, 6)])
def test_a_training_step_against_64_bits(T, H, E, K):
    """Every operator is in fp32 here, off by some 2^-18 of the parts it adds; the chain of six of them, with products between in fp32
    over H terms, stays below 2^-12 of the largest value of each gradient."""
    d = _training_data(T, H, E, 5)
    total, counts, idx, *grads = _step(d, K)
    names = ("x", "pre", "router", "post", "nxt", "gate")
    v = {n: d[n].detach().double().requires_grad_(True) for n in names}
    y = _rms(v["x"], v["pre"])
    logits = y @ v["router"].t()
    s = torch.sigmoid(logits)
    w = s.gather(-1, idx.long())
    w = 1.5 * w / w.sum(-1, keepdim=True)
    p = torch.softmax(logits, -1)   # the balance loss takes softmax scores unless told otherwise
    n = torch.bincount(idx.flatten().long(), minlength=E)
    loss = E * (n.double() / (T * K) * p.mean(0)).sum()
    r = v["x"] + v["gate"] * _rms(y * w.sum(-1, keepdim=True) * w[:, :1], v["post"])
    z = _rms(r, v["nxt"])
    ref = loss + (r * d["dr"]).mean() + (z * d["dr"]).mean()
    assert torch.equal(counts.long(), n) and abs(total.double() - ref) <= 2.0 ** -12 * abs(ref)
    for name, got, want in zip(names, grads, torch.autograd.grad(ref, [v[k] for k in names])):
        assert (got.double() - want).abs().max() <= 2.0 ** -12 * want.abs().max(), name


def test_a_training_step_captured_and_replayed():
    """Forward and backward in one graph, on leaves of its own, replayed on new values."""
    T, H, E, K = 600, 1024, 64, 6
    d = _training_data(T, H, E, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _step(d, K)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _step(d, K)
    torch.cuda.synchronize()
    for seed in (2, 3):
        fresh = _training_data(T, H, E, seed)
        with torch.no_grad():
            for k in d:
                d[k].copy_(fresh[k])
        want = [t.detach().clone() for t in _step(fresh, K)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(out, want):
            assert torch.equal(got, ref)


def test_calls_on_two_streams_at_once(nv):
    """The same operators on two streams side by side give what they give alone: nothing is shared between calls."""
    from nvshmem_b200.ops import balance_loss, block_norms, gemm_mxfp4, moe_route, quantize_mxfp4

    def calls(d):
        r, z = block_norms(d["h"], d["x"], d["w"], d["w"], d["w"])
        idx, weight = moe_route(z[:, :64], 4)
        loss, counts = balance_loss(z[:, :64], idx)
        q = quantize_mxfp4(z)
        return [r, z, idx, weight, loss, counts, q.data, gemm_mxfp4(z, d["q"]), gemm_mxfp4(z[:20], d["q"])]

    data = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
        data.append({"h": rn(700, 2048), "x": rn(700, 2048), "w": rn(2048), "q": quantize_mxfp4(rn(1024, 2048))})
    want = [[t.clone() for t in calls(d)] for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(5):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(calls(d))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for t, ref in zip(a, b):
                assert torch.equal(t, ref)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_moe_block_with_the_fused_router(nv, score):
    from nvshmem_b200.models import ExpertParallelMoE
    from nvshmem_b200.ops import fused_gemm as fg
    T, H, F, E, K = 192, 256, 384, 8, 2
    plain = ExpertParallelMoE(T, H, F, E, K, seed=3)
    block = ExpertParallelMoE(T, H, F, E, K, seed=3, router="fused", score=score)
    torch.manual_seed(17)
    x = torch.randn(T, H, device="cuda").to(BF16)
    idx, weight = block.route(x)
    pidx, pweight = plain.route(x)
    logits = x @ block.router.t()
    clear = logits.float().sort(-1, descending=True).values[:, :K + 1].diff(dim=-1).abs().min(-1).values > 0   # tokens without equal logits at the border
    assert torch.equal(idx[clear], pidx[clear]) and clear.float().mean() > 0.9
    if score == "softmax":
        assert (weight - pweight)[clear].abs().max() <= 1e-6
        got, want = block(x)[clear], plain(x)[clear]
        assert torch.equal(got, want) or (got.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
    block.router_bias = torch.zeros(E, device="cuda")
    block.router_bias[3] = 100.0
    assert (block.route(x)[0][:, 0] == 3).all()
    torch.cuda.synchronize()
    fg.check_errors()
    plain.close()
    block.close()
    with pytest.raises(ValueError):
        ExpertParallelMoE(T, H, F, E, K, score="sigmoid")


FAILED = """
import torch
from nvshmem_b200.ops import gemm_mxfp4, moe_route, norms, quantize_mxfp4
torch.cuda.set_device(0)
x, w, y = torch.randn(300, 512, device="cuda"), torch.ones(512, device="cuda"), torch.empty(300, 512, device="cuda")
logits, q, out = torch.randn(4, 8, device="cuda"), quantize_mxfp4(x), torch.empty(300, 300, device="cuda", dtype=torch.bfloat16)
plan = norms._settings(None, x, None, w, None, 300, 512, 0, 1.0, 1.0, 1e-6, 0.0)
plan.device = 0
def norm():
    a = norms._Args(*plan.head, *plan.strides(None, x, None), 0, 0, *plan.scales, residual=x.data_ptr(), pre=w.data_ptr(), y=y.data_ptr(), error_flag=flag)
    plan.launch(norms._lib().bshmem_block_norms, a, "bshmem_block_norms")
flag = norms._error_flag(x.device).data_ptr()
call = dict(norm=norm, gemm=lambda: gemm_mxfp4(q, q, out=out))[CALL]   # neither takes memory
call()
want = [t.clone() for t in moe_route(logits, 2)]
torch.cuda.synchronize()
refused = ""
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            torch.cuda.current_stream().synchronize()   # not allowed here: from now on every launch of this capture fails
        except RuntimeError:
            pass
        try:
            call()
        except RuntimeError as e:
            refused = str(e)
except RuntimeError:
    pass
assert refused.startswith("bshmem"), refused
for a, b in zip(moe_route(logits, 2), want):   # its own launch is fine
    assert torch.equal(a, b)
"""


@pytest.mark.parametrize("call", ["norm", "gemm"])
def test_a_launch_that_fails_is_not_blamed_on_the_next_call(call):
    """In a process of its own: a capture that was made invalid on the host refuses launches."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", f"CALL = {call!r}\n" + FAILED], cwd=root, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]


def test_the_routers_bias_is_part_of_the_block(nv):
    """It is saved and loaded with the block, moves with it and stays in 32 bits."""
    from nvshmem_b200.models import ExpertParallelMoE
    T, H, F, E, K = 128, 256, 128, 8, 2
    make = lambda: ExpertParallelMoE(T, H, F, E, K, seed=3, router="fused", score="sigmoid")
    block = make()
    assert block.router_bias is None and "router_bias" not in block.state_dict()
    plain = {k: v.clone() for k, v in block.state_dict().items()}
    bias = torch.randn(E, device="cuda")
    block.router_bias = bias.clone()
    state = {k: v.clone() for k, v in block.state_dict().items()}
    assert torch.equal(state["router_bias"], bias)
    other = make()
    other.load_state_dict(state)
    x = torch.randn(T, H, device="cuda").to(BF16)
    assert torch.equal(other.router_bias, bias) and other.router_bias.is_cuda and torch.equal(other.route(x)[0], block.route(x)[0])
    other.to(BF16)
    assert other.router_bias.dtype == F32 and torch.equal(other.router_bias, bias)
    other.load_state_dict({**state, "router_bias": (bias + 1).cpu()})
    assert torch.equal(other.router_bias, bias + 1) and other.router_bias.is_cuda
    with pytest.raises(RuntimeError):       # a block with a bias, a checkpoint without
        other.load_state_dict(plain)
    fresh = make()
    fresh.load_state_dict(plain)
    assert fresh.router_bias is None
    for b in (block, other, fresh):
        b.close()


def test_sigmoid_scores_and_a_bias_in_the_moe_block(nv):
    """The block's weights are the chosen experts' sigmoids over their sum, whatever bias chose them, and its output is that of the plain form:
    three roundings to bf16 on the way (activation, experts' output, result), 2^-8 each of the largest value."""
    from nvshmem_b200.models import ExpertParallelMoE
    from nvshmem_b200.ops import fused_gemm as fg
    T, H, F, E, K = 192, 256, 384, 8, 2
    block = ExpertParallelMoE(T, H, F, E, K, seed=3, router="fused", score="sigmoid")
    torch.manual_seed(18)
    x = torch.randn(T, H, device="cuda").to(BF16)
    s = torch.sigmoid((x @ block.router.t()).double())
    for bias in (None, torch.linspace(-0.4, 0.4, E, device="cuda")):
        block.router_bias = bias
        idx, weight = block.route(x)
        order = s if bias is None else s + bias.double()
        top = order.sort(dim=-1, descending=True, stable=True)
        assert torch.equal(idx.long(), top.indices[:, :K])
        want = s.gather(-1, idx.long())
        want = want / want.sum(-1, keepdim=True)
        assert ((weight.double() - want).abs() <= 2.0 ** -18 * want).all()
        out = torch.zeros(T, H, device="cuda")
        for e in range(E):
            tok, slot = (idx == e).nonzero(as_tuple=True)
            a = x[tok].float() @ block.w_in[e].float().t()
            a = torch.nn.functional.silu(a[:, :F]) * a[:, F:]
            out.index_add_(0, tok, (a @ block.w_out[e].float().t()) * weight[tok, slot].unsqueeze(-1))
        assert (block(x).float() - out).abs().max() <= 3 * 2.0 ** -8 * out.abs().max()
    torch.cuda.synchronize()
    fg.check_errors()
    block.close()


def test_gradients_that_would_be_lost_are_refused():
    """The 4-bit floats record no gradients, and say so where one is asked for."""
    from nvshmem_b200.ops import gemm_mxfp4, quantize_mxfp4
    from nvshmem_b200.ops.fused_gemm import FusedGemmError
    x = torch.randn(5, 64, device="cuda", requires_grad=True)
    with torch.no_grad():
        q = quantize_mxfp4(x)
        want = gemm_mxfp4(x, q)
    for call in (lambda: quantize_mxfp4(x), lambda: quantize_mxfp4(x * 2), lambda: gemm_mxfp4(x, q), lambda: gemm_mxfp4(x * 2, q)):
        with pytest.raises(FusedGemmError, match="no_grad"):
            call()
    out = torch.zeros(5, 5, device="cuda", dtype=BF16, requires_grad=True)
    with pytest.raises(FusedGemmError, match="no_grad"):
        gemm_mxfp4(x.detach(), q, out=out)
    assert torch.equal(gemm_mxfp4(x.detach(), quantize_mxfp4(x.detach())), want)


def test_tangents_are_refused():
    """Forward-mode derivatives are not computed: a call with a tangent on an input raises, with and without a gradient asked for."""
    import torch.autograd.forward_ad as fwd
    from nvshmem_b200.ops import balance_loss, block_norms, gemm_mxfp4, moe_route, quantize_mxfp4, rms_norm
    x, w = torch.randn(6, 64, device="cuda"), torch.ones(64, device="cuda")
    idx, q = moe_route(x, 2)[0], quantize_mxfp4(x)
    calls = [lambda t: rms_norm(t, w), lambda t: rms_norm(x, t[0]), lambda t: block_norms(t, x, w)[0], lambda t: block_norms(x, t)[0], lambda t: block_norms(x, x, gate=t)[0],
             lambda t: moe_route(t, 2)[1], lambda t: balance_loss(t, idx)[0], lambda t: quantize_mxfp4(t), lambda t: gemm_mxfp4(t, q)]
    with fwd.dual_level():
        for call in calls:
            call(x)      # no tangent: as outside
            dual = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(dual)
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                call(dual)


def test_offsets_beyond_32_bits():
    """More than 2^31 values a tensor: the last rows give what they give alone (the sums over rows aside)."""
    from nvshmem_b200.ops import balance_loss, block_norms, fused_gemm, gemm_mxfp4, moe_route, quantize_mxfp4, rms_norm
    T, H, tail = 263000, 8192, 200
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, H, device="cuda", generator=g, dtype=BF16)
    w, gate = (torch.rand(H, device="cuda", generator=g) + 0.5).to(BF16), torch.rand(T, 1, device="cuda", generator=g).to(BF16)
    assert x.numel() > 2 ** 31

    def norms(x, gate):
        x = x.detach().requires_grad_(True)
        y = rms_norm(x, w)
        (dy,) = torch.autograd.grad(y, x, x.detach())
        r, z = block_norms(x, x, w, w, gate)
        (dr,) = torch.autograd.grad([r, z], x, [x.detach(), x.detach()])
        return y.detach(), dy, r.detach(), z.detach(), dr

    whole = [t[-tail:].clone() for t in norms(x, gate)]
    alone = norms(x[-tail:], gate[-tail:])
    for a, b in zip(whole, alone):   # other kernels take few rows: the same sums in another order, so a rounding may fall the other way
        assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -14 * b.float().abs().max()).all()
    torch.cuda.empty_cache()
    q, wq = quantize_mxfp4(x), quantize_mxfp4(torch.randn(H, H, device="cuda", generator=g))
    tq = quantize_mxfp4(x[-tail:])
    assert torch.equal(q.data[-tail:], tq.data) and torch.equal(q.codes[-tail:], tq.codes)
    assert torch.equal(q.dequantize()[-tail:], tq.dequantize())
    out = gemm_mxfp4(x, wq)     # 2^31 values come out as well
    want = tq.dequantize(F32).double() @ wq.dequantize(F32).double().t()
    mag = tq.dequantize(F32).double().abs() @ wq.dequantize(F32).double().abs().t()
    assert ((out[-tail:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * mag).all()
    assert torch.equal(out[:tail], gemm_mxfp4(x[:2 * 8192], wq)[:tail])
    del out, q, whole, alone
    torch.cuda.empty_cache()
    logits = x.view(-1, 256)[:8400000]
    assert logits.numel() > 2 ** 31

    def route(l):
        l = l.detach().requires_grad_(True)
        idx, weight = moe_route(l, 8, renormalize=False)
        (dl,) = torch.autograd.grad(weight, l, torch.ones_like(weight) * torch.arange(8, device="cuda"))
        return idx, weight.detach(), dl

    whole, alone = route(logits), route(logits[-tail:])
    for a, b in zip(whole, alone):
        assert torch.equal(a[-tail:], b)
    idx = whole[0]
    del whole
    l = logits.detach().requires_grad_(True)
    loss, counts = balance_loss(l, idx)
    assert torch.equal(counts.long(), torch.bincount(idx.view(-1), minlength=256))
    (dl,) = torch.autograd.grad(loss, l)
    p = torch.softmax(l.detach()[-tail:].double(), -1)
    c = counts.double() * 256 / (8 * float(len(idx)) ** 2)
    want = p * (c - (p * c).sum(-1, keepdim=True))
    assert ((dl[-tail:].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * p * c.max()).all()
    torch.cuda.synchronize()
    fused_gemm.check_errors()


FIRST_CALL = """
import torch
from nvshmem_b200.ops import fused_gemm as fg
from nvshmem_b200.ops import gemm_mxfp4, quantize_mxfp4, rms_norm
torch.cuda.set_device(0)
x, w = torch.randn(300, 512, device="cuda"), torch.ones(512, device="cuda")
if CALL == "norm":
    call, want = lambda: rms_norm(x, w), x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
else:
    q = quantize_mxfp4(x)
    call, want = lambda: gemm_mxfp4(q, q).float(), q.dequantize(torch.float32) @ q.dequantize(torch.float32).t()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = call()
fg.check_errors()
fg._error_flag(x.device).fill_(1)      # as a kernel does that gave up on a wait
graph.replay()
assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7).all()
assert fg.take_error() == 1 and fg.take_error() == 0
graph.replay()
fg.check_errors()
"""


@pytest.mark.parametrize("call", ["norm", "gemm"])
def test_a_first_call_that_is_captured_keeps_errors(call):
    """In a process of its own: the error word is made by the first call; a replay must not take an error back that nobody has read."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", f"CALL = {call!r}\n" + FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
