"""Performance cases of the operators around a block: what a user's program has this framework do on one GPU.

`listed()` names the cases, `draw(rng)` gives more of the same ranges, `prepare` makes what a program has in hand before the
call, `run` is one pass, `exact` the same result in 64 bits.  With `own` false `run` computes the plain form (elementary torch
operations in 32 bits or more), with `own` true it calls the framework.  Kinds of case:

* ``norm``     ``ops.norms``: the norm before a block (part "in"), the norm after it with gate and scaled residual (part "out"),
               and that with the next block's norm in the same pass (part "out_in"); forward, or forward and backward
* ``route``    ``ops.routing.moe_route``: the experts of every token and their weights; forward, or forward and backward
* ``balance``  ``ops.routing.balance_loss``: balance loss and per-expert counts; forward and backward
* ``quant``    ``ops.mxfp4``: quantisation to microscaled 4-bit floats and reading the values back
* ``product``  ``ops.mxfp4.gemm_mxfp4``: activations (quantised in the call) times weights kept in microscaled 4-bit floats
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # decode: eight sequences, one token each, between two blocks; latency of one call
        {"name": "norm_decode", "kind": "norm", "part": "out_in", "T": 8, "H": 7168, "dtype": "bf16", "res": "bf16", "wt": "bf16", "gate": "channel", "back": False},
        # prefill of 4096 tokens between two blocks of the benchmark's hidden size
        {"name": "norm_prefill", "kind": "norm", "part": "out_in", "T": 4096, "H": 8192, "dtype": "bf16", "res": "bf16", "wt": "bf16", "gate": "channel", "back": False},
        # a training step's pass between two blocks, with the residual stream and the parameters in 32 bits
        {"name": "norm_train", "kind": "norm", "part": "out_in", "T": 4096, "H": 8192, "dtype": "bf16", "res": "f32", "wt": "f32", "gate": "channel", "back": True},
        # odd sizes, fp16, one gate value per token, no norm that follows
        {"name": "norm_train_ragged", "kind": "norm", "part": "out", "T": 777, "H": 1001, "dtype": "f16", "res": "f16", "wt": "f16", "gate": "token", "back": True},
        # decode batch of a large MoE layer
        {"name": "route_decode", "kind": "route", "T": 64, "E": 256, "K": 8, "dtype": "f32", "score": "softmax", "bias": False, "norm": True, "mask": False, "back": False},
        # training batch; the choice is corrected by a bias per expert
        {"name": "route_train", "kind": "route", "T": 8192, "E": 256, "K": 8, "dtype": "f32", "score": "sigmoid", "bias": True, "norm": True, "mask": False, "back": True},
        # a short padded batch of a small layer with 16-bit logits
        {"name": "balance_ragged", "kind": "balance", "T": 61, "E": 40, "K": 3, "dtype": "bf16", "score": "softmax", "mask": True},
        # training batch of a large MoE layer
        {"name": "balance_train", "kind": "balance", "T": 8192, "E": 256, "K": 8, "dtype": "f32", "score": "softmax", "mask": False},
        # odd number of rows, 32-bit values, a few blocks a row
        {"name": "quant_ragged", "kind": "quant", "R": 1001, "K": 1184, "dtype": "f32"},
        # a weight matrix of the benchmark's MLP, or 8192 tokens' activations
        {"name": "quant_large", "kind": "quant", "R": 8192, "K": 8192, "dtype": "bf16"},
        # decode: 16 tokens against a large weight matrix, which is read once
        {"name": "product_decode", "kind": "product", "M": 16, "N": 8192, "K": 8192},
        # the benchmark's product
        {"name": "product_prefill", "kind": "product", "M": 8192, "N": 8192, "K": 3584},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, lo, hi, step):
    return min(hi, max(lo, round(_log(rng, lo, hi) / step) * step))


def draw(rng):
    kind = rng.choice(["norm", "norm", "route", "balance", "quant", "product", "product"])
    if kind == "norm":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        part = rng.choice(["in", "out", "out_in", "out_in"])
        h = rng.choice([_log(rng, 64, 8192), _mult(rng, 64, 8192, 64)])
        gate = rng.choice(["none", "channel", "token", "full"])
        most = 4096 * 8192 // (2 if dtype == "f32" or gate == "full" else 1) // h
        return {"kind": kind, "part": part, "T": min(_log(rng, 1, 4096), most), "H": h, "dtype": dtype, "res": rng.choice([dtype, "f32"]),
                "wt": rng.choice([dtype, "f32"]), "gate": gate, "back": rng.choice([True, False])}
    if kind in ("route", "balance"):
        e = rng.choice([_log(rng, 2, 256), rng.choice([8, 16, 32, 64, 128, 256])])
        case = {"kind": kind, "T": _log(rng, 1, 8192), "E": e, "K": rng.randint(1, min(e, 10)), "dtype": rng.choice(["f32", "f32", "bf16"]),
                "score": rng.choice(["softmax", "sigmoid"]), "mask": rng.choice([True, False])}
        if kind == "route":
            case.update(bias=rng.choice([True, False]), norm=rng.choice([True, False]), back=rng.choice([True, False]))
        return case
    if kind == "quant":
        dtype = rng.choice(["bf16", "f16", "f32"])
        return {"kind": kind, "R": _log(rng, 1, 6000 if dtype == "f32" else 8192), "K": _mult(rng, 32, 8192, 32), "dtype": dtype}
    m, n = _log(rng, 1, 8192), rng.choice([_log(rng, 8, 8192), _mult(rng, 64, 8192, 64)])
    return {"kind": kind, "M": m, "N": n, "K": min(_mult(rng, 32, 8192, 32), (8192 * 8192 * 3584 // (m * n)) // 32 * 32)}


# ------------------------------------------------------------------ inputs
def _randn(gen, *shape, scale=1.0, shift=0.0, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).mul_(scale).add_(shift).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k = case["kind"]
    if k == "norm":
        T, H, dt, rt, wt = case["T"], case["H"], DTYPES[case["dtype"]], DTYPES[case["res"]], DTYPES[case["wt"]]
        d = {"pre": _randn(gen, H, scale=0.1, shift=1.0, dtype=wt)}
        if case["part"] == "in":
            d["x"] = _randn(gen, T, H, scale=2.0, dtype=dt)
        else:
            d["h"], d["residual"] = _randn(gen, T, H, scale=0.5, dtype=dt), _randn(gen, T, H, scale=2.0, dtype=rt)
            d["post"] = _randn(gen, H, scale=0.1, shift=1.0, dtype=wt)
            shape = {"channel": (H,), "token": (T, 1), "full": (T, H)}.get(case["gate"])
            d["gate"] = _randn(gen, *shape, scale=0.2, shift=0.5, dtype=wt) if shape else None
        if case["back"]:
            if case["part"] != "in":
                d["dr"] = _randn(gen, T, H, dtype=rt)
            if case["part"] != "out":
                d["dy"] = _randn(gen, T, H, dtype=dt)
        return d
    if k in ("route", "balance"):
        T, E, K = case["T"], case["E"], case["K"]
        d = {"logits": _randn(gen, T, E, scale=1.5, dtype=DTYPES[case["dtype"]]), "valid": None}
        if case["mask"]:  # the batch's tail is padding, and so are a few rows inside
            d["valid"] = (torch.arange(T, device="cuda") < max(1, T - T // 5)) & (torch.rand(T, device="cuda", generator=gen) > 0.05)
        if k == "route":
            d["bias"] = _randn(gen, E, scale=0.05, dtype=torch.float32) if case["bias"] else None
            d["dw"] = _randn(gen, T, K, dtype=torch.float32) if case["back"] else None
        else:
            d["idx"] = torch.rand(T, E, device="cuda", generator=gen).argsort(-1)[:, :K].to(torch.int32).contiguous()
            if case["mask"]:
                d["idx"].masked_fill_(~d["valid"].unsqueeze(-1), -1)
            d["dloss"] = torch.rand((), device="cuda", generator=gen) * 0.01 + 0.001
        return d
    if k == "quant":
        x = _randn(gen, case["R"], case["K"], dtype=torch.float32)
        x *= torch.exp2(torch.randint(-6, 7, (case["R"], case["K"] // 32, 1), device="cuda", generator=gen).float()).expand(-1, -1, 32).reshape(x.shape)
        return {"x": x.to(DTYPES[case["dtype"]])}
    return {"x": _randn(gen, case["M"], case["K"]), "w": _randn(gen, case["N"], case["K"], scale=0.02)}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own and case["kind"] == "product":
        from nvshmem_b200.ops import mxfp4
        s["w"] = mxfp4.quantize_mxfp4(s["w"])
    elif case["kind"] == "product":
        s["w"] = _plain_quantize(s["w"])
    elif own and case.get("back", case["kind"] == "balance"):
        for name in _leaves(case):
            s[name].requires_grad_(True)
    return s


def _leaves(case):
    if case["kind"] != "norm":
        return ["logits"]
    if case["part"] == "in":
        return ["x", "pre"]
    return ["h", "residual", "post"] + (["pre"] if case["part"] == "out_in" else []) + (["gate"] if case["gate"] != "none" else [])


A_SCALE, B_SCALE = 0.75, 1.25   # of the residual and of the block's output


# ------------------------------------------------------------------ the framework's operators
def _run_own(s):
    c, k = s["case"], s["case"]["kind"]
    if k == "norm":
        from nvshmem_b200.ops import norms
        if c["part"] == "in":
            outs = {"y": norms.rms_norm(s["x"], s["pre"], eps=EPS)}
        else:
            r, y = norms.block_norms(s["h"], s["residual"], post_weight=s["post"], pre_weight=s["pre"] if c["part"] == "out_in" else None, gate=s["gate"],
                                     residual_scale=A_SCALE, branch_scale=B_SCALE, eps=EPS)
            outs = {"r": r, "y": y} if c["part"] == "out_in" else {"r": r}
        if not c["back"]:
            return outs
        names = _leaves(c)
        grads = torch.autograd.grad(list(outs.values()), [s[n] for n in names], [s["d" + n] for n in outs])
        return {**{n: o.detach() for n, o in outs.items()}, **{"d_" + n: g for n, g in zip(names, grads)}}
    if k == "route":
        from nvshmem_b200.ops import routing
        idx, weight = routing.moe_route(s["logits"], c["K"], score=c["score"], bias=s["bias"], renormalize=c["norm"], scale=1.0, valid=s["valid"])
        if not c["back"]:
            return {"idx": idx, "weight": weight}
        return {"idx": idx, "weight": weight.detach(), "d_logits": torch.autograd.grad(weight, s["logits"], s["dw"])[0]}
    if k == "balance":
        from nvshmem_b200.ops import routing
        loss, counts = routing.balance_loss(s["logits"], s["idx"], score=c["score"], valid=s["valid"])
        return {"loss": loss.detach(), "counts": counts, "d_logits": torch.autograd.grad(loss, s["logits"], s["dloss"])[0]}
    from nvshmem_b200.ops import mxfp4
    if k == "quant":
        return mxfp4.quantize_mxfp4(s["x"]).dequantize(torch.float32)
    return mxfp4.gemm_mxfp4(s["x"], s["w"])


# ------------------------------------------------------------------ plain forms
def _rms(v):
    return torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)


def _rms_backward(v, inv, dv):
    n = v * inv
    return inv * (dv - n * (dv * n).mean(-1, keepdim=True))


def _plain_norm(s):
    c = s["case"]
    pre, pt = s["pre"].float(), s["pre"].dtype
    if c["part"] == "in":
        x = s["x"].float()
        inv = _rms(x)
        outs = {"y": (x * inv * pre).to(s["x"].dtype)}
        if c["back"]:
            dy = s["dy"].float()
            outs["d_x"] = _rms_backward(x, inv, dy * pre).to(s["x"].dtype)
            outs["d_pre"] = (dy * x * inv).sum(0).to(pt)
        return outs
    h, res, post = s["h"].float(), s["residual"].float(), s["post"].float()
    gate = None if s["gate"] is None else s["gate"].float()
    inv = _rms(h)
    z = h * inv * post
    r = A_SCALE * res + B_SCALE * (z if gate is None else gate * z)
    outs = {"r": r.to(s["residual"].dtype)}
    if c["part"] == "out_in":
        inv_r = _rms(r)
        outs["y"] = (r * inv_r * pre).to(s["h"].dtype)
    if not c["back"]:
        return outs
    g = s["dr"].float()
    if c["part"] == "out_in":
        dy = s["dy"].float()
        g = g + _rms_backward(r, inv_r, dy * pre)
    dz = B_SCALE * (g if gate is None else g * gate)
    outs["d_h"] = _rms_backward(h, inv, dz * post).to(s["h"].dtype)
    outs["d_residual"] = (A_SCALE * g).to(s["residual"].dtype)
    outs["d_post"] = (dz * h * inv).sum(0).to(pt)
    if c["part"] == "out_in":
        outs["d_pre"] = (dy * r * inv_r).sum(0).to(pt)
    if gate is not None:
        dg = B_SCALE * g * z
        outs["d_gate"] = (dg.sum(0) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "token" else dg).to(pt)
    return outs


def _scores(logits, score):
    """Scores of one row's experts, in the logits' precision here."""
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_route(s):
    c, K = s["case"], s["case"]["K"]
    p = _scores(s["logits"].double(), c["score"])             # 64 bits: neighbours in the order may be that close
    key = s["logits"].double() if s["bias"] is None else p + s["bias"].double()
    idx = key.sort(dim=-1, descending=True, stable=True).indices[:, :K]
    p = p.float()
    chosen = p.gather(-1, idx)
    total = chosen.sum(-1, keepdim=True)
    weight = chosen / total if c["norm"] else chosen
    outs = {"idx": idx.to(torch.int32), "weight": weight}
    if s["valid"] is not None:
        outs = {"idx": outs["idx"].masked_fill(~s["valid"].unsqueeze(-1), -1), "weight": weight.masked_fill(~s["valid"].unsqueeze(-1), 0.0)}
    if c["back"]:
        dw = s["dw"] if s["valid"] is None else s["dw"] * s["valid"].unsqueeze(-1)
        ds = (dw - (dw * weight).sum(-1, keepdim=True)) / total if c["norm"] else dw
        dp = torch.zeros_like(p).scatter_(-1, idx, ds)
        dl = dp * p * (1.0 - p) if c["score"] == "sigmoid" else p * (dp - (dp * p).sum(-1, keepdim=True))
        outs["d_logits"] = dl.to(s["logits"].dtype)
    return outs


def _plain_balance(s):
    c, E, K = s["case"], s["case"]["E"], s["case"]["K"]
    l = s["logits"].float()
    sc = _scores(l, c["score"])
    p = sc if c["score"] == "softmax" else sc / sc.sum(-1, keepdim=True)
    mask = torch.ones(c["T"], device=l.device) if s["valid"] is None else s["valid"].float()
    n = mask.sum().clamp(min=1.0)
    counts = (s["idx"].unsqueeze(-1) == torch.arange(E, device=l.device)).sum((0, 1)).to(torch.int32)
    f = counts.float() / (n * K)
    p = p * mask.unsqueeze(-1)
    loss = E * (f * (p.sum(0) / n)).sum()
    g = s["dloss"] * E * f / n
    dl = p * (g - (p * g).sum(-1, keepdim=True))
    if c["score"] == "sigmoid":
        dl = dl * (1.0 - sc)
    return {"loss": loss, "counts": counts, "d_logits": dl.to(s["logits"].dtype)}


def _plain_quantize(x):
    """Codes of the magnitudes (0 to 7), signs, and the exponents of the blocks' scales."""
    b = x.float().reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    exponent = ((amax.view(torch.int32) >> 23) - 129).clamp(min=-127)   # floor(log2(amax)) - 2
    a = torch.ldexp(b.abs(), -exponent)
    code = sum((a >= v if up else a > v).to(torch.uint8) for v, up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)))
    return code, b < 0, exponent


def _plain_values(q):
    code, negative, exponent = q
    v = torch.tensor(E2M1, device=code.device)[code.int()]
    return torch.ldexp(torch.where(negative, -v, v), exponent).flatten(1)


def run(s):
    if own:
        return _run_own(s)
    k = s["case"]["kind"]
    if k == "norm":
        return _plain_norm(s)
    if k == "route":
        return _plain_route(s)
    if k == "balance":
        return _plain_balance(s)
    if k == "quant":
        return _plain_values(_plain_quantize(s["x"]))
    return (_plain_values(_plain_quantize(s["x"])) @ _plain_values(s["w"]).t()).to(torch.bfloat16)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    k = case["kind"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if k == "norm":
        T, H, hs, rs, ws = case["T"], case["H"], size[case["dtype"]], size[case["res"]], size[case["wt"]]
        if case["part"] == "in":
            return {"bytes": T * H * hs * (4 if case["back"] else 2) + H * ws * (2 if case["back"] else 1), "flops": T * H * (14 if case["back"] else 4)}
        following = case["part"] == "out_in"
        gate = {"none": 0, "channel": H, "token": T, "full": T * H}[case["gate"]]
        passes = 2 if case["back"] else 1   # every input has a gradient, every output a gradient that is read
        return {"bytes": passes * (T * H * (hs + 2 * rs + (hs if following else 0)) + (H * (2 if following else 1) + gate) * ws),
                "flops": T * H * (30 if case["back"] else 12)}
    if k == "route":
        T, E, K = case["T"], case["E"], case["K"]
        b = T * E * size[case["dtype"]]
        return {"bytes": b + 8 * T * K + (b + 4 * T * K if case["back"] else 0), "flops": T * E * (8 if case["back"] else 4)}
    if k == "balance":
        T, E, K = case["T"], case["E"], case["K"]
        return {"bytes": 2 * T * E * size[case["dtype"]] + 4 * T * K + 4 * E, "flops": 10 * T * E}
    if k == "quant":
        n = case["R"] * case["K"]
        return {"bytes": n * size[case["dtype"]] + 2 * (n * 17 // 32) + 4 * n, "flops": 4 * n}
    M, N, K = case["M"], case["N"], case["K"]
    return {"bytes": 2 * M * K + N * K * 17 // 32 + 2 * M * N, "flops": 2 * M * N * K}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_norm(case, d):
    names = _leaves(case)
    v = {n: d[n].double().requires_grad_(case["back"]) for n in names}

    def norm(t, weight):
        return t / torch.sqrt((t * t).sum(-1, keepdim=True) / t.shape[-1] + EPS) * weight

    if case["part"] == "in":
        outs = {"y": norm(v["x"], v["pre"])}
    else:
        branch = norm(v["h"], v["post"]) * v.get("gate", 1.0)
        outs = {"r": v["residual"] * A_SCALE + branch * B_SCALE}
        if case["part"] == "out_in":
            outs["y"] = norm(outs["r"], v["pre"])
    if not case["back"]:
        return outs
    grads = torch.autograd.grad(list(outs.values()), [v[n] for n in names], [d["d" + n].double() for n in outs])
    return {**{n: o.detach() for n, o in outs.items()}, **{"d_" + n: g for n, g in zip(names, grads)}}


def _exact_route(case, d):
    l = d["logits"].double().requires_grad_(case["back"])
    p = torch.softmax(l, -1) if case["score"] == "softmax" else torch.sigmoid(l)
    order = p.detach() + d["bias"].double() if case["bias"] else l.detach()
    idx = torch.argsort(-order, dim=-1, stable=True)[:, :case["K"]]
    w = torch.take_along_dim(p, idx, -1)
    if case["norm"]:
        w = w / w.sum(-1, keepdim=True)
    if d["valid"] is not None:
        idx = torch.where(d["valid"][:, None], idx, -1)
        w = torch.where(d["valid"][:, None], w, 0.0)
    outs = {"idx": idx.to(torch.int32), "weight": w.detach()}
    if case["back"]:
        outs["d_logits"] = torch.autograd.grad(w, l, d["dw"].double())[0]
    return outs


def _exact_balance(case, d):
    E, K = case["E"], case["K"]
    l = d["logits"].double().requires_grad_(True)
    p = torch.softmax(l if case["score"] == "softmax" else torch.nn.functional.logsigmoid(l), -1)
    rows = d["valid"].nonzero()[:, 0] if case["mask"] else torch.arange(case["T"], device=l.device)
    n = max(1, rows.numel())
    ids = d["idx"].long().flatten()
    counts = torch.bincount(ids[ids >= 0], minlength=E)
    loss = E * (counts.double() / (n * K) @ p[rows].sum(0)) / n
    return {"loss": loss.detach(), "counts": counts.to(torch.int32), "d_logits": torch.autograd.grad(loss, l, d["dloss"].double())[0]}


def _exact_values(x):
    """Nearest multiple of the step of each value's binade (half a unit below 1), ties to the even multiple."""
    b = x.double().reshape(x.shape[0], -1, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    scale = torch.exp2((e - 3).clamp(min=-127).double())
    scale = torch.where(b.abs().amax(-1, keepdim=True) > 0, scale, 1.0)
    v = b / scale
    _, e = torch.frexp(v.abs())
    step = torch.exp2((e - 2).clamp(min=-1).double())
    return (torch.round(v / step) * step).clamp(-6.0, 6.0).mul(scale).flatten(1)


def exact(case, seed):
    d, k = _inputs(case, seed), case["kind"]
    if k == "norm":
        return _exact_norm(case, d)
    if k == "route":
        return _exact_route(case, d)
    if k == "balance":
        return _exact_balance(case, d)
    if k == "quant":
        return _exact_values(d["x"])
    return _exact_values(d["x"]) @ _exact_values(d["w"]).t()
