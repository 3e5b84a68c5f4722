"""Norms around a block, on the framework's own kernels (``libbshmem_fused.so``).

* :func:`rms_norm` – the norm before a block.
* :func:`block_norms` – what lies between two blocks in one pass: the norm after the first one, its gate, the scaled
  residual, and the norm before the next one.

Both are differentiable in every tensor argument.  Rows are ``[T, H]`` in bf16, fp16 or fp32 with ``H <= 16384``; statistics and
sums over rows are kept in fp32 and every result is rounded once.  The residual stream may be fp32 beside 16-bit blocks, and so may
the parameters.  Gradients that are sums over rows are added in a fixed order.  Work is issued on the current stream; all tensors lie
on the current device.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._launch import device_of, first_order, stream_of
from .fused_gemm import _error_flag, fused_lib

MAX_H = 16384
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NONE, _CHANNEL, _TOKEN, _FULL = range(4)
_ERRORS = {1: "bad arguments", 2: "shape", 3: "CUDA launch error"}


class NormError(RuntimeError):
    pass


class _Args(C.Structure):
    _fields_ = [("T", C.c_int), ("H", C.c_int), ("type", C.c_int), ("res_type", C.c_int), ("wt_type", C.c_int), ("gate_mode", C.c_int),
                ("h_stride", C.c_int64), ("res_stride", C.c_int64), ("gate_stride", C.c_int64), ("dr_stride", C.c_int64), ("dy_stride", C.c_int64),
                ("residual_scale", C.c_float), ("branch_scale", C.c_float), ("eps", C.c_float), ("weight_offset", C.c_float),
                ("h", C.c_void_p), ("residual", C.c_void_p), ("post", C.c_void_p), ("pre", C.c_void_p), ("gate", C.c_void_p),
                ("r", C.c_void_p), ("y", C.c_void_p), ("stat", C.c_void_p), ("dr", C.c_void_p), ("dy", C.c_void_p),
                ("dh", C.c_void_p), ("dresidual", C.c_void_p), ("dpost", C.c_void_p), ("dpre", C.c_void_p), ("dgate", C.c_void_p), ("error_flag", C.c_void_p), ("partials", C.c_void_p)]


def _lib():
    lib = fused_lib()
    if not hasattr(lib, "_norms_ready"):
        for fn in (lib.bshmem_block_norms, lib.bshmem_block_norms_backward):
            fn.restype, fn.argtypes = C.c_int, [C.POINTER(_Args), C.c_void_p]
        lib.bshmem_block_norms_partials.restype, lib.bshmem_block_norms_partials.argtypes = C.c_size_t, [C.c_int, C.c_int]
        lib._norms_ready = True
    return lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with neighbouring values of a row next to one another."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


class _Plan:
    """The settings of a call: everything that is not a tensor."""
    __slots__ = ("T", "H", "device", "gate_mode", "residual_scale", "branch_scale", "eps", "weight_offset", "dtype")

    def launch(self, fn, name, h, residual, post, pre, gate, r=None, y=None, stat=None, dr=None, dy=None, dh=None, dresidual=None, dpost=None, dpre=None,
               dgate=None, partials=None) -> None:
        wt = post if post is not None else pre if pre is not None else gate
        t = _TYPES[self.dtype]
        a = _Args(self.T, self.H, t, _TYPES[residual.dtype], t if wt is None else _TYPES[wt.dtype], self.gate_mode, 0 if h is None else h.stride(0), residual.stride(0),
                  gate.stride(0) if self.gate_mode == _FULL else 0, 0 if dr is None else dr.stride(0), 0 if dy is None else dy.stride(0), self.residual_scale,
                  self.branch_scale, self.eps, self.weight_offset, _ptr(h), residual.data_ptr(), _ptr(post), _ptr(pre), _ptr(gate), _ptr(r), _ptr(y), _ptr(stat),
                  _ptr(dr), _ptr(dy), _ptr(dh), _ptr(dresidual), _ptr(dpost), _ptr(dpre), _ptr(dgate), _error_flag(residual.device).data_ptr(), _ptr(partials))
        st = fn(C.byref(a), stream_of(self.device))
        if st != 0:
            raise NormError(f"{name}: {_ERRORS.get(st, st)}")


def _forward(plan: _Plan, h, residual, post, pre, gate, want_r: bool, want_stat: bool):
    r = _dense_like(residual) if want_r else None
    y = _dense_like(residual if h is None else h) if pre is not None else None
    stat = residual.new_empty((2, plan.T), dtype=torch.float32) if want_stat else None
    plan.launch(_lib().bshmem_block_norms, "bshmem_block_norms", h, residual, post, pre, gate, r, y, stat)
    return r, y, stat


def _backward(plan: _Plan, h, residual, post, pre, gate, stat, dr, dy, needs):
    """Gradients of (h, residual, post, pre, gate), None where `needs` is false."""
    grads = [_dense_like(t) if need and t is not None else None for t, need in zip((h, residual, post, pre, gate), needs)]
    dh, dres, dpost, dpre, dgate = grads
    if plan.T == 0 or (dr is None and dy is None):
        return [g if g is None else g.zero_() for g in grads]
    if dy is None and dpre is not None:
        dpre.zero_()
    partials = None
    if dpost is not None or dpre is not None or (dgate is not None and plan.gate_mode == _CHANNEL):
        partials = residual.new_empty(_lib().bshmem_block_norms_partials(plan.T, plan.H), dtype=torch.float32)
    plan.launch(_lib().bshmem_block_norms_backward, "bshmem_block_norms_backward", h, residual, post, pre, gate, None, None, stat, None if dr is None else _rows(dr),
                None if dy is None else _rows(dy), dh, dres, dpost, None if dy is None else dpre, dgate, partials)
    return grads


class _BlockNorms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan: _Plan, want_r: bool, h, residual, post, pre, gate):
        r, y, stat = _forward(plan, h, residual, post, pre, gate, want_r, True)
        ctx.plan = plan
        ctx.want_r = want_r
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, residual, post, pre, gate, stat)
        outs = [t for t in (r, y) if t is not None]
        return tuple(outs) if len(outs) > 1 else outs[0]

    @staticmethod
    @first_order
    def backward(ctx, *grads):
        h, residual, post, pre, gate, stat = ctx.saved_tensors
        grads = list(grads)
        dr = grads.pop(0) if ctx.want_r else None
        dy = grads.pop(0) if pre is not None else None
        return (None, None, *_backward(ctx.plan, h, residual, post, pre, gate, stat, dr, dy, ctx.needs_input_grad[2:]))


def _check_rows(name: str, t: torch.Tensor, shape) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise NormError(f"{name} must be a [T, H] tensor" + (f" of shape {tuple(shape)}" if shape is not None else ""))
    if t.dtype not in _TYPES:
        raise NormError(f"{name} must be bfloat16, float16 or float32, not {t.dtype}")
    if t.shape[0] >= 2 ** 31 or not 1 <= t.shape[1] <= MAX_H:
        raise NormError(f"fewer than 2^31 rows of 1 to {MAX_H} values, not {tuple(t.shape)}")


def _check_weights(plan: _Plan, **weights) -> None:
    seen = None
    for name, w in weights.items():
        if w is None:
            continue
        if w.dtype not in (plan.dtype, torch.float32):
            raise NormError(f"{name} must be {plan.dtype} or float32")
        if seen is not None and w.dtype != seen:
            raise NormError("the weights and the gate must be of one type")
        seen = w.dtype
        if name != "gate" and tuple(w.shape) != (plan.H,):
            raise NormError(f"{name} must be of shape {(plan.H,)}")


def _run(plan: _Plan, want_r: bool, h, residual, post, pre, gate):
    tensors = (h, residual, post, pre, gate)
    plan.device = device_of(NormError, *tensors)
    residual = _rows(residual)
    h = None if h is None else _rows(h)
    if post is not None:
        post = post.contiguous()
    if pre is not None:
        pre = pre.contiguous()
    if gate is not None:
        gate = _rows(gate) if plan.gate_mode == _FULL else gate.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        out = _BlockNorms.apply(plan, want_r, h, residual, post, pre, gate)
        if want_r and pre is not None:
            return out
        return (out, None) if want_r else (None, out)
    return _forward(plan, h, residual, post, pre, gate, want_r, False)[:2]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, weight_offset: float = 0.0) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * (weight + weight_offset)`` row by row: ``x [T, H]``, ``weight [H]`` of x's type or fp32;
    the result has x's type.  Rows may lie apart (any stride between rows)."""
    _check_rows("x", x, None)
    plan = _Plan()
    plan.T, plan.H = x.shape
    plan.dtype, plan.gate_mode = x.dtype, _NONE
    plan.residual_scale, plan.branch_scale, plan.eps, plan.weight_offset = 1.0, 1.0, float(eps), float(weight_offset)
    if weight is None:
        raise NormError("weight must be given")
    _check_weights(plan, weight=weight)
    return _run(plan, False, None, x, None, weight, None)[1]


def block_norms(h: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None,
                gate: torch.Tensor | None = None, residual_scale: float = 1.0, branch_scale: float = 1.0, eps: float = 1e-6,
                weight_offset: float = 0.0) -> tuple[torch.Tensor, torch.Tensor | None]:
    """What lies between two blocks, row by row over ``[T, H]``::

        z = norm(h) * (post_weight + weight_offset)                   # the block's output h; z = h without post_weight
        r = residual_scale * residual + branch_scale * gate * z       # the new residual stream
        y = norm(r) * (pre_weight + weight_offset)                    # the next block's input; None without pre_weight

    with ``norm(v) = v * rsqrt(mean(v^2) + eps)``; returns ``(r, y)``, ``r`` of the residual's type and ``y`` of h's.  ``residual`` is
    of h's type or fp32; the weights and the gate are all of h's type or all fp32.  ``gate`` is None, one value per channel ``[H]``,
    per token ``[T, 1]``, or ``[T, H]``.  ``y`` is computed from ``r`` before its rounding."""
    _check_rows("h", h, None)
    _check_rows("residual", residual, h.shape)
    plan = _Plan()
    plan.T, plan.H = h.shape
    plan.dtype = h.dtype
    if residual.dtype not in (h.dtype, torch.float32):
        raise NormError(f"residual must be {h.dtype} or float32")
    _check_weights(plan, post_weight=post_weight, pre_weight=pre_weight, gate=gate)
    if gate is None:
        plan.gate_mode = _NONE
    elif tuple(gate.shape) == (plan.H,):
        plan.gate_mode = _CHANNEL
    elif tuple(gate.shape) == (plan.T, 1):
        plan.gate_mode = _TOKEN
    elif tuple(gate.shape) == (plan.T, plan.H):
        plan.gate_mode = _FULL
    else:
        raise NormError(f"gate must be of shape {(plan.H,)}, {(plan.T, 1)} or {(plan.T, plan.H)}, not {tuple(gate.shape)}")
    plan.residual_scale, plan.branch_scale = float(residual_scale), float(branch_scale)
    plan.eps, plan.weight_offset = float(eps), float(weight_offset)
    return _run(plan, True, h, residual, post_weight, pre_weight, gate)
