"""Norms around a block, on the framework's own kernels (``libbshmem_fused.so``).

* :func:`rms_norm` – the norm before a block.
* :func:`block_norms` – what lies between two blocks in one pass: the norm after the first one, its gate, the scaled
  residual, and the norm before the next one.

Both are differentiable in every tensor argument.  Rows are ``[T, H]`` in bf16, fp16 or fp32 with ``H <= 16384``; statistics and
sums over rows are kept in fp32 and every result is rounded once.  The residual stream may be fp32 beside 16-bit blocks, and so may
the parameters.  Gradients that are sums over rows are added in a fixed order.  Work is issued on the current stream; all tensors lie
on the current device.
A backward pass may be captured into a CUDA graph, on leaves of which no eager autograd graph is still alive (torch ties a leaf to the stream that
used it first): drop the outputs of warm-up calls before the capture.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._launch import device_of, first_order, forward_mode, stream_of
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
    """The settings of a call: everything that is not a tensor.  `head`: the first six fields of the C arguments."""
    __slots__ = ("T", "H", "device", "gate_mode", "head", "scales")

    def strides(self, h, residual, gate):
        return 0 if h is None else h.stride(0), residual.stride(0), gate.stride(0) if self.gate_mode == _FULL else 0

    def launch(self, fn, a: _Args, name: str) -> None:
        st = fn(C.byref(a), stream_of(self.device))
        if st != 0:
            raise NormError(f"{name}: {_ERRORS.get(st, st)}")


def _forward(plan: _Plan, h, residual, post, pre, gate, want_r: bool, want_stat: bool):
    r = _dense_like(residual) if want_r else None
    y = _dense_like(residual if h is None else h) if pre is not None else None
    stat = residual.new_empty((2, plan.T), dtype=torch.float32) if want_stat else None
    a = _Args(*plan.head, *plan.strides(h, residual, gate), 0, 0, *plan.scales, _ptr(h), residual.data_ptr(), _ptr(post), _ptr(pre), _ptr(gate), _ptr(r), _ptr(y), _ptr(stat),
              0, 0, 0, 0, 0, 0, 0, _error_flag(residual.device).data_ptr(), 0)
    plan.launch(_lib().bshmem_block_norms, a, "bshmem_block_norms")
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
    if dr is not None:
        dr = _rows(dr)
    if dy is not None:
        dy = _rows(dy)
    a = _Args(*plan.head, *plan.strides(h, residual, gate), 0 if dr is None else dr.stride(0), 0 if dy is None else dy.stride(0), *plan.scales, _ptr(h), residual.data_ptr(),
              _ptr(post), _ptr(pre), _ptr(gate), 0, 0, stat.data_ptr(), _ptr(dr), _ptr(dy), _ptr(dh), _ptr(dres), _ptr(dpost), 0 if dy is None else _ptr(dpre), _ptr(dgate),
              _error_flag(residual.device).data_ptr(), _ptr(partials))
    plan.launch(_lib().bshmem_block_norms_backward, a, "bshmem_block_norms_backward")
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


def _check_rows(name: str, t: torch.Tensor) -> tuple[int, int]:
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.dtype not in _TYPES:
        raise NormError(f"{name} must be a [T, H] tensor of bfloat16, float16 or float32")
    T, H = t.shape
    if T >= 2 ** 31 or not 1 <= H <= MAX_H:
        raise NormError(f"fewer than 2^31 rows of 1 to {MAX_H} values, not {(T, H)}")
    return T, H


def _settings(h, residual, post, pre, gate, T, H, gate_mode, residual_scale, branch_scale, eps, weight_offset) -> _Plan:
    """The plan of a call, after a look at the parameters' types and shapes."""
    dtype, wt = (residual if h is None else h).dtype, None
    for name, w in (("the weight after the block", post), ("the weight before the block", pre), ("gate", gate)):
        if w is None:
            continue
        if w.dtype is not dtype and w.dtype is not torch.float32:
            raise NormError(f"{name} must be {dtype} or float32, not {w.dtype}")
        if wt is not None and w.dtype is not wt:
            raise NormError("the weights and the gate must be of one type")
        wt = w.dtype
        if name != "gate" and (w.dim() != 1 or w.shape[0] != H):
            raise NormError(f"{name} must be of shape {(H,)}, not {tuple(w.shape)}")
    plan = _Plan()
    plan.T, plan.H, plan.gate_mode = T, H, gate_mode
    plan.head = T, H, _TYPES[dtype], _TYPES[residual.dtype], _TYPES[wt or dtype], gate_mode
    plan.scales = float(residual_scale), float(branch_scale), float(eps), float(weight_offset)
    return plan


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
    if (torch.is_grad_enabled() and (residual.requires_grad or any([t is not None and t.requires_grad for t in tensors]))) or forward_mode():
        out = _BlockNorms.apply(plan, want_r, h, residual, post, pre, gate)
        if want_r and pre is not None:
            return out
        return (out, None) if want_r else (None, out)
    return _forward(plan, h, residual, post, pre, gate, want_r, False)[:2]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, weight_offset: float = 0.0) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * (weight + weight_offset)`` row by row: ``x [T, H]``, ``weight [H]`` of x's type or fp32;
    the result has x's type.  Rows may lie apart (any stride between rows)."""
    T, H = _check_rows("x", x)
    if weight is None:
        raise NormError("weight must be given")
    return _run(_settings(None, x, None, weight, None, T, H, _NONE, 1.0, 1.0, eps, weight_offset), False, None, x, None, weight, None)[1]


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
    T, H = _check_rows("h", h)
    if not isinstance(residual, torch.Tensor) or residual.shape != h.shape or (residual.dtype is not h.dtype and residual.dtype is not torch.float32):
        raise NormError(f"residual must be a tensor of shape {(T, H)} in {h.dtype} or float32")
    if gate is None:
        mode = _NONE
    else:
        shape = tuple(gate.shape)
        mode = _CHANNEL if shape == (H,) else _TOKEN if shape == (T, 1) else _FULL if shape == (T, H) else None
        if mode is None:
            raise NormError(f"gate must be of shape {(H,)}, {(T, 1)} or {(T, H)}, not {shape}")
    plan = _settings(h, residual, post_weight, pre_weight, gate, T, H, mode, residual_scale, branch_scale, eps, weight_offset)
    return _run(plan, True, h, residual, post_weight, pre_weight, gate)
