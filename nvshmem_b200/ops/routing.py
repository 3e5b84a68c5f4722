"""Expert router and balance loss of a mixture-of-experts layer, on the framework's own kernels (``libbshmem_fused.so``).

* :func:`moe_route` – from router logits to what :class:`~nvshmem_b200.ops.moe.MoeDispatchCombine` takes: the experts of every token
  (int32) and their weights (fp32).
* :func:`balance_loss` – the auxiliary loss that keeps the experts evenly loaded, and how many tokens each expert got.

Both are differentiable in the logits, which are ``[T, E]`` in fp32, bf16 or fp16 (rows may lie apart); up to 1024 experts, top-16.
Everything is computed in fp32.  Work is issued on the current stream; all tensors lie on the current device.
A backward pass may be captured into a CUDA graph, on leaves of which no eager autograd graph is still alive (torch ties a leaf to the stream that
used it first): drop the outputs of warm-up calls before the capture.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._launch import device_of, first_order, forward_mode, stream_of
from .fused_gemm import fused_lib

MAX_EXPERTS, MAX_TOPK = 1024, 16
SCORES = {"softmax": 0, "sigmoid": 1}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ERRORS = {1: "bad arguments", 2: "shape", 3: "CUDA launch error"}


class RoutingError(RuntimeError):
    pass


class _Args(C.Structure):
    _fields_ = [("T", C.c_int), ("E", C.c_int), ("K", C.c_int), ("type", C.c_int), ("score", C.c_int), ("renormalize", C.c_int), ("stride", C.c_int64),
                ("scale", C.c_float), ("logits", C.c_void_p), ("bias", C.c_void_p), ("valid", C.c_void_p), ("idx", C.c_void_p), ("weight", C.c_void_p),
                ("dweight", C.c_void_p), ("dlogits", C.c_void_p), ("loss", C.c_void_p), ("counts", C.c_void_p), ("coef", C.c_void_p),
                ("workspace", C.c_void_p), ("dloss", C.c_void_p)]


def _lib():
    lib = fused_lib()
    if not hasattr(lib, "_routing_ready"):
        for fn in (lib.bshmem_route, lib.bshmem_route_backward, lib.bshmem_balance, lib.bshmem_balance_backward):
            fn.restype, fn.argtypes = C.c_int, [C.POINTER(_Args), C.c_void_p]
        lib.bshmem_balance_workspace.restype, lib.bshmem_balance_workspace.argtypes = C.c_size_t, [C.c_int, C.c_int]
        lib._routing_ready = True
    return lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _launch(fn, name, logits, K, score, renormalize=0, scale=1.0, bias=None, valid=None, idx=None, weight=None, dweight=None, dlogits=None, loss=None, counts=None,
            coef=None, workspace=None, dloss=None) -> None:
    T, E = logits.shape
    a = _Args(T, E, K, _TYPES[logits.dtype], score, renormalize, logits.stride(0), scale, logits.data_ptr(), _ptr(bias), _ptr(valid), _ptr(idx), _ptr(weight), _ptr(dweight),
              _ptr(dlogits), _ptr(loss), _ptr(counts), coef, workspace, _ptr(dloss))
    st = fn(C.byref(a), stream_of(logits.get_device()))
    if st != 0:
        raise RoutingError(f"{name}: {_ERRORS.get(st, st)}")


def _route(logits, K, score, bias, renormalize, scale, valid):
    idx = logits.new_empty((logits.shape[0], K), dtype=torch.int32)
    weight = logits.new_empty((logits.shape[0], K), dtype=torch.float32)
    _launch(_lib().bshmem_route, "bshmem_route", logits, K, score, renormalize, scale, bias, valid, idx, weight)
    return idx, weight


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, K, score, bias, renormalize, scale, valid):
        idx, weight = _route(logits, K, score, bias, renormalize, scale, valid)
        ctx.save_for_backward(logits, idx, weight)
        ctx.settings = (K, score, renormalize, scale)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return idx, weight

    @staticmethod
    @first_order
    def backward(ctx, _, dweight):
        if dweight is None:
            return (None,) * 7
        logits, idx, weight = ctx.saved_tensors
        K, score, renormalize, scale = ctx.settings
        dlogits = torch.empty_like(logits, memory_format=torch.contiguous_format)
        _launch(_lib().bshmem_route_backward, "bshmem_route_backward", logits, K, score, renormalize, scale, idx=idx, weight=weight, dweight=dweight.contiguous(), dlogits=dlogits)
        return dlogits, None, None, None, None, None, None


def _balance(logits, idx, score, valid):
    T, E = logits.shape
    loss, counts = logits.new_empty((), dtype=torch.float32), logits.new_empty(E, dtype=torch.int32)
    # dloss / dp per expert (kept for backward), then the kernel's workspace
    buffer = logits.new_empty(4 * E + _lib().bshmem_balance_workspace(T, E), dtype=torch.uint8)
    at = buffer.data_ptr()
    _launch(_lib().bshmem_balance, "bshmem_balance", logits, idx.shape[1], score, valid=valid, idx=idx, loss=loss, counts=counts, coef=at, workspace=at + 4 * E)
    return loss, counts, buffer


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, score, valid):
        loss, counts, buffer = _balance(logits, idx, score, valid)
        ctx.save_for_backward(logits, buffer, valid)
        ctx.settings = (idx.shape[1], score)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @first_order
    def backward(ctx, dloss, _):
        if dloss is None:
            return None, None, None, None
        logits, buffer, valid = ctx.saved_tensors
        dlogits = torch.empty_like(logits, memory_format=torch.contiguous_format)
        _launch(_lib().bshmem_balance_backward, "bshmem_balance_backward", logits, *ctx.settings, valid=valid, dlogits=dlogits, coef=buffer.data_ptr(), dloss=dloss)
        return dlogits, None, None, None


def _check(logits, topk, score, valid) -> None:
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in _TYPES:
        raise RoutingError("logits must be a [T, E] tensor of float32, bfloat16 or float16")
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS or not 1 <= topk <= min(MAX_TOPK, E):
        raise RoutingError(f"1 to {MAX_EXPERTS} experts and 1 to {MAX_TOPK} of them per token, not {topk} of {E}")
    if T * topk >= 2 ** 31:
        raise RoutingError("too many (token, choice) pairs for 32-bit numbers")
    if score not in SCORES:
        raise RoutingError("score is 'softmax' or 'sigmoid'")
    if valid is not None and (valid.dtype != torch.bool or tuple(valid.shape) != (T,)):
        raise RoutingError(f"valid must be a bool tensor of shape {(T,)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def moe_route(logits: torch.Tensor, topk: int, score: str = "softmax", bias: torch.Tensor | None = None, renormalize: bool = True, scale: float = 1.0,
              valid: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``topk`` experts of every token and their weights: ``(idx int32 [T, topk], weight fp32 [T, topk])``, in descending order.

    ``score`` is the softmax over all experts or the sigmoid of each; the weights are the scores of the chosen experts, divided by their
    sum where ``renormalize`` is set, times ``scale``.  ``bias`` (fp32 ``[E]``) is added to the scores for the choice only: it changes
    neither weights nor gradients.  Ties go to the lowest expert.  An expert whose logit (or score + bias) is -inf or NaN is
    never chosen; a place that is left over gets expert -1, which dispatch and combine skip, and weight 0.  ``valid`` (bool ``[T]``): tokens where it is False
    get -1 and 0 everywhere and a gradient of 0.  A NaN or +inf among a token's logits makes the softmax weights of all its chosen experts NaN; the choice
    (with a bias: by the softmax over the logits that are numbers, which those of +inf share evenly) is made all the same."""
    _check(logits, topk, score, valid)
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (logits.shape[1],)):
        raise RoutingError(f"bias must be float32 of shape {(logits.shape[1],)}")
    device_of(RoutingError, logits, bias, valid)
    logits = _rows(logits)
    bias = None if bias is None else bias.detach().contiguous()
    valid = None if valid is None else valid.contiguous()
    if (torch.is_grad_enabled() and logits.requires_grad) or forward_mode():
        return _Route.apply(logits, topk, SCORES[score], bias, int(renormalize), float(scale), valid)
    return _route(logits, topk, SCORES[score], bias, int(renormalize), float(scale), valid)


def balance_loss(logits: torch.Tensor, idx: torch.Tensor, score: str = "softmax", valid: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)``: the balance loss (fp32 scalar) of the choice ``idx`` (int32 ``[T, K]``; entries outside ``[0, E)`` are skipped) and
    the tokens per expert (int32 ``[E]``)::

        loss = E * sum_e f_e P_e      f_e = counts_e / (n K),  P_e = mean of p_te over the n valid tokens

    with ``p`` the softmax of the logits, or their sigmoids divided by the token's sum.  It is 1 for an even load.  The gradient flows
    through ``p``.  Tokens where ``valid`` (bool ``[T]``) is False count nowhere; a token whose logits are all -inf has p = 0.  Without valid
    tokens the loss is 0."""
    if not isinstance(idx, torch.Tensor) or idx.dim() != 2 or idx.dtype != torch.int32:
        raise RoutingError("idx must be an int32 [T, K] tensor")
    _check(logits, idx.shape[1], score, valid)
    if idx.shape[0] != logits.shape[0]:
        raise RoutingError(f"idx is of {idx.shape[0]} tokens, logits of {logits.shape[0]}")
    device_of(RoutingError, logits, idx, valid)
    logits, idx = _rows(logits), idx.contiguous()
    valid = None if valid is None else valid.contiguous()
    if (torch.is_grad_enabled() and logits.requires_grad) or forward_mode():
        return _Balance.apply(logits, idx, SCORES[score], valid)
    return _balance(logits, idx, SCORES[score], valid)[:2]
