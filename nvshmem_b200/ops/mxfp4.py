"""Microscaled 4-bit floating point, on the framework's own kernels (``libbshmem_fused.so``).

* :func:`quantize_mxfp4` – a matrix ``[R, K]`` as E2M1 values with one power-of-two scale per 32 of them along K (17/32 of a byte a value).
* :meth:`MxFp4.dequantize` – the values back.
* :func:`gemm_mxfp4` – ``x @ w.T`` of two such matrices on the tensor cores' block-scaled form, accumulated in fp32; a bf16,
  fp16 or fp32 ``x`` is quantised in the call.

For serving: weights are quantised once, activations in every call, and nothing here records gradients: a tensor that requires one is refused unless the
call is under ``torch.no_grad()`` (or ``inference_mode``).  K is a multiple of 32; rows and columns of the product may be
any number.  Work is issued on the current stream; all tensors lie on the current device.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._launch import device_of, stream_of, wants_gradient
from .fused_gemm import _check_out, _error_flag, fused_lib, FusedGemmError

BLOCK = 32
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ERRORS = {1: "bad arguments", 2: "shape: K must be a multiple of 32 and below 2^26", 3: "operands must be 16-byte aligned", 4: "CUDA driver/runtime error"}


class _GemmArgs(C.Structure):
    _fields_ = [("x", C.c_void_p), ("x_scales", C.c_void_p), ("w", C.c_void_p), ("w_scales", C.c_void_p), ("out", C.c_void_p), ("M", C.c_int64), ("N", C.c_int64),
                ("K", C.c_int64), ("wait_limit_ms", C.c_uint32), ("error_flag", C.c_void_p), ("raw_x", C.c_void_p), ("raw_type", C.c_int), ("raw_stride", C.c_int64)]


def _lib():
    lib = fused_lib()
    if not hasattr(lib, "_mxfp4_ready"):
        lib.bshmem_mxfp4_scale_bytes.restype, lib.bshmem_mxfp4_scale_bytes.argtypes = C.c_size_t, [C.c_int64, C.c_int64]
        lib.bshmem_mxfp4_quantize.restype = C.c_int
        lib.bshmem_mxfp4_quantize.argtypes = [C.c_void_p, C.c_int, C.c_int64, C.c_int64, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p]
        lib.bshmem_mxfp4_dequantize.restype = C.c_int
        lib.bshmem_mxfp4_dequantize.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int, C.c_void_p, C.c_void_p]
        lib.bshmem_mxfp4_gemm.restype, lib.bshmem_mxfp4_gemm.argtypes = C.c_int, [C.POINTER(_GemmArgs), C.c_void_p]
        lib._mxfp4_ready = True
    return lib


def _raise(st: int, name: str) -> None:
    if st != 0:
        raise FusedGemmError(f"{name}: {_ERRORS.get(st, st)}")


def _scale_shape(R: int, K: int) -> tuple[int, int, int]:
    return (R + 127) // 128, (K + 255) // 256 * 2, 512


class MxFp4:
    """A matrix ``[R, K]`` in microscaled 4-bit floats.

    ``data``: uint8 ``[R, K / 2]``, two values a byte, the lower K in the low four bits.  ``scales``: uint8 ``[R / 128, K / 128, 512]`` (both
    rounded up, the second to an even number): E8M0 scales in the order of the tensor core's scale operand, row r and scale s of a block
    at ``(r % 32) * 16 + (r / 32) * 4 + s``; zero for rows and columns past the end.
    """
    __slots__ = ("data", "scales", "shape")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int]):
        R, K = shape
        if K < BLOCK or K % BLOCK:
            raise FusedGemmError(f"K must be a multiple of {BLOCK}, not {K}")
        for name, t, want in (("data", data, (R, K // 2)), ("scales", scales, _scale_shape(R, K))):
            if t.dtype != torch.uint8 or tuple(t.shape) != want or not t.is_contiguous():
                raise FusedGemmError(f"{name} must be a contiguous uint8 tensor of shape {want}")
        self.data, self.scales, self.shape = data, scales, (R, K)

    @classmethod
    def from_codes(cls, data: torch.Tensor, codes: torch.Tensor) -> "MxFp4":
        """From packed values ``[R, K / 2]`` and E8M0 scales ``[R, K / 32]`` (both uint8), the order that checkpoints use."""
        if codes.dim() != 2 or data.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[0] != data.shape[0] or codes.shape[1] * 16 != data.shape[1]:
            raise FusedGemmError(f"data {tuple(data.shape)} and codes {tuple(codes.shape)} {codes.dtype} do not belong together")
        R, S = codes.shape
        rb, kb, _ = _scale_shape(R, S * BLOCK)
        padded = torch.zeros(rb * 128, kb * 4, dtype=torch.uint8, device=codes.device)
        padded[:R, :S] = codes
        scales = padded.view(rb, 4, 32, kb, 4).permute(0, 3, 2, 1, 4).reshape(rb, kb, 512).contiguous()
        return cls(data.contiguous(), scales, (R, S * BLOCK))

    @property
    def codes(self) -> torch.Tensor:
        """E8M0 scales by row and block, uint8 ``[R, K / 32]``: scale ``2 ** (code - 127)``, 255 for NaN."""
        R, K = self.shape
        rb, kb, _ = self.scales.shape
        return self.scales.view(rb, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, kb * 4)[:R, :K // BLOCK].contiguous()

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values, ``[R, K]``.  Exact in bf16 and fp32 (of scales from 2 ** 126 on, which quantisation does not make, the largest
        elements are infinite); fp16 rounds where its range ends."""
        if dtype not in _TYPES:
            raise FusedGemmError("dtype must be bfloat16, float16 or float32")
        device = device_of(FusedGemmError, self.data, self.scales)
        R, K = self.shape
        out = self.data.new_empty((R, K), dtype=dtype)
        _raise(_lib().bshmem_mxfp4_dequantize(self.data.data_ptr(), self.scales.data_ptr(), R, K, _TYPES[dtype], out.data_ptr(), stream_of(device)),
               "bshmem_mxfp4_dequantize")
        return out


def quantize_mxfp4(x: torch.Tensor) -> MxFp4:
    """``x [R, K]`` (bf16, fp16 or fp32; rows may lie apart) in microscaled 4-bit floats.

    A block of 32 values along K gets the scale ``2 ** (floor(log2(max|x|)) - 2)``, at least ``2 ** -127``; its values are ``x / scale``
    rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to even) and saturated at 6.  A block with an infinity or a
    NaN gets the scale NaN, and so do all its values."""
    x, device = _checked(x)
    R, K = x.shape
    data = x.new_empty((R, K // 2), dtype=torch.uint8)
    scales = x.new_empty(_scale_shape(R, K), dtype=torch.uint8)
    _raise(_lib().bshmem_mxfp4_quantize(x.data_ptr(), _TYPES[x.dtype], R, K, x.stride(0), data.data_ptr(), scales.data_ptr(), stream_of(device)), "bshmem_mxfp4_quantize")
    q = MxFp4.__new__(MxFp4)   # the shapes are right by construction
    q.data, q.scales, q.shape = data, scales, (R, K)
    return q


def _no_gradient(name: str, t: torch.Tensor | None) -> None:
    if t is not None and wants_gradient(t):
        raise FusedGemmError(f"{name} requires a gradient, which 4-bit floats do not have: detach it or call under torch.no_grad()")


def _checked(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """`x` as a matrix that can be quantised, and its device."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.dtype not in _TYPES:
        raise FusedGemmError("x must be a [R, K] tensor of bfloat16, float16 or float32")
    _no_gradient("x", x)
    K = x.shape[1]
    if K < BLOCK or K % BLOCK:
        raise FusedGemmError(f"K must be a multiple of {BLOCK}, not {K}")
    device = device_of(FusedGemmError, x)
    return (x if x.stride(1) == 1 else x.contiguous()), device


def gemm_mxfp4(x: torch.Tensor | MxFp4, w: MxFp4, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x[M, K] @ w[N, K].T`` -> bf16 ``[M, N]`` on the block-scaled tensor-core path, accumulated in fp32 and rounded once.  An
    ``x`` that is not quantised yet is quantised in the call (:func:`quantize_mxfp4`).  M and N may be any number.  The sum over K is
    divided by a rule on M, N and K, so the last bits of a row may differ with the number of rows in the call; the same call gives the same bits."""
    if not isinstance(w, MxFp4):
        raise FusedGemmError("w must be quantised (quantize_mxfp4)")
    raw = not isinstance(x, MxFp4)
    if raw:
        x, _ = _checked(x)
    (M, K), N = x.shape, w.shape[0]
    if K != w.shape[1]:
        raise FusedGemmError(f"shape mismatch: x {tuple(x.shape)} w {w.shape}")
    dev = w.data.device
    if raw:
        device = device_of(FusedGemmError, w.data, w.scales, out)
        # room for x as it is quantised: the values, then the scales
        rb, kb, _ = _scale_shape(M, K)
        room = w.data.new_empty((M * K // 2 + 127) // 128 * 128 + rb * kb * 512)
        data = room.data_ptr()
        operand = data, data + (M * K // 2 + 127) // 128 * 128
        source = x.data_ptr(), _TYPES[x.dtype], x.stride(0)
    else:
        device = device_of(FusedGemmError, x.data, x.scales, w.data, w.scales, out)
        operand, source = (x.data.data_ptr(), x.scales.data_ptr()), (None, 0, 0)
    if out is None:
        out = w.data.new_empty((M, N), dtype=torch.bfloat16)
    else:
        _no_gradient("out", out)
        _check_out(out, M, N)
    a = _GemmArgs(*operand, w.data.data_ptr(), w.scales.data_ptr(), out.data_ptr(), M, N, K, 0, _error_flag(dev).data_ptr(), *source)
    _raise(_lib().bshmem_mxfp4_gemm(C.byref(a), stream_of(device)), "bshmem_mxfp4_gemm")
    return out
