"""What every call of an operator needs: the device of its tensors, the stream, and a backward that is differentiable once.

The calls take a few microseconds on the GPU, so the host's share counts: each helper asks torch once."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def device_of(error: type[Exception], *tensors: torch.Tensor | None) -> int:
    """Index of the current device, on which all of `tensors` (Nones aside) have to lie."""
    here = _current_device() if torch.cuda.is_initialized() else None
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise error("tensors must be on the GPU" if not t.is_cuda else "tensors must be on the current device")
    return here


def stream_of(device: int) -> int:
    """Handle of the device's current stream."""
    return _current_stream(device)


def forward_mode() -> bool:
    """Whether tangents may be about (``torch.autograd.forward_ad``): a call then goes by its autograd function, which refuses them."""
    return _forward_ad._current_level >= 0


def wants_gradient(t: torch.Tensor) -> bool:
    """Whether a derivative with respect to `t` is being asked for, in reverse or forward mode."""
    return (t.requires_grad and torch.is_grad_enabled()) or (forward_mode() and _forward_ad.unpack_dual(t).tangent is not None)


def first_order(backward):
    """`backward` of an autograd function whose kernels record no graph.  A graph of the gradients (create_graph) may be asked for; going
    through it raises, as with ``once_differentiable``, whose wrapper takes 5 us a call and is entered only then."""
    recorded = once_differentiable(backward)

    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run
