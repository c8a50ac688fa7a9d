"""Tensor plumbing for the C ABI: device checks, pointers, dtype codes, stream."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

_ACT = {torch.float32: _lib.QW_F32, torch.bfloat16: _lib.QW_BF16, torch.float16: _lib.QW_F16}
# 16-bit float types and the codes of their plain and tiled weight formats
HALF = {torch.bfloat16: (_lib.QW_BF16, _lib.QW_BF16T), torch.float16: (_lib.QW_F16, _lib.QW_F16T)}
FLOAT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def require_device(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda" or not torch.cuda.is_available():
        raise RuntimeError(f"{what}: the HIP MoE kernels need a ROCm (cuda) device tensor, got {t.device}")


def act_code(t: torch.Tensor, what: str) -> int:
    try:
        return _ACT[t.dtype]
    except KeyError:
        raise ValueError(f"{what}: dtype {t.dtype} is not supported (float32, bfloat16 or float16)") from None


def ptr(t: torch.Tensor | None) -> int | None:
    """Device address of a tensor for a `void*` argument (ctypes converts the
    int; None is NULL)."""
    return None if t is None else t.data_ptr()


def stream(device: torch.device) -> int:
    """The current HIP stream of `device`, for a `void* stream` argument."""
    return torch.cuda.current_stream(device).cuda_stream


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


# The current stream of a device as its handle, without a Stream object (half a
# microsecond less per call, which single-token operators notice).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(device: torch.device) -> int:
    """The current HIP stream of `device` for a `void* stream` argument."""
    return stream(device) if _raw_stream is None or device.index is None else _raw_stream(device.index)


def call_on(device: torch.device, name: str, *args) -> None:
    """An entry point called with `device` as the current one (a launch goes to
    the current device, whatever device its stream and tensors are on)."""
    if device.index is None or device.index == torch.cuda.current_device():
        _lib.call(name, *args)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args)


def refuse_tangent(t: torch.Tensor, what: str) -> None:
    """Called by an operator that hands `t` to its kernel without an autograd node:
    a forward-mode tangent of t would be lost on the way."""
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{what}: forward-mode derivatives are not supported")


_STREAM_KEY = "quantaweave stream"


def gradient_node(t: torch.Tensor) -> torch.autograd.graph.Node:
    """The node that takes t's gradient (grad mode on, `t` requiring grad), marked
    with the stream it is first seen on.  A leaf holds its node weakly: a
    differentiable operator keeps the returned one until its own node refers to it,
    or the mark is gone with it."""
    node = t.view_as(t).grad_fn.next_functions[0][0] if t.grad_fn is None else t.grad_fn
    node.metadata.setdefault(_STREAM_KEY, raw_stream(t.device))
    return node


def note_stream(t: torch.Tensor | torch.autograd.graph.Node, what: str, device: torch.device | None = None) -> None:
    """Called by a differentiable operator's backward pass with the node that its
    gradient goes to (of a tensor on `device`; or with the tensor, whose node is
    marked then).  That node is bound to the stream it was made on and lives as long
    as any graph through it does.  A backward pass recorded into a HIP graph while it
    is bound to another stream makes that stream wait inside the capture, which ends
    the process at the capture's end; so it is refused here, before the gradient is
    handed on.  It is known of nodes that these operators met before the capture;
    those that other operations alone have met carry no mark."""
    if isinstance(t, torch.Tensor):
        t, device = gradient_node(t), t.device
    here = raw_stream(device)
    if t.metadata.get(_STREAM_KEY, here) != here and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: the input still belongs to a graph made on another stream, so its backward pass "
                           "cannot be captured; drop that graph's results (or detach the input) before the capture")
