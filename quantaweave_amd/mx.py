"""Microscaled 4-bit floating point: quantisation, the product with a
microscaled matrix, and the SwiGLU experts on microscaled weights.

A row is stored as blocks of 32 numbers: 4-bit codes (sign, two exponent bits,
one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one 8-bit power of two per
block.  ``codes`` is uint8 [..., rows, padded / 2] (the even column in the low
nibble), ``scales`` uint8 [..., rows, padded / 32] (the scale is
2^(s - 127), 255 is NaN), with the columns padded to whole 128 by zeros.  The
products multiply such rows on the matrix cores as they are: 4.25 bits per
weight are read and nothing is widened on the way.

Activations are quantised by the same rule on their way into a product, so a
product of ``x`` is the product of the values that ``mx_quantize(x)`` stands
for, summed in fp32 and rounded once to ``x``'s type.  No counterpart in the
reference, whose 4-bit weights are integers (src/quantization.py:21-75).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _hip, _lib

BLOCK = 32   # columns that share a scale
STEP = 128   # stored columns are padded to whole steps of the matrix instruction


def padded_cols(cols: int) -> int:
    """Stored columns of a row of `cols` numbers."""
    return -(-cols // STEP) * STEP


def _rows(x: Tensor, what: str) -> tuple[Tensor, int]:
    """x as [rows, cols] with unit column stride (a view where its strides allow), and its row stride."""
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"{what}: rows of at least one column are needed, got shape {tuple(x.shape)}")
    if x.requires_grad:
        x = x.detach()
    flat = x if x.dim() == 2 else x.reshape(-1, x.size(-1))
    rows, cols = flat.shape
    step, unit = flat.stride()
    if unit != 1 and cols > 1 or step < 0:
        flat = flat.contiguous()
        step = cols
    return flat, step if rows > 1 else cols


def _device(x: Tensor, what: str) -> torch.device:
    if not x.is_cuda:
        _hip.require_device(x, what)
    return x.device


def _stored(codes: Tensor, scales: Tensor, dims: int, cols: int, device: torch.device, what: str) -> tuple[Tensor, Tensor]:
    """Checks a stored matrix (or stack): shapes, types, device; contiguous and aligned for the kernels."""
    p = padded_cols(cols)
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise ValueError(f"{what}: codes and scales are uint8, got {codes.dtype} and {scales.dtype}")
    shape, of = codes.shape, scales.shape
    if len(shape) != dims or shape[-1] != p // 2:
        raise ValueError(f"{what}: codes of {cols} columns have {dims} dimensions and {p // 2} bytes a row, "
                         f"got shape {tuple(shape)}")
    if len(of) != dims or of[-1] != p // BLOCK or of[:-1] != shape[:-1]:
        raise ValueError(f"{what}: scales have shape {(*shape[:-1], p // BLOCK)}, got {tuple(of)}")
    if codes.device != device or scales.device != device:
        raise ValueError(f"{what}: codes and scales must be on {device}")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 16:
        codes = codes.clone()
    if scales.data_ptr() % 4:
        scales = scales.clone()
    return codes, scales


def mx_quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """(codes, scales) of the rows of x [..., cols] (float32, bfloat16 or float16).

    Per block: scale 2^(floor(log2 max|x|) - 2), at least 2^-127; x / scale
    rounded to the nearest code, ties to the even one, saturating at 6.  A
    block holding an infinity or a NaN becomes NaN.  Not differentiable."""
    dev = _device(x, "mx_quantize")
    act = _hip.act_code(x, "mx_quantize")
    flat, stride = _rows(x, "mx_quantize")
    rows, cols = flat.shape
    p = padded_cols(cols)
    codes = torch.empty((*x.shape[:-1], p // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((*x.shape[:-1], p // BLOCK), dtype=torch.uint8, device=dev)
    if rows:
        _hip.call_on(dev, "qw_mx_quantize", _hip.ptr(flat), act, rows, cols, stride, _hip.ptr(codes),
                     _hip.ptr(scales), _hip.raw_stream(dev))
    return codes, scales


def mx_dequantize(codes: Tensor, scales: Tensor, cols: int, dtype: torch.dtype = torch.float32) -> Tensor:
    """The values [..., cols] that codes and scales stand for, rounded once to `dtype`."""
    dev = _device(codes, "mx_dequantize")
    if cols < 1 or codes.dim() < 1:
        raise ValueError(f"mx_dequantize: cols must be positive, got {cols} and codes of shape {tuple(codes.shape)}")
    codes, scales = _stored(codes, scales, codes.dim(), cols, dev, "mx_dequantize")
    out = torch.empty((*codes.shape[:-1], cols), dtype=dtype, device=dev)
    act = _hip.act_code(out, "mx_dequantize")
    rows = codes.numel() // codes.size(-1)
    if rows:
        _hip.call_on(dev, "qw_mx_dequantize", _hip.ptr(codes), _hip.ptr(scales), rows, cols, _hip.ptr(out),
                     act, _hip.raw_stream(dev))
    return out


def _matmul(x: Tensor, codes: Tensor, scales: Tensor) -> Tensor:
    flat, stride = _rows(x, "mx_matmul")
    (rows, k), n = flat.shape, codes.size(0)
    dev = flat.device
    out = torch.empty((*x.shape[:-1], n), dtype=flat.dtype, device=dev)
    if rows and n:
        act, at = _hip.act_code(flat, "mx_matmul"), _hip.ptr(flat)
        nbytes = _lib.load().qw_mx_matmul_workspace_bytes(at, act, stride, rows, n, k)
        ws = _hip.workspace(nbytes, dev) if nbytes else None
        _hip.call_on(dev, "qw_mx_matmul", at, act, stride, rows, _hip.ptr(codes), _hip.ptr(scales), n, k,
                     _hip.ptr(out), _hip.ptr(ws), nbytes, _hip.raw_stream(dev))
    return out


class _MxMatmul(torch.autograd.Function):
    """mx_matmul with the gradient of its rows: grad_x = grad_out @ W, the
    rounding of x to microscaled values passing the gradient on unchanged.
    The stored matrix is whole numbers and gets none."""

    @staticmethod
    def forward(ctx, x: Tensor, codes: Tensor, scales: Tensor) -> Tensor:
        ctx.save_for_backward(codes, scales)
        ctx.shape, ctx.dtype = x.shape, x.dtype
        return _matmul(x, codes, scales)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        if not ctx.needs_input_grad[0]:
            return None, None, None
        _hip.note_stream(ctx.next_functions[0][0], "mx_matmul", grad.device)
        codes, scales = ctx.saved_tensors
        grad = grad.to(ctx.dtype).contiguous()
        if grad.data_ptr() % 16:
            grad = grad.clone()  # the matrix cores' loads
        gx = torch.empty(ctx.shape, dtype=ctx.dtype, device=grad.device)
        n, k = codes.size(0), ctx.shape[-1]
        rows = gx.numel() // k
        if rows and n:
            act = _hip.act_code(grad, "mx_matmul")
            nbytes = _lib.load().qw_mx_matmul_backward_workspace_bytes(rows, n, k, act)
            ws = _hip.workspace(nbytes, grad.device)
            _hip.call_on(grad.device, "qw_mx_matmul_backward", _hip.ptr(grad), act, rows, _hip.ptr(codes),
                         _hip.ptr(scales), n, k, _hip.ptr(gx), _hip.ptr(ws), nbytes, _hip.raw_stream(grad.device))
        else:
            gx.zero_()
        return gx, None, None


def mx_matmul(x: Tensor, codes: Tensor, scales: Tensor) -> Tensor:
    """x [..., in] times a stored matrix [out, in], transposed: [..., out] of x's type.

    x (float32, bfloat16 or float16) is quantised on the way; the sum is fp32,
    rounded once.  Differentiable in x (the stored matrix takes no gradient):
    grad_x = grad_out @ W, summed in fp32 and rounded once, with stored values
    of 2^128 and more (scales 253 and 254) infinite.  Second and forward-mode
    derivatives are refused."""
    dev = _device(x, "mx_matmul")
    _hip.act_code(x, "mx_matmul")
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"mx_matmul: rows of at least one column are needed, got shape {tuple(x.shape)}")
    _hip.refuse_tangent(x, "mx_matmul")
    codes, scales = _stored(codes, scales, 2, x.size(-1), dev, "mx_matmul")
    if x.requires_grad and torch.is_grad_enabled():
        node = _hip.gradient_node(x)  # held until the result's graph holds it
        return _MxMatmul.apply(x, codes, scales)
    return _matmul(x, codes, scales)


def mx_grouped_swiglu(x: Tensor, gate: tuple, up: tuple, down: tuple, offsets: Tensor,
                      max_rows: Optional[int] = None) -> Tensor:
    """SwiGLU experts over expert-sorted rows: expert e's rows are x[offsets[e]:offsets[e + 1]].

    x [rows, d]; gate and up (codes, scales) stacks [experts, ffn, d], down
    [experts, d, ffn]; offsets int32 [experts + 1] on x's device, ascending from
    0 (rows past the last offset give zeros); max_rows bounds an expert's rows
    (None: unknown) and only chooses the height of the tiles that more than
    sixteen rows an expert on average go to.  x and the hidden rows
    silu(gate) * up are quantised on the way, sums are fp32, the result is
    rounded once to x's type.  Not differentiable."""
    what = "mx_grouped_swiglu"
    _device(x, what)
    act = _hip.act_code(x, what)
    if x.dim() != 2 or x.size(1) < 1:
        raise ValueError(f"{what}: x is [rows, d], got shape {tuple(x.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("gradients through quantised experts are not supported")
    _hip.refuse_tangent(x, what)
    d = x.size(1)
    gate, up = (_stored(*m, 3, d, x.device, f"{what} {n}") for m, n in ((gate, "gate"), (up, "up")))
    experts, ffn = gate[0].shape[:2]
    if experts < 1 or ffn < 1 or up[0].shape != gate[0].shape:
        raise ValueError(f"{what}: gate and up have one shape, got {tuple(gate[0].shape)} and {tuple(up[0].shape)}")
    down = _stored(*down, 3, ffn, x.device, f"{what} down")
    if tuple(down[0].shape[:2]) != (experts, d):
        raise ValueError(f"{what}: down is [{experts}, {d}, ...], got shape {tuple(down[0].shape)}")
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (experts + 1,) or offsets.device != x.device:
        raise ValueError(f"{what}: offsets are int32 [{experts + 1}] on {x.device}")
    if max_rows is not None and max_rows < 0:
        raise ValueError(f"{what}: max_rows must be >= 0")
    flat, stride = _rows(x, what)
    rows = flat.size(0)
    out = torch.empty(rows, d, dtype=x.dtype, device=x.device)
    if rows:
        offsets = offsets.contiguous()
        nbytes = _lib.load().qw_mx_experts_workspace_bytes(rows, experts, d, ffn)
        ws = _hip.workspace(nbytes, x.device)
        _hip.call_on(x.device, "qw_mx_experts", _hip.ptr(flat), act, stride, _hip.ptr(offsets), experts, d, ffn, rows,
                     min(max_rows or 0, rows), _hip.ptr(gate[0]), _hip.ptr(gate[1]), _hip.ptr(up[0]),
                     _hip.ptr(up[1]), _hip.ptr(down[0]), _hip.ptr(down[1]), 1, _hip.ptr(out), _hip.ptr(ws), nbytes,
                     _hip.raw_stream(x.device))
    return out
