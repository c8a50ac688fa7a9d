"""Microscaled 4-bit numbers, their product and experts, and the scored routing
in 64 bits on the CPU, straight from the definitions."""

from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
MID = (GRID[1:] + GRID[:-1]) / 2
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # the smallest subnormal
EPS24 = 2.0 ** -24


def padded(cols: int) -> int:
    return -(-cols // 128) * 128


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes as whole numbers 0..15 [rows, padded], scale bytes [rows, padded / 32]) of x [rows, cols]."""
    v = x.detach().cpu().double()
    rows, cols = v.shape
    v = torch.cat((v, v.new_zeros(rows, padded(cols) - cols)), 1).view(rows, padded(cols) // 32, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad.unsqueeze(-1), 0.0, v)
    top = v.abs().amax(-1)
    exponent = torch.frexp(top)[1].double() - 1  # floor(log2)
    byte = torch.where(top > 0, (exponent - 2 + 127).clamp(min=0), 0.0)
    a = v.abs() / torch.exp2(byte - 127).unsqueeze(-1)
    up = torch.bucketize(a, MID, right=False)    # codes below a midpoint keep it out: ties down
    down = torch.bucketize(a, MID, right=True)   # ties up
    code = torch.where(up % 2 == 0, up, down)    # of the two, the even one
    code = code + 8 * torch.signbit(v)
    byte = torch.where(bad, 255.0, byte)
    return code.flatten(1).to(torch.uint8), byte.to(torch.uint8)


def pack(code: torch.Tensor) -> torch.Tensor:
    return code[..., 0::2] | (code[..., 1::2] << 4)


def values(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    """The numbers [..., cols] that stored codes and scales stand for, in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu()
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = torch.where(n >= 8, -1.0, 1.0).double() * GRID[n & 7]
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)[..., :cols]


def on_grid(x: torch.Tensor) -> torch.Tensor:
    code, byte = quantize(x)
    return values(pack(code), byte, x.size(1))


def stored(gen: torch.Generator, *shape, low: int = 118, high: int = 122) -> tuple[torch.Tensor, torch.Tensor]:
    """A random stored matrix [..., out, cols] with zero padding."""
    *lead, cols = shape
    p = padded(cols)
    code = torch.randint(0, 16, (*lead, p), generator=gen, dtype=torch.uint8)
    code[..., cols:] = 0
    return pack(code), torch.randint(low, high, (*lead, p // 32), generator=gen, dtype=torch.uint8)


def rows(gen: torch.Generator, n: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    x = torch.randn(n, cols, generator=gen) * torch.exp2(torch.randn(cols, generator=gen))
    return x.to(dtype)


def matmul(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(result, allowed error before the rounding to the output type): exact
    products, at most cols + 8 additions in fp32."""
    cols = x.size(1)
    a, w = on_grid(x), values(codes, scales, cols)
    return a @ w.t(), (padded(cols) + 8) * EPS24 * (a.abs() @ w.abs().t())


def allowed(y: torch.Tensor, err: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """err and the rounding of a value within err of y to `dtype`."""
    return err + HALF[dtype] * (y.abs() + err) + TINY[dtype]


def swiglu(x: torch.Tensor, gate, up, down) -> tuple[torch.Tensor, torch.Tensor]:
    """One expert: (y, allowed error before the last rounding).

    The hidden row is quantised from fp32 sums, so an entry whose exact value
    lies within the sums' error of a midpoint of the grid may take the code on
    its other side, one step away; and a block whose largest entry lies within
    it of a power of two may take the other scale, whose grid is at most twice
    as coarse (entries then move by at most a step of the coarser grid, 2 scale
    units times 2).  Everything else has to be the exact code."""
    g, ge = matmul(x, *gate)
    u, ue = matmul(x, *up)
    s = torch.sigmoid(g)
    h = g * s * u
    # |silu'| <= 1.1; silu itself in fp32: exp of an argument rounded to 2^-24 |g| (relative error up to
    # |g| 2^-23), two roundings, a reciprocal of one step, two products
    silu_err = 1.1 * ge + (g.abs() + 8) * 2.0 ** -23 * (g * s).abs()
    he = silu_err * (u.abs() + ue) + (g * s).abs() * ue + 2.0 ** -24 * h.abs() + 2.0 ** -149
    n, cols = h.shape
    pad = padded(cols) - cols
    hb = torch.cat((h, h.new_zeros(n, pad)), 1).view(n, -1, 32)
    eb = torch.cat((he, he.new_zeros(n, pad)), 1).view(n, -1, 32)
    top = hb.abs().amax(-1, keepdim=True)
    top_err = torch.where(hb.abs() + eb >= top - eb, eb, 0.0).amax(-1, keepdim=True)
    exponent = torch.frexp(top)[1].double() - 1
    unit = torch.exp2(torch.where(top > 0, (exponent - 2).clamp(min=-127), -127.0))
    power = torch.exp2(exponent)
    other_scale = (top > 0) & ((top - top_err < power) | (top + top_err >= 2 * power))
    a = hb.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)) * unit
    near = ((a.unsqueeze(-1) - MID).abs().amin(-1) * unit <= eb)
    slack = torch.where(near, step, 0.0)
    slack = torch.where(other_scale, 4.0 * unit, slack)
    slack = slack.flatten(1)[:, :cols]
    hq = on_grid(h)
    w = values(*down, cols)
    y = hq @ w.t()
    err = slack @ w.abs().t() + (padded(cols) + 8) * EPS24 * ((hq.abs() + slack) @ w.abs().t())
    return y, err


def route(logits, top_k, score, bias=None, groups=1, top_groups=1, group_score="top2", renormalize=True, scale=1.0):
    """(index, weight, scores) in 64 bits; differentiable in logits."""
    z = logits
    if score == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-z))
    else:
        m = z.detach().amax(-1, keepdim=True)
        e = torch.exp(z - torch.where(torch.isinf(m) & (m < 0), 0.0, m))
        total = e.sum(-1, keepdim=True)
        s = e / torch.where(total == 0, 1.0, total)
    c = s.detach() if bias is None else s.detach() + bias
    c = torch.where(torch.isnan(c), float("-inf"), c)
    per = c.unflatten(-1, (groups, -1))
    n = min(2, per.size(-1)) if group_score == "top2" else 1
    v = per.sort(-1, descending=True).values[..., :n].sum(-1)
    v = torch.where(torch.isnan(v), float("-inf"), v)
    order = v.sort(dim=-1, descending=True, stable=True).indices[..., :top_groups]
    out = torch.ones_like(v, dtype=torch.bool).scatter(-1, order, False).repeat_interleave(per.size(-1), -1)
    # experts of groups left out go behind every other, a -infinity of a kept group included
    first = torch.where(out, 1, 0)
    by_choice = c.sort(dim=-1, descending=True, stable=True).indices
    by_group = torch.gather(first, -1, by_choice).sort(dim=-1, stable=True).indices
    index = torch.gather(by_choice, -1, by_group)[..., :top_k]
    picked = s.gather(-1, index)
    weight = picked / (picked.sum(-1, keepdim=True) + 1e-20) if renormalize else picked
    return index, weight * scale, s
