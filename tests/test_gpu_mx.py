"""Microscaled quantisation, product and experts against their definitions in 64 bits."""

import pytest
import torch

import quantaweave_amd as qa
from quantaweave_amd import _hip, _lib
from tests import mx_oracle as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def cuda(pair):
    return tuple(t.cuda() for t in pair)


def close(got: torch.Tensor, want: torch.Tensor, err: torch.Tensor) -> None:
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= err)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - want).abs() / err.clamp_min(1e-300)).max()}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (1, 32), (5, 33), (7, 128), (2, 129), (33, 200), (300, 1000),
                                       (64, 2048), (1, 4096)])
def test_quantise_is_exact(dtype, rows, cols):
    x = ref.rows(gen(rows * 7 + cols), rows, cols, dtype)
    codes, scales = qa.mx_quantize(x.cuda())
    code, byte = ref.quantize(x)
    assert torch.equal(scales.cpu(), byte)
    # a negative number that rounds to zero keeps its sign bit: compare values and codes
    assert torch.equal(codes.cpu(), ref.pack(code))
    back = qa.mx_dequantize(codes, scales, cols, dtype)
    assert torch.equal(back.cpu().double(), ref.values(codes, scales, cols))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantise_edges(dtype):
    """Midpoints and their neighbours, saturation, subnormals, zeros, the largest numbers, infinities, NaN."""
    info = torch.finfo(dtype)
    mids = ref.MID.repeat(5)[:31]
    base = torch.cat((mids, torch.tensor([4.0]).double()))
    out = []
    for e in (-20, -3, 0, 5, 12):
        v = (base * 2.0 ** e).to(dtype)
        out += [v, -v, torch.nextafter(v.float(), v.float() * 2).to(dtype), torch.nextafter(v.float(), v.float() * 0).to(dtype)]
    out.append(torch.linspace(4, 8, 33)[:32].to(dtype))
    out.append(torch.zeros(32, dtype=dtype))
    out.append(-torch.zeros(32, dtype=dtype))
    out.append((torch.arange(32) * float(info.tiny) / 16).to(dtype))
    out.append((torch.arange(32) * float(info.smallest_normal) * info.eps).to(dtype))
    out.append(torch.linspace(-float(info.max), float(info.max), 32).to(dtype))
    for bad in (float("inf"), -float("inf"), float("nan")):
        v = torch.linspace(-3, 3, 32).to(dtype)
        v[9] = bad
        out.append(v)
    x = torch.stack(out)
    codes, scales = qa.mx_quantize(x.cuda())
    code, byte = ref.quantize(x)
    assert torch.equal(scales.cpu(), byte)
    assert torch.equal(codes.cpu(), ref.pack(code))
    back, want = qa.mx_dequantize(codes, scales, 32).cpu().double(), ref.values(codes, scales, 32)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(back), torch.nan_to_num(want))


def test_quantise_strides_and_shapes():
    g = gen(3)
    x = torch.randn(6, 10, 96, generator=g).cuda()
    for v in (x, x[:, ::2], x[..., 8:72], x[..., 1:90], x.transpose(0, 1), x[:, :, ::3], x[2, 3], x[:0],
              x[0, :1].expand(4, 96)):
        codes, scales = qa.mx_quantize(v)
        c = v.size(-1)
        flat = v.reshape(-1, c)
        code, byte = ref.quantize(flat)
        assert torch.equal(codes.cpu().reshape(-1, codes.size(-1)), ref.pack(code))
        assert torch.equal(scales.cpu().reshape(-1, scales.size(-1)), byte)
        assert torch.equal(qa.mx_dequantize(codes, scales, c).cpu().double().reshape(-1, c), ref.on_grid(flat))


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantise_rounds_once(dtype):
    """Every code under scales from subnormal to overflowing; values past the type's range become infinite or zero."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)[:, :64].contiguous()
    scales = torch.arange(256, dtype=torch.uint8).unsqueeze(1).expand(256, 4).contiguous()
    got = qa.mx_dequantize(codes.cuda(), scales.cuda(), 128, dtype).cpu()
    want = ref.values(codes, scales, 128).float().to(dtype)  # exact in fp32 except above 2^128: infinite there too
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


SHAPES = [(1, 64, 7), (1, 2048, 7168), (3, 200, 33), (16, 1408, 64), (17, 128, 130), (40, 33, 16), (64, 512, 256),
          (65, 1000, 301), (130, 640, 96), (200, 2048, 512), (333, 384, 1000), (1, 1, 1), (700, 256, 260),
          (2, 4500, 40), (16, 9000, 33), (20, 5000, 70)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_matmul(dtype, rows, cols, n):
    g = gen(rows + 3 * cols + n)
    x, w = ref.rows(g, rows, cols, dtype), ref.stored(g, n, cols)
    want, err = ref.matmul(x, *w)
    close(qa.mx_matmul(x.cuda(), *cuda(w)), want, ref.allowed(want, err, dtype))


def test_matmul_leading_dims_strides_and_alignment():
    g = gen(11)
    w = ref.stored(g, 48, 192)
    wc = cuda(w)
    base = torch.randn(4, 9, 200, generator=g).bfloat16().cuda()
    odd = torch.empty(48 * 128 + 1, dtype=torch.uint8, device="cuda")[1:].view(48, 128).copy_(wc[0])  # off 16 bytes
    for x in (base[..., :192], base[..., 3:195], base[:, ::2, 8:], base.transpose(0, 1)[..., :192], base[1, 2, :192],
              base[:0, :, :192], base[0, :1, :192].expand(5, 192)):
        want, err = ref.matmul(x.reshape(-1, 192), *w)
        for codes in (wc[0], odd):
            got = qa.mx_matmul(x, codes, wc[1])
            assert got.shape == (*x.shape[:-1], 48)
            close(got.reshape(-1, 48), want, ref.allowed(want, err, torch.bfloat16))


@pytest.mark.parametrize("rows", [3, 17])  # both kernels
def test_matmul_of_a_matrix_past_32_bit_offsets(rows):
    n, k = (1 << 20) + 300, 8192  # 4.3 GB of codes
    x = ref.rows(gen(17), rows, k, torch.bfloat16)
    on_gpu = torch.Generator("cuda").manual_seed(17)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=on_gpu)
    scales = torch.randint(120, 132, (n, k // 32), dtype=torch.uint8, device="cuda", generator=on_gpu)
    got = qa.mx_matmul(x.cuda(), codes, scales)
    for at in (0, 256, n // 2 + 5, (1 << 20) - 30, n - 60):
        part = slice(at, at + 60)
        want, err = ref.matmul(x, codes[part].cpu(), scales[part].cpu())
        close(got[:, part], want, ref.allowed(want, err, torch.bfloat16))


def test_a_second_derivative_is_refused():
    g = gen(19)
    x, w = torch.randn(4, 96, generator=g).cuda().requires_grad_(True), cuda(ref.stored(g, 8, 96))
    z = torch.randn(4, 16, generator=g).cuda().requires_grad_(True)
    for y, leaf in ((qa.mx_matmul(x, *w), x), (qa.route_experts(z, 2)[1], z)):
        (first,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()


def test_matmul_nan_and_infinite_rows_stay_in_their_rows():
    g = gen(5)
    for rows in (5, 80):
        x, w = ref.rows(g, rows, 300, torch.float32), ref.stored(g, 64, 300)
        x[1, 7], x[3, 299] = float("nan"), float("inf")
        got = qa.mx_matmul(x.cuda(), *cuda(w)).cpu()
        assert torch.isnan(got[1]).all() and torch.isnan(got[3]).all()
        keep = [i for i in range(rows) if i not in (1, 3)]
        want, err = ref.matmul(x[keep], *w)
        close(got[keep], want, ref.allowed(want, err, torch.float32))


def test_rows_do_not_depend_on_their_neighbours():
    """A row alone and the same row among others: the same bits, where the same kernel takes both."""
    g = gen(6)
    x, w = ref.rows(g, 12, 1024, torch.float32).cuda(), cuda(ref.stored(g, 96, 1024))
    many = qa.mx_matmul(x, *w)
    assert torch.equal(many[4:5], qa.mx_matmul(x[4:5], *w))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,n", [(1, 64, 7), (5, 200, 33), (130, 256, 128), (257, 1000, 192), (300, 512, 320)])
def test_matmul_gradient(dtype, rows, cols, n):
    g = gen(rows * cols + n)
    x, w = ref.rows(g, rows, cols, dtype), ref.stored(g, n, cols)
    dy = torch.randn(rows, n, generator=g).to(dtype)
    xc = x.cuda().requires_grad_(True)
    y = qa.mx_matmul(xc, *cuda(w))
    (gx,) = torch.autograd.grad(y, xc, dy.cuda())
    wv = ref.values(*w, cols)  # exact in every type: scales near 1
    want = dy.double() @ wv
    err = (n + 8) * ref.EPS24 * (dy.double().abs() @ wv.abs())  # products of two 16-bit numbers are exact in fp32
    if dtype == torch.float32:
        err = err + ref.EPS24 * (dy.double().abs() @ wv.abs())
    close(gx, want, ref.allowed(want, err, dtype))
    # quantised rows are the result's rows: the result is the same with and without a gradient
    assert torch.equal(y.detach(), qa.mx_matmul(x.cuda(), *cuda(w)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,n", [(64, 1000, 3001), (1, 1000, 301), (700, 1000, 97), (2000, 333, 65),
                                         (130, 12, 100), (33, 4, 7), (257, 1001, 192), (300, 6, 64), (40, 1, 1),
                                         (5, 100, 128), (1200, 2052, 130)])
def test_matmul_gradient_of_any_width(dtype, rows, cols, n):
    """Widths that are no whole slices or loads of the matrix cores; a grad_out off 16 bytes; through the C entry
    point a grad_out and a grad_x off 16 bytes, rows behind grad_x left as they were."""
    g = gen(rows + cols * n)
    w = ref.stored(g, n, cols)
    dy = torch.randn(rows, n, generator=g).to(dtype)
    wv = ref.values(*w, cols)
    want = dy.double() @ wv
    # fp32 sums of n exact products, of 2 n with fp16's two parts; fp32's own products are rounded
    terms = {torch.float32: 2 * n + 8, torch.bfloat16: n + 8, torch.float16: (2 * n + 8) * (1 + 2.0 ** -7)}[dtype]
    err = ref.allowed(want, terms * ref.EPS24 * (dy.double().abs() @ wv.abs()), dtype)
    x = ref.rows(g, rows, cols, dtype).cuda().requires_grad_(True)
    y = qa.mx_matmul(x, *cuda(w))
    off = torch.empty(rows * n + 1, dtype=dtype, device="cuda")[1:].view(rows, n).copy_(dy)
    for grad in (dy.cuda(), off):
        close(torch.autograd.grad(y, x, grad, retain_graph=True)[0], want, err)
    act, (codes, scales), lib = _hip.act_code(dy, "test"), cuda(w), _lib.load()
    nbytes = lib.qw_mx_matmul_backward_workspace_bytes(rows, n, cols, act)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    for grad, start in ((dy.cuda(), 1), (off, 0)):
        out = torch.full((start + rows * cols + 64,), 3.0, dtype=dtype, device="cuda")
        _lib.call("qw_mx_matmul_backward", _hip.ptr(grad), act, rows, _hip.ptr(codes), _hip.ptr(scales), n, cols,
                  _hip.ptr(out[start:]), _hip.ptr(ws), nbytes, _hip.stream(out.device))
        close(out[start:start + rows * cols].view(rows, cols), want, err)
        assert (out[:start] == 3.0).all() and (out[start + rows * cols:] == 3.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,n", [(65535 * 64 + 70, 32, 4), (70, 16, (1 << 22) + 72)])
def test_matmul_gradient_of_what_the_product_takes(dtype, rows, cols, n):
    """More rows, and more outputs, than one grid or one tile's 32-bit offsets hold."""
    g = torch.Generator("cuda").manual_seed(rows % 1000)
    codes = torch.randint(0, 256, (n, 64), dtype=torch.uint8, device="cuda", generator=g)
    codes[:, cols // 2:] = 0
    scales = torch.randint(118, 122, (n, 4), dtype=torch.uint8, device="cuda", generator=g)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype).requires_grad_(True)
    y = qa.mx_matmul(x, codes, scales)
    dy = torch.randn(rows, n, device="cuda", generator=g).to(dtype)
    (gx,) = torch.autograd.grad(y, x, dy)
    act, lib = _hip.act_code(dy, "test"), _lib.load()
    nbytes = lib.qw_mx_matmul_backward_workspace_bytes(rows, n, cols, act)
    ws, out = torch.empty(nbytes, dtype=torch.uint8, device="cuda"), torch.empty_like(gx)
    off = torch.empty(rows * n + 1, dtype=dtype, device="cuda")[1:].view(rows, n).copy_(dy)  # off 16 bytes
    _lib.call("qw_mx_matmul_backward", _hip.ptr(off), act, rows, _hip.ptr(codes), _hip.ptr(scales), n, cols,
              _hip.ptr(out), _hip.ptr(ws), nbytes, _hip.stream(out.device))
    for r in sorted({0, max(rows - 500, 0)}):  # the first rows and the last
        d = dy[r:r + 500]
        want = torch.zeros(d.size(0), cols, dtype=torch.float64, device="cuda")
        total = torch.zeros_like(want)
        for at in range(0, n, 1 << 18):
            wv = qa.mx_dequantize(codes[at:at + (1 << 18)], scales[at:at + (1 << 18)], cols).double()
            part = d[:, at:at + (1 << 18)].double()
            want += part @ wv
            total += part.abs() @ wv.abs()
        # n terms (2 n of fp16's parts, n products rounded of fp32), each addition off by 2^-24 of the sum's magnitudes
        err = (2 * n + 8) * (1 + 2.0 ** -7) * ref.EPS24 * total
        # where n is past 2^20 that is no bound; the additions' errors are as good as independent: sixteen deviations
        err = torch.minimum(err, 16 * (2 * n) ** 0.5 * ref.EPS24 * total)
        for got in (gx, out):
            close(got[r:r + 500], want.cpu(), ref.allowed(want, err, dtype).cpu())


@pytest.mark.parametrize("rows,cols,n", [(1, 33, 7), (5, 96, 64), (70, 264, 130), (300, 512, 200)])
@pytest.mark.parametrize("low,high", [(87, 158), (90, 91), (100, 101), (141, 142), (150, 151), (60, 230)])
def test_fp16_gradient_over_the_range_of_the_scales(rows, cols, n, low, high):
    """Stored weights past fp16 at either end: what fp16 can hold of the result is right, the rest is infinite or 0."""
    g = gen(rows + cols + low)
    w = ref.stored(g, n, cols, low=low, high=high)
    # a block of columns has the scales of its first row give or take two, so that the results have every size
    w = (w[0], (w[1][:1].int() + torch.randint(-2, 3, w[1].shape, generator=g)).clamp(0, 254).to(torch.uint8))
    dy = torch.randn(rows, n, generator=g) * torch.exp2(torch.randint(-14, 8, (rows, 1), generator=g))
    dy[torch.rand(rows, n, generator=g) < 0.3] = 0.0
    dy[0] = 0.0
    dy = dy.half()
    x = ref.rows(g, rows, cols, torch.float16).cuda().requires_grad_(True)
    (gx,) = torch.autograd.grad(qa.mx_matmul(x, *cuda(w)), x, dy.cuda())
    gx = gx.cpu().double()
    assert not gx[0].any() and not torch.isnan(gx).any()
    wv = ref.values(*w, cols)
    want = dy.double() @ wv
    # dy as two numbers whose magnitudes add up to at most 1 + 2^-7 of it: 2 n products, each exact, and their sums
    err = (2 * n + 8) * ref.EPS24 * (1 + 2.0 ** -7) * (dy.double().abs() @ wv.abs())
    beyond = want.abs() + err >= 65520.0  # rounds to an infinity, or may
    assert torch.isinf(gx[want.abs() - err >= 65520.0]).all()
    bad = ~beyond & ~((gx - want).abs() <= ref.allowed(want, err, torch.float16))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}"


def test_matmul_gradient_is_a_difference_of_the_product_on_the_grid():
    """Where x moves from grid value to grid value the product's difference is the gradient times it."""
    g = gen(21)
    w = ref.stored(g, 40, 64)
    x = torch.full((1, 64), 4.0)
    x[0, 5] = 2.0
    moved = x.clone()
    moved[0, 5] = 3.0
    xc = x.cuda().requires_grad_(True)
    y = qa.mx_matmul(xc, *cuda(w))
    dy = torch.randn(1, 40, generator=g)
    (gx,) = torch.autograd.grad(y, xc, dy.cuda())
    diff = ((qa.mx_matmul(moved.cuda(), *cuda(w)) - y.detach()).cpu().double() * dy.double()).sum()
    # both results carry 72 fp32 additions of terms up to 4 * 6 * 2^-6
    bound = 2 * 72 * ref.EPS24 * float((ref.values(*w, 64).abs().sum(1) * 4 * dy.double().abs().squeeze(0)).sum())
    assert abs(float(diff) - float(gx[0, 5])) <= bound


def grouped(g, counts, d, f, dtype, tail=0):
    e = len(counts)
    x = ref.rows(g, sum(counts) + tail, d, dtype)
    gate, up, down = ref.stored(g, e, f, d), ref.stored(g, e, f, d), ref.stored(g, e, d, f)
    offsets = torch.tensor([0] + list(counts)).cumsum(0).int()
    y = torch.zeros(x.size(0), d, dtype=torch.float64)
    err = torch.zeros_like(y)
    for i in range(e):
        a, b = int(offsets[i]), int(offsets[i + 1])
        if b > a:
            y[a:b], err[a:b] = ref.swiglu(x[a:b], *(tuple(t[i] for t in m) for m in (gate, up, down)))
    return x, gate, up, down, offsets, y, err


GROUPS = [([1], 64, 128), ([0, 5, 37, 1, 0, 64, 33, 2], 128, 96), ([3, 0, 17], 200, 264), ([16, 15, 1], 256, 33),
          ([0, 0, 0], 64, 64), ([90, 300, 0, 21], 384, 320), ([2] * 40, 512, 128), ([129, 1], 1000, 200),
          ([0, 70, 0, 1, 0, 0, 3], 256, 128), ([3, 1], 2300, 160), ([2, 5], 264, 2400)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,d,f", GROUPS)
@pytest.mark.parametrize("bound", [None, "max"])
def test_grouped_swiglu(dtype, counts, d, f, bound):
    x, gate, up, down, offsets, want, err = grouped(gen(sum(counts) + d + f), counts, d, f, dtype)
    got = qa.mx_grouped_swiglu(x.cuda(), cuda(gate), cuda(up), cuda(down), offsets.cuda(),
                               max_rows=max(counts) if bound else None)
    close(got, want, ref.allowed(want, err, dtype))


def test_grouped_swiglu_rows_past_the_last_group_are_zero():
    x, gate, up, down, offsets, want, err = grouped(gen(9), [5, 0, 70, 2], 256, 128, torch.bfloat16, tail=37)
    got = qa.mx_grouped_swiglu(x.cuda(), cuda(gate), cuda(up), cuda(down), offsets.cuda())
    close(got, want, ref.allowed(want, err, torch.bfloat16))
    assert not got[77:].any()


@pytest.mark.parametrize("tail", [12, 200])  # few rows per expert, and the tiles
@pytest.mark.parametrize("zero", [0, 1])
def test_experts_entry_point_leaves_or_clears_the_rows_behind_the_last_group(tail, zero):
    x, gate, up, down, offsets, want, err = grouped(gen(9), [5, 0, 30, 2], 256, 128, torch.bfloat16, tail=tail)
    rows, x = x.size(0), x.cuda()
    y = torch.full((rows, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    m = [t for pair in (gate, up, down) for t in cuda(pair)]
    offsets = offsets.cuda()
    nbytes = _lib.load().qw_mx_experts_workspace_bytes(rows, 4, 256, 128)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    _lib.call("qw_mx_experts", _hip.ptr(x), _lib.QW_BF16, 256, _hip.ptr(offsets), 4, 256, 128, rows, 30,
              *(_hip.ptr(t) for t in m), zero, _hip.ptr(y), _hip.ptr(ws), nbytes, _hip.stream(x.device))
    close(y[:37], want[:37], ref.allowed(want[:37], err[:37], torch.bfloat16))
    assert (y[37:] == (0.0 if zero else 7.0)).all()


def test_grouped_swiglu_without_rows():
    _, gate, up, down, offsets, _, _ = grouped(gen(9), [0, 0], 64, 64, torch.bfloat16)
    got = qa.mx_grouped_swiglu(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), cuda(gate), cuda(up),
                               cuda(down), offsets.cuda())
    assert got.shape == (0, 64)


def test_route_then_experts_together():
    """Tokens routed by scores, sorted by expert and taken through microscaled experts, as a layer does."""
    g = gen(31)
    tokens, e, k, d, f = 70, 16, 4, 256, 128
    x = ref.rows(g, tokens, d, torch.bfloat16)
    logits, bias = torch.randn(tokens, e, generator=g), 0.1 * torch.randn(e, generator=g)
    index, weight, _ = qa.route_experts(logits.cuda(), k, score="sigmoid", bias=bias.cuda(), groups=4, top_groups=2)
    want_index, want_weight, _ = ref.route(logits.double(), k, "sigmoid", bias.double(), 4, 2)
    assert torch.equal(index.cpu().long(), want_index)
    flat = index.flatten().long()
    order = flat.argsort(stable=True)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.bincount(flat, minlength=e).cumsum(0)
    gate, up, down = ref.stored(g, e, f, d), ref.stored(g, e, f, d), ref.stored(g, e, d, f)
    y = qa.mx_grouped_swiglu(x.cuda()[order // k], cuda(gate), cuda(up), cuda(down), offsets)
    out = torch.zeros(tokens, d, device="cuda").index_add_(0, order // k, y.float() * weight.flatten()[order, None])
    want, err = torch.zeros(tokens, d, dtype=torch.float64), torch.zeros(tokens, d, dtype=torch.float64)
    for t in range(tokens):
        for j in range(k):
            m = [tuple(s[int(want_index[t, j])] for s in w) for w in (gate, up, down)]
            yy, ee = ref.swiglu(x[t:t + 1], *m)
            w = float(want_weight[t, j])
            want[t] += w * yy[0]
            # y's rounding, the weight's and the product's and the k additions' in fp32
            err[t] += w * (ref.allowed(yy, ee, torch.bfloat16)[0] + (k + 16) * ref.EPS24 * (yy[0].abs() + ee[0]))
    close(out, want, err + (k + 1) * ref.EPS24 * want.abs())


def test_graph_replays_and_streams():
    g = gen(41)
    w, x = cuda(ref.stored(g, 96, 320)), ref.rows(g, 50, 320, torch.bfloat16).cuda()
    xs, gate, up, down, offsets, _, _ = grouped(g, [9, 0, 40, 3], 128, 64, torch.bfloat16)
    xs, gate, up, down, offsets = xs.cuda(), cuda(gate), cuda(up), cuda(down), offsets.cuda()
    logits = torch.randn(33, 64, generator=g).cuda()

    def step():
        return (qa.mx_matmul(x, *w), qa.mx_grouped_swiglu(xs, gate, up, down, offsets), *qa.mx_quantize(x),
                *qa.route_experts(logits, 4, score="sigmoid", groups=8, top_groups=4))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):  # a second graph beside the first, its workspaces its own
        out2 = step()
    for seed in range(3):
        gg = gen(100 + seed)
        x.copy_(ref.rows(gg, 50, 320, torch.bfloat16))
        xs.copy_(ref.rows(gg, xs.size(0), 128, torch.bfloat16))
        logits.copy_(torch.randn(33, 64, generator=gg))
        eager = [t.clone() for t in step()]
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(eager, out, out2):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_backward_captured_and_replayed():
    g = gen(43)
    w, x = cuda(ref.stored(g, 128, 256)), ref.rows(g, 64, 256, torch.bfloat16).cuda().requires_grad_(True)
    z = torch.randn(40, 64, generator=g).cuda().requires_grad_(True)
    dy, dw = torch.randn(64, 128, generator=g).bfloat16().cuda(), torch.randn(40, 4, generator=g).cuda()

    def step():
        y, (_, weight, _) = qa.mx_matmul(x, *w), qa.route_experts(z, 4, score="sigmoid", groups=8, top_groups=4)
        return torch.autograd.grad((y, weight), (x, z), (dy, dw))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(ref.rows(gen(200 + seed), 64, 256, torch.bfloat16))
            z.copy_(torch.randn(40, 64, generator=gen(300 + seed)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_backward_captured_beside_an_eager_graph_of_its_leaf_is_refused():
    """And a forward pass captured beside it is not; without the eager graph both are captured."""
    g = gen(47)
    w, x = cuda(ref.stored(g, 64, 128)), ref.rows(g, 24, 128, torch.bfloat16).cuda().requires_grad_(True)
    z = torch.randn(24, 32, generator=g).cuda().requires_grad_(True)
    for op, leaf in ((lambda: qa.mx_matmul(x, *w), x), (lambda: qa.route_experts(z, 4)[1], z)):
        kept = op()
        dy = torch.ones_like(kept)
        (eager,) = torch.autograd.grad(kept, leaf, dy, retain_graph=True)
        forward, refused, both = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(forward):
            alone = op()
        for _ in range(2):
            forward.replay()
            torch.cuda.synchronize()
            assert torch.equal(alone, kept)
        del alone
        with pytest.raises(RuntimeError, match="another stream"):
            with torch.cuda.graph(refused):
                torch.autograd.grad(op(), leaf, dy)
        del kept
        with torch.cuda.graph(both):
            (captured,) = torch.autograd.grad(op(), leaf, dy)
        for _ in range(2):
            both.replay()
            torch.cuda.synchronize()
            assert torch.equal(captured, eager)


def test_refusals():
    g = gen(1)
    x = torch.randn(4, 96, generator=g).cuda()
    codes, scales = cuda(ref.stored(g, 8, 96))
    for bad, match in (((codes.int(), scales), "uint8"), ((codes[:, :40], scales), "bytes a row"),
                       ((codes, scales[:, :2]), "scales have shape"), ((codes[0], scales[0]), "dimensions"),
                       ((codes.cpu(), scales), "must be on")):
        with pytest.raises(ValueError, match=match):
            qa.mx_matmul(x, *bad)
    with pytest.raises(ValueError, match="dtype"):
        qa.mx_matmul(x.double(), codes, scales)
    with pytest.raises(ValueError, match="dtype"):
        qa.mx_quantize(x.int())
    with pytest.raises(ValueError, match="one column"):
        qa.mx_quantize(torch.empty(3, 0, device="cuda"))
    with pytest.raises(ValueError, match="dtype"):
        qa.mx_dequantize(codes, scales, 96, torch.float64)
    with pytest.raises(ValueError, match="cols"):
        qa.mx_dequantize(codes, scales, 0)
    gate, up, down = (cuda(ref.stored(g, 2, *s)) for s in ((64, 96), (64, 96), (96, 64)))
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="offsets"):
        qa.mx_grouped_swiglu(x, gate, up, down, off.long())
    with pytest.raises(ValueError, match="offsets"):
        qa.mx_grouped_swiglu(x, gate, up, down, off[:2])
    with pytest.raises(ValueError, match="down"):
        qa.mx_grouped_swiglu(x, gate, up, gate, off)
    with pytest.raises(ValueError, match="one shape"):
        qa.mx_grouped_swiglu(x, gate, tuple(t[:, :32].contiguous() for t in up), down, off)
    with pytest.raises(NotImplementedError, match="quantised experts"):
        qa.mx_grouped_swiglu(x.clone().requires_grad_(True), gate, up, down, off)
