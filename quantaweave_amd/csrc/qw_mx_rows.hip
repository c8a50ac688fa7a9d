// Microscaled products of few rows (decoding): each weight is read once per
// sixteen rows of its group, straight from memory into the matrix instruction.
//
// One workgroup of eight waves owns sixteen rows of a group and 32 columns of
// the result (two matrices: 32 gate and the matching 32 up columns, one block of
// the hidden row).  A wave takes every eighth step of 128 columns: its lanes hold
// 16 weight rows by four blocks, one 16-byte load and one scale byte per lane and
// 16 columns of the result; rows given as numbers become codes in the registers
// of the lane that multiplies them, whose 32 numbers are one block.  The eight
// partial sums meet in LDS and are added in wave order (the same sum whatever
// the rows beside it).  Bound by HBM where all experts are touched, by latency
// for a single matrix.
#include "qw_mx_product.h"

namespace qw {

namespace {

constexpr int kRowsWaves = 8, kRowsThreads = kRowsWaves * kWave;
constexpr int kRowsM = 16, kRowsN = 32;
constexpr int kStored = -1;  // XDT of rows that are stored microscaled

// The workgroups past the groups' last tile: zeros in the rows behind the last
// group, sixteen rows by 32 columns each.
__device__ void zero_rows(const int32_t* __restrict__ offsets, int groups, int rows, int chunk, int ct, int n,
                          void* __restrict__ out, int out_dtype) {
  const int lane = threadIdx.x % kWave;
  int tiles = 0;
  for (int e0 = 0; e0 < groups; e0 += kWave) {
    int c = 0;
    if (e0 + lane < groups) {
      const int lo = min(max(offsets[e0 + lane], 0), rows), hi = min(offsets[e0 + lane + 1], rows);
      c = hi > lo ? (hi - lo + kRowsM - 1) / kRowsM : 0;
    }
    tiles += wave_sum_i(c);
  }
  const int64_t row = static_cast<int64_t>(max(offsets[groups], 0)) + static_cast<int64_t>(chunk - tiles) * kRowsM +
                      threadIdx.x / kRowsN;
  const int col = ct * kRowsN + threadIdx.x % kRowsN;
  if (row >= rows || col >= n) return;
  if (out_dtype == QW_F32) static_cast<float*>(out)[row * n + col] = 0.0f;
  else static_cast<uint16_t*>(out)[row * n + col] = 0;
}

template <int XDT, bool GATEUP>
__global__ __launch_bounds__(kRowsThreads) void mx_rows_kernel(
    const void* __restrict__ x, int64_t x_stride, bool x_aligned, const uint8_t* __restrict__ x_scales,
    const int32_t* __restrict__ row_index, const int32_t* __restrict__ offsets, int groups, int rows, MxMatrix wa,
    MxMatrix wb, int n, int k, int col_tiles, void* __restrict__ out, int out_dtype, bool zero_rest, uint8_t* __restrict__ h_codes,
    uint8_t* __restrict__ h_scales) {
  constexpr int TILES = GATEUP ? 4 : 2;  // 16 weight rows each: two of gate, two of up
  __shared__ f32x4 part[kRowsWaves][TILES][kWave];
  const int ct = blockIdx.x % col_tiles, chunk = blockIdx.x / col_tiles;
  int e = 0, local = chunk;
  int r0 = chunk * kRowsM, end = rows;
  if (offsets) {
    e = find_tile(offsets, groups, rows, kRowsM, chunk, &local);
    if (e < 0) {
      if (!GATEUP && zero_rest) zero_rows(offsets, groups, rows, chunk, ct, n, out, out_dtype);
      return;
    }
    r0 = max(offsets[e], 0) + local * kRowsM;
    end = min(offsets[e + 1], rows);
  }
  const int count = min(end - r0, kRowsM);
  if (count <= 0) return;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int l16 = lane % 16, lq = lane / 16;
  const int n0 = ct * kRowsN;
  const int64_t pitch = (k + kMxStep - 1) / kMxStep * static_cast<int64_t>(kMxStep);
  const int64_t cb = pitch / 2, sb = pitch / kMxBlock;
  const int steps = static_cast<int>(pitch / kMxStep);

  // rows past the count repeat the last one; their results are not stored
  const int rr = r0 + min(l16, count - 1);
  const int64_t row = row_index ? row_index[rr] : rr;
  const uint8_t* w_codes[TILES];
  const uint8_t* w_scales[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const MxMatrix& m = t < 2 ? wa : wb;
    const int64_t wr = static_cast<int64_t>(e) * n + min(n0 + (t % 2) * 16 + l16, n - 1);
    w_codes[t] = m.codes + wr * cb + lq * 16;
    w_scales[t] = m.scales + wr * sb + lq;
  }
  f32x4 acc[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = wave; s < steps; s += kRowsWaves) {
    u32x4 w[TILES];
    uint32_t ws[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      w[t] = *reinterpret_cast<const u32x4*>(w_codes[t] + static_cast<int64_t>(s) * 64);
      ws[t] = w_scales[t][s * 4];
    }
    u32x4 xc;
    uint32_t xs;
    if constexpr (XDT == kStored) {
      xc = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(x) + row * cb + s * 64 + lq * 16);
      xs = x_scales[row * sb + s * 4 + lq];
    } else {
      const int col = s * kMxStep + lq * kMxBlock;
      MxPiece<XDT> v[4];
      uint32_t top = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        v[q] = mx_load_piece<XDT>(x, row * x_stride + col + 8 * q, k - col - 8 * q, x_aligned);
#pragma unroll
      for (int q = 0; q < 4; ++q) top = mx_top_max<XDT>(top, mx_piece_top<XDT>(v[q]));
      xs = mx_scale_of(mx_top_bits<XDT>(top));
#pragma unroll
      for (int q = 0; q < 4; ++q) xc[q] = mx_piece_codes<XDT>(v[q], xs);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[t] = mx_mfma(w[t], xc, acc[t], ws[t], xs);
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // thread -> (row m, column c): a lane's four sums are columns 4 lq .. 4 lq + 3 of row l16
  const int m = tid / kRowsN, c = tid % kRowsN;
  auto total = [&](int t) {
    const int at = m + 16 * (c % 16 / 4);
    float v = part[0][t][at][c % 4];
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) v += part[w][t][at][c % 4];
    return v;
  };
  const int64_t orow = r0 + m;
  if constexpr (!GATEUP) {
    const float v = total(c / 16);
    if (m < count && n0 + c < n) {
      if (out_dtype == QW_F32) store_act<QW_F32>(out, orow * n + n0 + c, v);
      else if (out_dtype == QW_F16) store_act<QW_F16>(out, orow * n + n0 + c, v);
      else store_act<QW_BF16>(out, orow * n + n0 + c, v);
    }
  } else {
    const bool live = n0 + c < n;  // padding columns of the hidden row are zero codes
    const float h = live ? mx_swiglu(total(c / 16), total(2 + c / 16)) : 0.0f;
    uint32_t top = __float_as_uint(h) & 0x7fffffffu;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, kWave)));
    const uint32_t s = mx_scale_of(top);
    const float other = __shfl_xor(h, 1, kWave);
    const uint32_t code = s == kMxNan ? 0u : mx_pack_f32<0>(0u, h, other, mx_divisor(s));
    const int64_t np = (n + kMxStep - 1) / kMxStep * static_cast<int64_t>(kMxStep);
    if (m < count) {
      if (c % 2 == 0) h_codes[orow * (np / 2) + (n0 + c) / 2] = static_cast<uint8_t>(code);
      if (c == 0) h_scales[orow * (np / kMxBlock) + n0 / kMxBlock] = static_cast<uint8_t>(s);
    }
  }
}

template <int XDT>
int launch_t(const MxProduct& p, hipStream_t stream) {
  const bool gateup = p.h_codes != nullptr;
  // hidden rows are written to their padded width
  const int64_t col_tiles = ceil_div(gateup ? mx_padded(p.n) : p.n, kRowsN);
  const int64_t chunks = p.offsets ? ceil_div(p.rows, kRowsM) + p.groups + (p.zero_rest ? 1 : 0) : ceil_div(p.rows, kRowsM);
  const int64_t grid = col_tiles * chunks;
  if (grid > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows and columns for one microscaled product");
  const int size = XDT == QW_F32 ? 4 : 2;
  const bool aligned = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.x_stride * size % 16 == 0;
  const void* x = XDT == kStored ? p.x_codes : p.x;
  auto go = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(grid), kRowsThreads, 0, stream>>>(
        x, p.x_stride, aligned, p.x_scales, p.row_index, p.offsets, static_cast<int>(p.groups),
        static_cast<int>(p.rows), p.a, p.b, static_cast<int>(p.n), static_cast<int>(p.k), static_cast<int>(col_tiles),
        p.out, p.out_dtype, p.zero_rest, p.h_codes, p.h_scales);
  };
  if (gateup) go(mx_rows_kernel<XDT, true>);
  else go(mx_rows_kernel<XDT, false>);
  QW_LAUNCH_CHECK("mx_rows_kernel");
  return QW_OK;
}

}  // namespace

int launch_mx_rows(const MxProduct& p, hipStream_t stream) {
  if (p.x_codes) return launch_t<kStored>(p, stream);
  if (p.x_dtype == QW_F32) return launch_t<QW_F32>(p, stream);
  if (p.x_dtype == QW_F16) return launch_t<QW_F16>(p, stream);
  return launch_t<QW_BF16>(p, stream);
}

}  // namespace qw
