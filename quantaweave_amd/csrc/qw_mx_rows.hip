// Microscaled products of few rows (decoding): each weight is read once per
// sixteen rows of its group, straight from memory into the matrix instruction.  (A
// group of many rows beside empty ones is so many passes over its weights: 1024 rows
// of 64 experts, d 2048, f 1024, evenly 118 us for the experts' products, all rows in
// one 347 us.)
//
// One workgroup owns sixteen rows of a group and 32 columns of the result (two
// matrices: 32 gate and the matching 32 up columns, one block of the hidden row).
// The K axis is split over its waves in turns of one or two steps of 128 columns:
// its lanes hold 16 weight rows by four blocks, one 16-byte load per lane, step and
// 16 columns of the result, and all loads of a turn go out before the first is
// waited for.  Rows given as numbers become codes in the registers of the lane that
// multiplies them, whose 32 numbers are one block.  The partial sums meet in LDS and
// are added in wave order (the same sum whatever the rows beside it).
//
// Bound by the weight stream where many experts are touched: 128 rows of 64 experts,
// d 2048, f 1024, gate and up 43 us (2.9 TB/s), down 20.6 us (3.0 TB/s).  Bound by
// latency for a single matrix (1 row, 2048 x 7168: 5.6 us, 1.4 TB/s).
#include "qw_mx_product.h"

namespace qw {

namespace {

constexpr int kRowsM = 16, kRowsN = 32;
constexpr int kStored = -1;  // XDT of rows that are stored microscaled
// Steps of 128 columns that a wave takes together.  Two make its two loads of a
// weight row one 128-byte line (the down product above, in an earlier form, with one
// 24.5 us and with two 19.2); two matrices and the numbers of a row leave the registers
// of two workgroups per unit only one (gate and up above with two, and the next two
// requested ahead, spilled eighteen registers: 58 us).
template <int XDT, bool GATEUP>
constexpr int kRowsSteps = GATEUP && XDT != kStored ? 1 : 2;
// Workgroups that share a group's row chunks: the grid is fixed before the groups'
// sizes are known, and a group has sixteen rows at most on average.
constexpr int kRowsLayers = 2;

// Eight numbers from a place on 16 bytes, or zeros.
template <int DT>
__device__ __forceinline__ MxPiece<DT> whole_piece(const char* __restrict__ p, bool there) {
  MxPiece<DT> r;
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (there) {
    const uint4* const at = reinterpret_cast<const uint4*>(p);
    a = at[0];
    if constexpr (DT == QW_F32) b = at[1];
  }
  r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  if constexpr (DT == QW_F32) r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  return r;
}

template <int XDT, bool GATEUP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave, 4) void mx_rows_kernel(
    const void* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ x_scales,
    const int32_t* __restrict__ offsets, int groups, int rows, MxMatrix wa, MxMatrix wb, int n, int k, int col_tiles, int layers, void* __restrict__ out, int out_dtype, bool zero_rest,
    uint8_t* __restrict__ h_codes, uint8_t* __restrict__ h_scales) {
  constexpr int TILES = GATEUP ? 4 : 2;  // 16 weight rows each: two of gate, two of up
  constexpr int THREADS = WAVES * kWave, STEPS = kRowsSteps<XDT, GATEUP>;
  __shared__ f32x4 part[WAVES][TILES][kWave];
  const int ct = blockIdx.x % col_tiles, place = blockIdx.x / col_tiles;
  const int e = offsets ? place % groups : 0, layer = offsets ? place / groups : place;
  int lo = 0, end = rows;
  if (offsets) {
    lo = max(offsets[e], 0);
    end = min(offsets[e + 1], rows);
  }
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int l16 = lane % 16, lq = lane / 16;
  const int n0 = ct * kRowsN;
  const int64_t pitch = (k + kMxStep - 1) / kMxStep * static_cast<int64_t>(kMxStep);
  const int64_t cb = pitch / 2, sb = pitch / kMxBlock;
  const int steps = static_cast<int>(pitch / kMxStep), turns = (steps + STEPS - 1) / STEPS;

  if (!GATEUP && zero_rest && offsets) {  // the rows behind the last group, shared by all workgroups
    for (int64_t r0 = static_cast<int64_t>(max(offsets[groups], 0)) + place * kRowsM; r0 < rows;
         r0 += static_cast<int64_t>(groups) * layers * kRowsM)
      for (int i = tid; i < kRowsM * kRowsN; i += THREADS) {
        const int64_t row = r0 + i / kRowsN;
        const int col = n0 + i % kRowsN;
        if (row >= rows || col >= n) continue;
        if (out_dtype == QW_F32) static_cast<float*>(out)[row * n + col] = 0.0f;
        else static_cast<uint16_t*>(out)[row * n + col] = 0;
      }
  }
  // a matrix's rows of this workgroup: uniform bases, a lane's two row offsets.  Rows
  // past the matrix repeat its last one; a tile of padding columns alone (hidden rows
  // are written to their padded width) lies on it wholly.  Their results are not used.
  const int first_row = min(n0, n - 1);
  const int64_t w0 = static_cast<int64_t>(e) * n + first_row;
  const uint8_t* const codes[2] = {wa.codes + w0 * cb, GATEUP ? wb.codes + w0 * cb : nullptr};
  const uint8_t* const scales[2] = {wa.scales + w0 * sb, GATEUP ? wb.scales + w0 * sb : nullptr};
  uint32_t w_off[2], s_off[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint32_t r = min(t * 16 + l16, n - 1 - first_row);
    w_off[t] = r * static_cast<uint32_t>(cb) + lq * 16;
    s_off[t] = r * static_cast<uint32_t>(sb);
  }
  for (int64_t r0 = lo + static_cast<int64_t>(layer) * kRowsM; r0 < end; r0 += static_cast<int64_t>(layers) * kRowsM) {
    const int count = min(static_cast<int>(end - r0), kRowsM);
    f32x4 acc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // rows past the count repeat the last one; their results are not stored
    const int64_t row = r0 + min(l16, count - 1);
    constexpr int kSize = XDT == QW_F32 ? 4 : 2;
    const char* const x_row = static_cast<const char*>(x) + (row * x_stride + lq * kMxBlock) * kSize;
#pragma unroll 1
    for (int p = wave; p < turns; p += WAVES) {
      u32x4 w[TILES][STEPS], xc[STEPS];
      uint32_t ws[TILES][STEPS], xs[STEPS];
      // all loads of a turn go out together; where the last turn of two holds one step,
      // the second rereads it and is not multiplied
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const int64_t s = min(STEPS * p + j, steps - 1);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          w[t][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(codes[t / 2] + s * 64 + w_off[t % 2]));
          ws[t][j] = *reinterpret_cast<const uint32_t*>(scales[t / 2] + s * 4 + s_off[t % 2]);
        }
      }
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const int s = min(STEPS * p + j, steps - 1);
        if constexpr (XDT == kStored) {
          xc[j] = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(x) + row * cb + s * 64 + lq * 16);
          xs[j] = x_scales[row * sb + s * 4 + lq];
        } else {  // a block of this row; its pieces exist whole or not at all
          const int col = s * kMxStep + lq * kMxBlock;
          MxPiece<XDT> v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            v[q] = whole_piece<XDT>(x_row + (s * kMxStep + 8 * q) * kSize, col + 8 * q < k);
          uint32_t top = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) top = mx_top_max<XDT>(top, mx_piece_top<XDT>(v[q]));
          xs[j] = mx_scale_of(mx_top_bits<XDT>(top));
#pragma unroll
          for (int q = 0; q < 4; ++q) xc[j][q] = mx_piece_codes<XDT>(v[q], xs[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
        if (j == 0 || STEPS * p + j < steps)
#pragma unroll
          for (int t = 0; t < TILES; ++t) acc[t] = mx_mfma(w[t][j], xc[j], acc[t], ws[t][j] >> (8 * lq), xs[j]);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    // thread -> (row m, column c): a lane's four sums are columns 4 lq .. 4 lq + 3 of row l16
#pragma unroll
    for (int i = tid; i < kRowsM * kRowsN; i += THREADS) {
      const int m = i / kRowsN, c = i % kRowsN;
      auto total = [&](int t) {
        const int at = m + 16 * (c % 16 / 4);
        float v = part[0][t][at][c % 4];
#pragma unroll
        for (int u = 1; u < WAVES; ++u) v += part[u][t][at][c % 4];
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
        for (int o = 16; o >= 1; o >>= 1)
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, kWave)));
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
    if (r0 + static_cast<int64_t>(layers) * kRowsM < end) __syncthreads();  // the sums are read before the next chunk's
  }
}

template <int XDT>
int launch_t(const MxProduct& p, hipStream_t stream) {
  const bool gateup = p.h_codes != nullptr;
  // hidden rows are written to their padded width
  const int64_t col_tiles = ceil_div(gateup ? mx_padded(p.n) : p.n, kRowsN);
  const int64_t chunks = ceil_div(p.rows, kRowsM);
  const int64_t layers = p.offsets ? std::min<int64_t>(chunks, kRowsLayers) : chunks;
  const int64_t grid = col_tiles * layers * p.groups;
  if (grid > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows and columns for one microscaled product");
  const void* x = XDT == kStored ? p.x_codes : p.x;
  auto go = [&](auto kernel, int waves) {
    kernel<<<static_cast<unsigned>(grid), waves * kWave, 0, stream>>>(
        x, p.x_stride, p.x_scales, p.offsets, static_cast<int>(p.groups),
        static_cast<int>(p.rows), p.a, p.b, static_cast<int>(p.n), static_cast<int>(p.k), static_cast<int>(col_tiles),
        static_cast<int>(layers), p.out, p.out_dtype, p.zero_rest, p.h_codes, p.h_scales);
  };
  // a wave per turn of steps, four or eight: more waves than turns would idle
  const int64_t steps = mx_padded(p.k) / kMxStep;
  if (gateup && steps > 4 * kRowsSteps<XDT, true>) go(mx_rows_kernel<XDT, true, 8>, 8);
  else if (gateup) go(mx_rows_kernel<XDT, true, 4>, 4);
  else if (steps > 4 * kRowsSteps<XDT, false>) go(mx_rows_kernel<XDT, false, 8>, 8);
  else go(mx_rows_kernel<XDT, false, 4>, 4);
  QW_LAUNCH_CHECK("mx_rows_kernel");
  return QW_OK;
}

}  // namespace

bool mx_rows_takes(const void* x, int dtype, int64_t stride, int64_t k) {
  return reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * (dtype == QW_F32 ? 4 : 2) % 16 == 0 && k % 8 == 0;
}

int launch_mx_rows(const MxProduct& p, hipStream_t stream) {
  if (p.x_codes) return launch_t<kStored>(p, stream);
  if (p.x_dtype == QW_F32) return launch_t<QW_F32>(p, stream);
  if (p.x_dtype == QW_F16) return launch_t<QW_F16>(p, stream);
  return launch_t<QW_BF16>(p, stream);
}

}  // namespace qw
