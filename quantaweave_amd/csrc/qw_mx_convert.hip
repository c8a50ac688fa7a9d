// Rows of numbers <-> microscaled rows (qw_mx.h).
#include "qw_mx_product.h"

namespace qw {

namespace {

constexpr int kConvertThreads = 256;

// Chunks of up to `chunk` rows of each group, in group order, by one workgroup:
// table[0].x their number, then {group, first row, rows, 0}.
__device__ void chunk_table(const int32_t* __restrict__ offsets, int groups, int rows, int chunk, int most,
                            int4* __restrict__ table) {
  __shared__ int wave_total[kConvertThreads / kWave], total;
  int carry = 0;
  for (int e0 = 0; e0 < groups; e0 += kConvertThreads) {
    const int e = e0 + threadIdx.x;
    int lo = 0, n = 0;
    if (e < groups) {
      lo = min(max(offsets[e], 0), rows);
      n = max(min(offsets[e + 1], rows) - lo, 0);
    }
    const int c = (n + chunk - 1) / chunk;
    const int at = carry + block_exclusive_scan(c, wave_total, &total);
    for (int i = 0; i < c && at + i < most; ++i)
      table[1 + at + i] = make_int4(e, lo + i * chunk, min(n - i * chunk, chunk), 0);
    carry += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) table[0] = make_int4(min(carry, most), 0, 0, 0);
}

// Four lanes make a block: each loads eight consecutive numbers (16 bytes of a
// 16-bit type), the largest magnitude goes round the four with two DPP moves.
template <int DT>
__device__ __forceinline__ uint32_t block_scale(const MxPiece<DT>& v) {
  uint32_t top = mx_piece_top<DT>(v);
  top = mx_top_max<DT>(top, dpp_u32<kDppXor1>(top));
  top = mx_top_max<DT>(top, dpp_u32<kDppXor2>(top));
  return mx_scale_of(mx_top_bits<DT>(top));
}

// Each lane stores four bytes of codes, a block's first lane its scale byte.
// Padding columns are written as zeros.  Bound by HBM (8192 x 2048 bf16, 42 MB:
// 9.0 us, 4.7 TB/s; a copy reaches 5.1).
template <int DT>
__global__ __launch_bounds__(kConvertThreads) void mx_quantize_kernel(const void* __restrict__ x, int64_t stride,
                                                                      int cols, uint32_t pieces, int64_t total,
                                                                      bool aligned, uint32_t* __restrict__ codes,
                                                                      uint8_t* __restrict__ scales) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kConvertThreads + threadIdx.x;
  if (i >= total) return;  // whole blocks: total is a multiple of 16 and the four lanes of a block go together
  const int64_t row = total <= INT32_MAX ? static_cast<uint32_t>(i) / pieces : i / pieces;
  const int col = static_cast<int>(i - row * pieces) * 8;
  const MxPiece<DT> v = mx_load_piece<DT>(x, row * stride + col, cols - col, aligned);
  const uint32_t s = block_scale<DT>(v);
  codes[i] = mx_piece_codes<DT>(v, s);
  if (threadIdx.x % 4 == 0) scales[i / 4] = static_cast<uint8_t>(s);
}

// Rows for the tile kernel, the scales step by step.  A workgroup holds
// sixteen rows by sixteen lanes, a step of 128 columns, and goes through up to
// kPrepareSteps of them: the scales of a step are one dword per row, sixteen rows
// side by side.  The last workgroup makes the chunk table; rows of no group are
// skipped and their results zeroed.  16384 x 2048 bf16: 17.1 us (86 MB, 5.0 TB/s);
// a row per workgroup took 18.3 us and the zeroing a fill of its own, 11 us.
constexpr int kPrepareRows = 16, kPrepareSteps = 4;

template <int DT>
__global__ __launch_bounds__(kConvertThreads) void mx_prepare_kernel(const void* __restrict__ x, int64_t stride,
                                                                     int rows, int cols, int steps, int step_groups,
                                                                     bool aligned, MxPrepare prep, int most,
                                                                     uint32_t* __restrict__ codes,
                                                                     uint32_t* __restrict__ scales) {
  if (prep.table != nullptr && blockIdx.x == gridDim.x - 1) {
    chunk_table(prep.offsets, static_cast<int>(prep.groups), rows, prep.chunk_rows, most, prep.table);
    return;
  }
  const int row = static_cast<int>(blockIdx.x / step_groups) * kPrepareRows + threadIdx.x / 16;
  const int s0 = static_cast<int>(blockIdx.x % step_groups) * kPrepareSteps;
  if (row >= rows) return;  // sixteen lanes together
  const int piece = threadIdx.x % 16;
  if (prep.offsets != nullptr && row >= prep.offsets[prep.groups]) {
    if (prep.zero_out != nullptr)
      for (int j = 0; j < kPrepareSteps; ++j)
        for (int k = 0; k < 8; ++k) {
          const int col = (s0 + j) * kMxStep + piece * 8 + k;
          if (col < cols) store_act<DT>(prep.zero_out, static_cast<int64_t>(row) * cols + col, 0.0f);
        }
    return;
  }
  const int64_t base = row * stride;
  MxPiece<DT> v[kPrepareSteps];
#pragma unroll
  for (int j = 0; j < kPrepareSteps; ++j) {
    const int col = (s0 + j) * kMxStep + piece * 8;
    v[j] = mx_load_piece<DT>(x, base + col, cols - col, aligned);
  }
#pragma unroll
  for (int j = 0; j < kPrepareSteps; ++j) {
    if (s0 + j >= steps) break;
    uint32_t s = block_scale<DT>(v[j]);
    codes[static_cast<int64_t>(row) * steps * 16 + (s0 + j) * 16 + piece] = mx_piece_codes<DT>(v[j], s);
    // the four blocks' bytes meet in the step's first lane
    s <<= 8 * (piece / 4);
    s |= dpp_u32<kDppHalfMirror>(s);
    s |= dpp_u32<kDppMirror>(s);
    if (piece == 0) scales[static_cast<int64_t>(s0 + j) * rows + row] = s;
  }
}

// A lane turns four bytes of codes into eight numbers: code times scale is exact
// in fp32 (subnormals included) and is rounded once to the output type.  Rows of
// `cols` columns are written, which may reach into the stored padding; with MORE the
// pieces from `stored` on are rows past the stored ones, written as zeros (a kernel of
// its own: the comparison took 0.8 us more of every call).  Bound by HBM (8192 x 2048
// to bf16, 42 MB: 9.0 us, 4.7 TB/s).
template <int DT, bool MORE>
__global__ __launch_bounds__(kConvertThreads) void mx_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                                        const uint8_t* __restrict__ scales, int cols,
                                                                        uint32_t pieces, int64_t total, bool aligned,
                                                                        void* __restrict__ out, int64_t stored) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kConvertThreads + threadIdx.x;
  if (i >= total) return;
  const int64_t row = total <= INT32_MAX ? static_cast<uint32_t>(i) / pieces : i / pieces;
  const int col = static_cast<int>(i - row * pieces) * 8;
  if (col >= cols) return;
  const bool there = !MORE || i < stored;
  const float s = there ? mx_scale_value(scales[i / 4]) : 0.0f;
  const uint32_t c = there ? codes[i] : 0u;
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3)};
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = p[k / 2][k % 2] * s;
  const int64_t o = row * cols + col;
  if (aligned && col + 8 <= cols) {
    store_vec<DT, 8>(out, o, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col + k < cols) store_act<DT>(out, o + k, v[k]);
  }
}

// Rows padded with zeros to `pitch` columns, a multiple of 4, four of them per lane.
template <typename T>
__global__ __launch_bounds__(kConvertThreads) void mx_pad_kernel(const T* __restrict__ x, int cols, int pitch,
                                                                 int64_t total, bool fours, T* __restrict__ out) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kConvertThreads + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / (pitch / 4);
  const int col = static_cast<int>(i - row * (pitch / 4)) * 4;
  const T* const at = x + row * cols + col;
  T4 v = {0, 0, 0, 0};
  if (fours && col < cols) {
    v = *reinterpret_cast<const T4*>(at);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < cols) v[k] = at[k];
  }
  reinterpret_cast<T4*>(out)[i] = v;
}

// fp16 numbers as the sum of two bf16 ones: the number rounded to eight bits, and
// the rest, which has three bits at most (0 beside an infinity or a NaN).  Rows are
// padded with zeros to `pitch` columns (whole eights).
__global__ __launch_bounds__(kConvertThreads) void mx_split_kernel(const void* __restrict__ x, int cols, int pitch,
                                                                   int64_t total, bool aligned,
                                                                   uint4* __restrict__ high, uint4* __restrict__ low) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kConvertThreads + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / (pitch / 8);
  const int col = static_cast<int>(i - row * (pitch / 8)) * 8;
  const MxPiece<QW_F16> v = mx_load_piece<QW_F16>(x, row * cols + col, cols - col, aligned);
  uint32_t h[4], l[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a[2], rest[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      a[u] = f16_to_f32(static_cast<uint16_t>(v.w[k] >> (16 * u)));
      const float d = a[u] - bf16_to_f32(f32_to_bf16(a[u]));
      rest[u] = d - d == 0.0f ? d : 0.0f;
    }
    h[k] = pack_half2<QW_BF16>(a[0], a[1]);
    l[k] = pack_half2<QW_BF16>(rest[0], rest[1]);
  }
  high[i] = make_uint4(h[0], h[1], h[2], h[3]);
  low[i] = make_uint4(l[0], l[1], l[2], l[3]);
}

}  // namespace

int mx_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, void* codes, void* scales,
                hipStream_t stream) {
  const int64_t pieces = mx_padded(cols) / 8, total = rows * pieces;
  if (total == 0) return QW_OK;
  const int64_t blocks = ceil_div(total, kConvertThreads);
  if (blocks > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows to quantise in one call");
  const int size = dtype == QW_F32 ? 4 : 2;
  const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * size % 16 == 0;
  auto go = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), kConvertThreads, 0, stream>>>(
        x, stride, static_cast<int>(cols), static_cast<uint32_t>(pieces), total, aligned,
        static_cast<uint32_t*>(codes), static_cast<uint8_t*>(scales));
  };
  if (dtype == QW_F32) go(mx_quantize_kernel<QW_F32>);
  else if (dtype == QW_F16) go(mx_quantize_kernel<QW_F16>);
  else go(mx_quantize_kernel<QW_BF16>);
  QW_LAUNCH_CHECK("mx_quantize_kernel");
  return QW_OK;
}

int mx_prepare(const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, uint8_t* codes, uint8_t* scales,
               const MxPrepare& prep, hipStream_t stream) {
  if (rows == 0) return QW_OK;
  const int64_t steps = mx_padded(cols) / kMxStep, step_groups = ceil_div(steps, kPrepareSteps);
  const int64_t blocks = ceil_div(rows, kPrepareRows) * step_groups + (prep.table ? 1 : 0);
  if (blocks > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows to quantise in one call");
  const int size = dtype == QW_F32 ? 4 : 2;
  const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * size % 16 == 0;
  const int most = prep.table ? static_cast<int>(mx_max_chunks(rows, prep.groups, prep.chunk_rows)) : 0;
  auto go = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), kConvertThreads, 0, stream>>>(
        x, stride, static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(steps),
        static_cast<int>(step_groups), aligned, prep, most, reinterpret_cast<uint32_t*>(codes),
        reinterpret_cast<uint32_t*>(scales));
  };
  if (dtype == QW_F32) go(mx_prepare_kernel<QW_F32>);
  else if (dtype == QW_F16) go(mx_prepare_kernel<QW_F16>);
  else go(mx_prepare_kernel<QW_BF16>);
  QW_LAUNCH_CHECK("mx_prepare_kernel");
  return QW_OK;
}

int mx_pad(const void* x, int size, int64_t rows, int64_t cols, int64_t pitch, void* out, hipStream_t stream) {
  const int64_t total = rows * (pitch / 4), blocks = ceil_div(total, kConvertThreads);
  if (blocks > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows to pad in one call");
  const bool fours = cols % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * size) == 0;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    mx_pad_kernel<T><<<static_cast<unsigned>(blocks), kConvertThreads, 0, stream>>>(
        static_cast<const T*>(x), static_cast<int>(cols), static_cast<int>(pitch), total, fours, static_cast<T*>(out));
  };
  if (size == 4) go(uint32_t{0});
  else go(uint16_t{0});
  QW_LAUNCH_CHECK("mx_pad_kernel");
  return QW_OK;
}

int mx_split(const void* x, int64_t rows, int64_t cols, int64_t pitch, void* high, void* low, hipStream_t stream) {
  const int64_t total = rows * (pitch / 8), blocks = ceil_div(total, kConvertThreads);
  if (blocks > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows to split in one call");
  const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && cols % 8 == 0;
  mx_split_kernel<<<static_cast<unsigned>(blocks), kConvertThreads, 0, stream>>>(
      x, static_cast<int>(cols), static_cast<int>(pitch), total, aligned, static_cast<uint4*>(high),
      static_cast<uint4*>(low));
  QW_LAUNCH_CHECK("mx_split_kernel");
  return QW_OK;
}

int mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int dtype,
                  int64_t out_rows, hipStream_t stream) {
  const int64_t pieces = mx_padded(cols) / 8, stored = rows * pieces, total = out_rows * pieces;
  if (total == 0) return QW_OK;
  const int64_t blocks = ceil_div(total, kConvertThreads);
  if (blocks > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many rows to dequantise in one call");
  const int size = dtype == QW_F32 ? 4 : 2;
  const bool aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0 && cols * size % 16 == 0;
  const unsigned g = static_cast<unsigned>(blocks);
  const int c = static_cast<int>(cols);
  const uint32_t p = static_cast<uint32_t>(pieces);
  const uint32_t* q = static_cast<const uint32_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  auto go = [&](auto kernel) { kernel<<<g, kConvertThreads, 0, stream>>>(q, s, c, p, total, aligned, out, stored); };
  const bool more = out_rows > rows;
  if (dtype == QW_F32) more ? go(mx_dequantize_kernel<QW_F32, true>) : go(mx_dequantize_kernel<QW_F32, false>);
  else if (dtype == QW_F16) go(mx_dequantize_kernel<QW_F16, false>);  // (the gradient holds the matrix in bf16)
  else more ? go(mx_dequantize_kernel<QW_BF16, true>) : go(mx_dequantize_kernel<QW_BF16, false>);
  QW_LAUNCH_CHECK("mx_dequantize_kernel");
  return QW_OK;
}

}  // namespace qw
