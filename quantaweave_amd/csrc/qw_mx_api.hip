// C ABI entry points of the microscaled (MX) operators: argument checks,
// workspace carving and kernel selection.
#include <algorithm>

#include "qw_mx_product.h"

namespace qw {

int grouped_matmul_backward(const void* gy, const void* x, const void* w, int dtype, int wfmt, int64_t E, int64_t N,
                            int64_t K, const int32_t* offsets, int64_t rows, int64_t max_rows_per_expert, void* gx,
                            int accumulate, void* gw, int gw_dtype, void* ws, size_t ws_bytes, hipStream_t stream);
int grouped_f32_dx(const float* gy, const float* w, int64_t N, int64_t K, int64_t w_pitch, const int32_t* offsets,
                   int64_t rows, float* gx, hipStream_t stream);
int gemm_dx(const void* gy, const void* w, int64_t N, int64_t K, int64_t w_pitch, const int32_t* offsets, int64_t rows,
            void* gx, hipStream_t stream);
bool gemm_tr_dx_fits(const void* gy, const void* w, const void* gx, int64_t E, int64_t N, int64_t K, int64_t rows,
                     bool pair, bool tiles128);
int gemm_tr_dx(const void* gy0, const void* gy1, const void* w0, const void* w1, int dtype, bool tiled, int64_t E,
               int64_t N, int64_t K, int64_t w_pitch, const int32_t* offsets, int64_t rows, void* gx,
               hipStream_t stream);
int gemm_tr_dx_split(const void* high, const void* low, const void* w, int64_t N, int64_t K, int64_t w_pitch,
                     const int32_t* offsets, int64_t rows, void* gx, hipStream_t stream);

namespace {

constexpr int64_t kMaxCols = int64_t{1} << 24;

int check_act(int dtype) {
  QW_REQUIRE(dtype == QW_F32 || dtype == QW_BF16 || dtype == QW_F16, "dtype must be f32, bf16 or f16");
  return QW_OK;
}

int check_sizes(int64_t rows, int64_t out_features, int64_t in_features) {
  QW_REQUIRE(rows >= 0 && rows <= INT32_MAX / 64, "rows out of range: %lld", (long long)rows);
  QW_REQUIRE(out_features >= 1 && out_features <= kMaxCols, "out_features out of range: %lld",
             (long long)out_features);
  QW_REQUIRE(in_features >= 1 && in_features <= kMaxCols, "in_features out of range: %lld", (long long)in_features);
  return QW_OK;
}

int check_matrix(const void* codes, const void* scales, const char* what) {
  QW_REQUIRE(codes && scales, "%s codes and scales are required", what);
  QW_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
             "%s codes must start on 16 bytes and its scales on 4", what);
  return QW_OK;
}

MxMatrix matrix(const void* codes, const void* scales) {
  return MxMatrix{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales)};
}

// Workspace of the rows' gradient, gx = gy . W on the framework's backward products.
//
// Whatever the widths, the matrix cores take it: W is dequantised into a copy of its
// own, so its rows are padded with zeros to the tiles' slices of the reduction (64
// rows; 4 in fp32) and its columns to whole loads, and gy is copied to the padded
// width where that differs (30 rows, 1000 columns, 3001 outputs, whole calls: bf16 448
// us on the vector ALU, 75 so; fp32 with 64 rows and 1001 columns 527 and 87).
//
// The matrix is held in bf16 for 16-bit rows, fp16 ones too: stored weights reach
// from 2^-128 to 6 * 2^127, past fp16 at both ends, and bf16 has their range and more
// bits than a code.  fp16's eleven bits of gy then go as two bf16 numbers whose fp32
// sums are added before the one rounding.  (The matrix in fp16 took half the
// instructions and was right for scales of 2^-23 to 2^13 alone: 1024 rows, 1024
// columns and 7168 outputs 110 us a call, 118 so; 8000 rows of 64 columns 104 and 161.)
struct RowsGradient {
  int64_t n, pitch;  // W's padded rows and columns
  bool copied;       // gy is taken from `rows`
  int32_t* offsets;
  void* w;
  void* rows;        // gy, padded; fp16: its high parts
  void* low;         // fp16: its low parts
  size_t bytes;
  RowsGradient(void* workspace, int64_t count, int64_t out_features, int64_t in_features, int dtype) {
    const int64_t slice = dtype == QW_F32 ? 4 : 64, load = dtype == QW_F32 ? 4 : 8, size = dtype == QW_F32 ? 4 : 2;
    n = ceil_div(out_features, slice) * slice;
    pitch = ceil_div(in_features, load) * load;
    // (the vector-ALU kernel, which takes a gy off 16 bytes, goes to 65535 * 64 outputs)
    copied = dtype == QW_F16 || n != out_features || n > 65535 * 64;
    Carver c(workspace);
    offsets = c.take<int32_t>(2);
    w = c.take<char>(static_cast<size_t>(n) * pitch * size);
    rows = c.take<char>(copied ? static_cast<size_t>(count) * n * size : 0);
    low = c.take<char>(dtype == QW_F16 ? static_cast<size_t>(count) * n * size : 0);
    bytes = c.used + 256;
  }
};

__global__ void mx_offsets_kernel(int32_t* offsets, int rows) {
  offsets[0] = 0;
  offsets[1] = rows;
}

}  // namespace

}  // namespace qw

using namespace qw;

extern "C" {

int qw_mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_row_stride, void* codes,
                   void* scales, void* stream) {
  clear_error();
  int st = check_act(x_dtype);
  if (st) return st;
  QW_REQUIRE(rows >= 0, "rows must be >= 0");
  QW_REQUIRE(cols >= 1 && cols <= kMaxCols, "cols out of range: %lld", (long long)cols);
  QW_REQUIRE(x_row_stride >= 0, "x_row_stride must be >= 0");
  if (rows == 0) return QW_OK;
  QW_REQUIRE(x != nullptr, "x is required");
  st = check_matrix(codes, scales, "output");
  if (st) return st;
  return mx_quantize(x, x_dtype, rows, cols, x_row_stride, codes, scales, as_stream(stream));
}

int qw_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int out_dtype,
                     void* stream) {
  clear_error();
  int st = check_act(out_dtype);
  if (st) return st;
  QW_REQUIRE(rows >= 0, "rows must be >= 0");
  QW_REQUIRE(cols >= 1 && cols <= kMaxCols, "cols out of range: %lld", (long long)cols);
  if (rows == 0) return QW_OK;
  QW_REQUIRE(out != nullptr, "out is required");
  st = check_matrix(codes, scales, "input");
  if (st) return st;
  return mx_dequantize(codes, scales, rows, cols, out, out_dtype, rows, as_stream(stream));
}

size_t qw_mx_matmul_workspace_bytes(const void* x, int act_dtype, int64_t x_row_stride, int64_t rows,
                                    int64_t out_features, int64_t in_features) {
  if (rows < 1 || out_features < 1 || in_features < 1) return 0;
  if (mx_few_rows(rows, 1) && mx_rows_takes(x, act_dtype, x_row_stride, in_features)) return 0;
  Carver c(nullptr);
  c.take<char>(static_cast<size_t>(rows) * mx_code_bytes(in_features));
  c.take<char>(static_cast<size_t>(rows) * mx_scale_bytes(in_features));
  return c.used + 256;
}

int qw_mx_matmul(const void* x, int act_dtype, int64_t x_row_stride, int64_t rows, const void* codes,
                 const void* scales, int64_t out_features, int64_t in_features, void* out, void* workspace,
                 size_t workspace_bytes, void* stream) {
  clear_error();
  int st = check_act(act_dtype);
  if (st) return st;
  st = check_sizes(rows, out_features, in_features);
  if (st) return st;
  QW_REQUIRE(x_row_stride >= 0, "x_row_stride must be >= 0");
  if (rows == 0) return QW_OK;
  QW_REQUIRE(x && out, "x and out are required");
  st = check_matrix(codes, scales, "weight");
  if (st) return st;
  const size_t need = qw_mx_matmul_workspace_bytes(x, act_dtype, x_row_stride, rows, out_features, in_features);
  const bool few = mx_few_rows(rows, 1), direct = need == 0;
  if (!direct && (workspace == nullptr || workspace_bytes < need))
    return set_error(QW_ERR_WORKSPACE, "mx_matmul needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
  MxProduct p;
  p.rows = rows, p.n = out_features, p.k = in_features;
  p.a = matrix(codes, scales);
  p.out = out, p.out_dtype = act_dtype;
  if (direct) {
    p.x = x, p.x_dtype = act_dtype, p.x_stride = x_row_stride;
    return launch_mx_rows(p, as_stream(stream));
  }
  Carver c(workspace);
  uint8_t* xq = c.take<uint8_t>(static_cast<size_t>(rows) * mx_code_bytes(in_features));
  uint8_t* xs = c.take<uint8_t>(static_cast<size_t>(rows) * mx_scale_bytes(in_features));
  p.x_codes = xq, p.x_scales = xs;
  if (few) {
    st = mx_quantize(x, act_dtype, rows, in_features, x_row_stride, xq, xs, as_stream(stream));
    return st ? st : launch_mx_rows(p, as_stream(stream));
  }
  st = mx_prepare(x, act_dtype, rows, in_features, x_row_stride, xq, xs, MxPrepare(), as_stream(stream));
  if (st) return st;
  p.chunk_rows = mx_dense_chunk(rows, out_features);
  return launch_mx_gemm(p, as_stream(stream));
}

size_t qw_mx_matmul_backward_workspace_bytes(int64_t rows, int64_t out_features, int64_t in_features, int dtype) {
  if (rows < 1 || out_features < 1 || in_features < 1) return 0;
  return RowsGradient(nullptr, rows, out_features, in_features, dtype).bytes;
}

int qw_mx_matmul_backward(const void* grad_out, int dtype, int64_t rows, const void* codes, const void* scales,
                          int64_t out_features, int64_t in_features, void* grad_x, void* workspace,
                          size_t workspace_bytes, void* stream) {
  clear_error();
  int st = check_act(dtype);
  if (st) return st;
  st = check_sizes(rows, out_features, in_features);
  if (st) return st;
  if (rows == 0) return QW_OK;
  QW_REQUIRE(grad_out && grad_x, "grad_out and grad_x are required");
  st = check_matrix(codes, scales, "weight");
  if (st) return st;
  const size_t need = qw_mx_matmul_backward_workspace_bytes(rows, out_features, in_features, dtype);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(QW_ERR_WORKSPACE, "mx_matmul_backward needs a workspace of %zu bytes, got %zu", need,
                     workspace_bytes);
  const RowsGradient g(workspace, rows, out_features, in_features, dtype);
  const hipStream_t s = as_stream(stream);
  mx_offsets_kernel<<<1, 1, 0, s>>>(g.offsets, static_cast<int>(rows));
  QW_LAUNCH_CHECK("mx_offsets_kernel");
  const int wdt = dtype == QW_F32 ? QW_F32 : QW_BF16;
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!g.copied && !aligned(grad_out)) {  // no copy and no 16-byte loads: the vector-ALU kernel
    st = mx_dequantize(codes, scales, out_features, in_features, g.w, wdt, out_features, s);
    const int64_t size = dtype == QW_F32 ? 4 : 2, most = 65535 * 64;  // rows of one grid
    for (int64_t r = 0; !st && r < rows; r += most) {
      const int64_t some = std::min(most, rows - r);
      st = grouped_matmul_backward(static_cast<const char*>(grad_out) + r * out_features * size, nullptr, g.w, dtype,
                                   dtype, 1, out_features, in_features, g.offsets, some, some,
                                   static_cast<char*>(grad_x) + r * in_features * size, 0, nullptr, dtype, nullptr, 0, s);
    }
    return st;
  }
  st = mx_dequantize(codes, scales, out_features, g.pitch, g.w, wdt, g.n, s);
  if (st) return st;
  if (dtype == QW_F16) st = mx_split(grad_out, rows, out_features, g.n, g.rows, g.low, s);
  else if (g.copied) st = mx_pad(grad_out, dtype == QW_F32 ? 4 : 2, rows, out_features, g.n, g.rows, s);
  if (st) return st;
  const void* const gy = g.copied ? g.rows : grad_out;
  if (dtype == QW_F32)
    return grouped_f32_dx(static_cast<const float*>(gy), static_cast<const float*>(g.w), g.n, in_features, g.pitch,
                          g.offsets, rows, static_cast<float*>(grad_x), s);
  if (dtype == QW_F16)
    return gemm_tr_dx_split(gy, g.low, g.w, g.n, in_features, g.pitch, g.offsets, rows, grad_x, s);
  // tiles of 128 x 128 as in the grouped backward, which need whole fours and 16-byte rows of results
  const bool tiles128 = in_features % 4 == 0 && aligned(grad_x);
  if (tiles128 && !gemm_tr_dx_fits(gy, g.w, grad_x, 1, g.n, in_features, rows, false, true))
    return gemm_dx(gy, g.w, g.n, in_features, g.pitch, g.offsets, rows, grad_x, s);
  return gemm_tr_dx(gy, nullptr, g.w, nullptr, QW_BF16, false, 1, g.n, in_features, g.pitch, g.offsets, rows, grad_x, s);
}

size_t qw_mx_experts_workspace_bytes(int64_t max_rows, int64_t experts, int64_t d_model, int64_t d_ff) {
  if (max_rows < 0 || experts < 1 || d_model < 1 || d_ff < 1) return 0;
  Carver c(nullptr);
  c.take<char>(static_cast<size_t>(max_rows) * mx_code_bytes(d_ff));
  c.take<char>(static_cast<size_t>(max_rows) * mx_scale_bytes(d_ff));
  c.take<char>(static_cast<size_t>(max_rows) * mx_code_bytes(d_model));
  c.take<char>(static_cast<size_t>(max_rows) * mx_scale_bytes(d_model));
  if (!mx_few_rows(max_rows, experts)) {
    c.take<int4>(static_cast<size_t>(mx_max_chunks(max_rows, experts, 64)) + 1);  // the smallest chunks
  }
  return c.used + 256;
}

int qw_mx_experts(const void* x, int act_dtype, int64_t x_row_stride, const int32_t* kept_offsets, int64_t experts,
                  int64_t d_model, int64_t d_ff, int64_t max_rows, int64_t max_rows_per_expert,
                  const void* gate_codes, const void* gate_scales, const void* up_codes, const void* up_scales,
                  const void* down_codes, const void* down_scales, int zero_rest, void* y, void* workspace,
                  size_t workspace_bytes, void* stream) {
  clear_error();
  int st = check_act(act_dtype);
  if (st) return st;
  st = check_sizes(max_rows, d_ff, d_model);
  if (st) return st;
  QW_REQUIRE(experts >= 1 && experts <= 65535, "experts out of range: %lld", (long long)experts);
  QW_REQUIRE(x_row_stride >= 0 && max_rows_per_expert >= 0, "strides and bounds must be >= 0");
  if (max_rows == 0) return QW_OK;
  QW_REQUIRE(x && y && kept_offsets, "x, y and kept_offsets are required");
  st = check_matrix(gate_codes, gate_scales, "gate");
  if (!st) st = check_matrix(up_codes, up_scales, "up");
  if (!st) st = check_matrix(down_codes, down_scales, "down");
  if (st) return st;
  const size_t need = qw_mx_experts_workspace_bytes(max_rows, experts, d_model, d_ff);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(QW_ERR_WORKSPACE, "mx_experts needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
  Carver c(workspace);
  MxProduct p, d;
  p.h_codes = c.take<uint8_t>(static_cast<size_t>(max_rows) * mx_code_bytes(d_ff));
  p.h_scales = c.take<uint8_t>(static_cast<size_t>(max_rows) * mx_scale_bytes(d_ff));
  p.offsets = kept_offsets, p.groups = experts, p.rows = max_rows;
  p.n = d_ff, p.k = d_model;
  p.a = matrix(gate_codes, gate_scales), p.b = matrix(up_codes, up_scales);
  d.x_codes = p.h_codes, d.x_scales = p.h_scales;
  d.offsets = kept_offsets, d.groups = experts, d.rows = max_rows;
  d.n = d_model, d.k = d_ff;
  d.a = matrix(down_codes, down_scales);
  d.out = y, d.out_dtype = act_dtype;
  uint8_t* xq = c.take<uint8_t>(static_cast<size_t>(max_rows) * mx_code_bytes(d_model));
  uint8_t* xs = c.take<uint8_t>(static_cast<size_t>(max_rows) * mx_scale_bytes(d_model));
  if (mx_few_rows(max_rows, experts)) {
    if (mx_rows_takes(x, act_dtype, x_row_stride, d_model)) {
      p.x = x, p.x_dtype = act_dtype, p.x_stride = x_row_stride;
    } else {
      st = mx_quantize(x, act_dtype, max_rows, d_model, x_row_stride, xq, xs, as_stream(stream));
      if (st) return st;
      p.x_codes = xq, p.x_scales = xs;
    }
    st = launch_mx_rows(p, as_stream(stream));
    d.zero_rest = zero_rest != 0;
    return st ? st : launch_mx_rows(d, as_stream(stream));
  }
  const int64_t cap = max_rows_per_expert > 0 && max_rows_per_expert < max_rows ? max_rows_per_expert : max_rows;
  MxPrepare prep;
  prep.offsets = kept_offsets, prep.groups = experts;
  prep.chunk_rows = p.chunk_rows = d.chunk_rows = mx_group_chunk(max_rows, experts, cap);
  prep.table = c.take<int4>(static_cast<size_t>(mx_max_chunks(max_rows, experts, prep.chunk_rows)) + 1);
  prep.zero_out = zero_rest ? y : nullptr;
  p.table = d.table = prep.table;
  st = mx_prepare(x, act_dtype, max_rows, d_model, x_row_stride, xq, xs, prep, as_stream(stream));
  if (st) return st;
  p.x_codes = xq, p.x_scales = xs;
  st = launch_mx_gemm(p, as_stream(stream));
  return st ? st : launch_mx_gemm(d, as_stream(stream));
}

}  // extern "C"
