// The products of microscaled rows and matrices: what the launchers take.
#pragma once
#include "qw_mx.h"

namespace qw {

// A stack of stored matrices [groups, n, padded]: codes and scales, 16-byte and
// 4-byte aligned.
struct MxMatrix {
  const uint8_t* codes;
  const uint8_t* scales;
};

// Rows times matrices.  Rows are grouped by `offsets` (device, groups + 1; NULL:
// one group holding all `rows`).  The rows are stored ones (x_codes, x_scales) or
// numbers of x_dtype (x, x_stride), quantised on the way; row_index picks the
// row behind each (NULL: the row itself).
//   one matrix  : out[r] = x[r] . a[n]               [rows, n] of out_dtype
//   two matrices: h[r] = silu(x[r] . a[n]) * (x[r] . b[n]), stored microscaled:
//                 h_codes [rows, padded(n) / 2], h_scales [rows, padded(n) / 32]
struct MxProduct {
  const void* x = nullptr;
  int x_dtype = QW_F32;
  int64_t x_stride = 0;
  const uint8_t* x_codes = nullptr;
  const uint8_t* x_scales = nullptr;
  const int32_t* row_index = nullptr;
  const int32_t* offsets = nullptr;
  int64_t groups = 1, rows = 0, x_rows = 0, row_cap = 0, n = 0, k = 0;  // x_rows: rows behind row_index
  MxMatrix a{nullptr, nullptr}, b{nullptr, nullptr};
  void* out = nullptr;
  int out_dtype = QW_F32;
  uint8_t* h_codes = nullptr;
  uint8_t* h_scales = nullptr;
};

// Few rows per group: weights streamed, K split over the waves of a workgroup.
int launch_mx_rows(const MxProduct& p, hipStream_t stream);
// Many rows (stored ones): tiles of the matrix instruction through LDS.
int launch_mx_gemm(const MxProduct& p, hipStream_t stream);

// Whether a product of `rows` rows in `groups` groups is one of few rows.
inline bool mx_few_rows(int64_t rows, int64_t groups) { return rows <= groups * 16; }

int mx_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, void* codes, void* scales,
                hipStream_t stream);
int mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int dtype,
                  hipStream_t stream);

}  // namespace qw
