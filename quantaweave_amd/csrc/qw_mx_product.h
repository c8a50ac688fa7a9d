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
// one group holding all `rows`).
//   one matrix  : out[r] = x[r] . a[n]               [rows, n] of out_dtype
//   two matrices: h[r] = silu(x[r] . a[n]) * (x[r] . b[n]), stored microscaled:
//                 h_codes [rows, padded(n) / 2] and h_scales
// launch_mx_rows takes numbers of x_dtype (x, x_stride) or stored rows (x_codes,
// x_scales), with the scales of stored rows and of h as [rows][padded / 32].
// launch_mx_gemm takes stored rows in row order, with the scales of rows and of h
// step by step, [padded / 128][rows][4], and grouped rows as a chunk table:
// table[0].x chunks, table[1 + i] = {group, first row, rows, 0} of up to chunk_rows.
struct MxProduct {
  const void* x = nullptr;
  int x_dtype = QW_F32;
  int64_t x_stride = 0;
  const uint8_t* x_codes = nullptr;
  const uint8_t* x_scales = nullptr;
  const int32_t* offsets = nullptr;
  const int4* table = nullptr;
  int chunk_rows = 0;
  int64_t groups = 1, rows = 0, n = 0, k = 0;
  MxMatrix a{nullptr, nullptr}, b{nullptr, nullptr};
  void* out = nullptr;
  int out_dtype = QW_F32;
  bool zero_rest = false;  // launch_mx_rows: rows of no group become zeros
  uint8_t* h_codes = nullptr;
  uint8_t* h_scales = nullptr;
};

// Few rows per group: weights streamed, K split over the waves of a workgroup.
// Rows as numbers have to be ones that mx_rows_takes.
bool mx_rows_takes(const void* x, int dtype, int64_t stride, int64_t k);
int launch_mx_rows(const MxProduct& p, hipStream_t stream);
// Many rows (stored ones): tiles of the matrix instruction through LDS.
int launch_mx_gemm(const MxProduct& p, hipStream_t stream);
// Row chunks of launch_mx_gemm: one dense group, and grouped rows with a bound on a group's.
int mx_dense_chunk(int64_t rows, int64_t n);
int mx_group_chunk(int64_t rows, int64_t groups, int64_t cap);
// Most chunks that `rows` rows in `groups` groups make, and the bytes of their table.
inline int64_t mx_max_chunks(int64_t rows, int64_t groups, int chunk) { return ceil_div(rows, chunk) + groups; }

// Whether a product of `rows` rows in `groups` groups is one of few rows: on average as
// many as the matrix instruction holds, so that launch_mx_rows reads a weight once
// where the groups are even (a group's further sixteens of rows are further passes over
// its weights there; the tile kernel's smallest tile is 64 rows).  Neither the bound nor
// the effect of uneven groups was timed with both kernels.
inline bool mx_few_rows(int64_t rows, int64_t groups) { return rows <= groups * 16; }

// What launch_mx_gemm's rows need beside quantisation, in the same pass.
struct MxPrepare {
  const int32_t* offsets = nullptr;    // grouped rows: the chunk table
  int64_t groups = 0;
  int4* table = nullptr;
  int chunk_rows = 0;
  void* zero_out = nullptr;            // rows of no group become zeros here ([rows, cols] of x's type)
};
int mx_prepare(const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, uint8_t* codes, uint8_t* scales,
               const MxPrepare& prep, hipStream_t stream);

int mx_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, void* codes, void* scales,
                hipStream_t stream);
// The first `cols` columns (the stored padding may be among them) of each row; rows
// behind the stored ones up to out_rows become zeros.
int mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int dtype,
                  int64_t out_rows, hipStream_t stream);
// Rows padded with zeros to `pitch` columns (both in elements of `size` bytes, 2 or 4).
int mx_pad(const void* x, int size, int64_t rows, int64_t cols, int64_t pitch, void* out, hipStream_t stream);
// Rows of fp16 numbers as sums of two bf16 rows, padded with zeros to `pitch` columns.
int mx_split(const void* x, int64_t rows, int64_t cols, int64_t pitch, void* high, void* low, hipStream_t stream);

}  // namespace qw
