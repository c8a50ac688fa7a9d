// Microscaled 4-bit floating point (MX): device pieces shared by its kernels.
//
// A row of numbers is cut into blocks of 32.  A block is one 8-bit scale s, the
// power of two 2^(s - 127) (255: NaN), and 32 codes of 4 bits: sign, two
// exponent bits and one mantissa bit, the values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives.  Stored rows have their columns padded to whole 128: one step
// of the matrix instruction, v_mfma_scale_f32_16x16x128_f8f6f4, in which lane l
// holds block l / 16 of row l % 16 (16 bytes of codes, the even column of a byte
// in its low nibble) and that block's scale.
//
// From numbers to a block: with m = max |v| the scale is 2^(floor(log2 m) - 2),
// at least 2^-127, so m / scale lies in [4, 8); v / scale is rounded to the
// nearest code, ties to the even one, and what lies past 6 becomes 6.  A block
// holding an infinity or a NaN gets the NaN scale and zero codes: everything it
// is multiplied with becomes NaN.  A block of zeros has scale byte 0.
#pragma once
#include "qw_mfma.h"

namespace qw {

constexpr int kMxBlock = 32;   // columns of a block
constexpr int kMxStep = 128;   // columns of a matrix-instruction step; rows are padded to whole steps
constexpr int kMxNan = 255;    // the scale byte that makes a block NaN

inline int64_t mx_padded(int64_t cols) { return ceil_div(cols, kMxStep) * kMxStep; }
inline int64_t mx_code_bytes(int64_t cols) { return mx_padded(cols) / 2; }
inline int64_t mx_scale_bytes(int64_t cols) { return mx_padded(cols) / kMxBlock; }

// Lanes of a wave have written LDS that others of it read next (or the reverse):
// the wave's LDS accesses are in order, the compiler has to keep them so.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ i32x8 mx_operand(u32x4 v) {
  return i32x8{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
}

// acc += the product of 128 columns: 16 rows of a (accumulator rows), 16 rows of b
// (accumulator columns); lane l holds block l / 16 of row l % 16.  Scales in byte
// 0 of sa and sb.  The products are exact and are added in fp32.
__device__ __forceinline__ f32x4 mx_mfma(u32x4 a, u32x4 b, f32x4 acc, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(a), mx_operand(b), acc, 4, 4, 0,
                                                          static_cast<int>(sa), 0, static_cast<int>(sb));
}

// The same for 64 columns of 32 by 32 rows: lane l holds block l / 32 of row
// l % 32, scales in byte BYTE; accumulator element e of a lane is row
// 8 (e / 4) + 4 (l / 32) + e % 4 of a, row l % 32 of b.
template <int BYTE>
__device__ __forceinline__ f32x16 mx_mfma32(u32x4 a, u32x4 b, f32x16 acc, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a), mx_operand(b), acc, 4, 4, BYTE,
                                                         static_cast<int>(sa), BYTE, static_cast<int>(sb));
}

// Scale byte of a block from the fp32 bits of its largest magnitude.
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t top_bits) {
  const int e = static_cast<int>(top_bits >> 23);  // floor(log2) + 127; 0 below the normal range
  return e == 255 ? kMxNan : static_cast<uint32_t>(max(e - 2, 0));
}

// 2^(s - 127); NaN for 255.  Byte 0 is the subnormal 2^-127.
__device__ __forceinline__ float mx_scale_value(uint32_t s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == kMxNan ? 0x7fc00000u : s << 23);
}

// The scale the conversion instructions divide by (their result is discarded
// where the block is NaN).
__device__ __forceinline__ float mx_divisor(uint32_t s) { return mx_scale_value(s == kMxNan ? 127u : s); }

// Two values onto byte SEL of `into`: v / scale, rounded to the nearest code
// (ties to even, saturating), which v_cvt_scalef32_pk_fp4_* do exactly for every
// power of two from 2^-127 to 2^125 (compared with the definition over the grid's
// midpoints, their neighbours and the saturated range).
template <int SEL>
__device__ __forceinline__ uint32_t mx_pack_f32(uint32_t into, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(into, a, b, scale, SEL);
}
template <int DT, int SEL>
__device__ __forceinline__ uint32_t mx_pack_half(uint32_t into, uint32_t pair, float scale) {
  if constexpr (DT == QW_F16) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(into, __builtin_bit_cast(f16x2_t, pair), scale, SEL);
  } else {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(into, __builtin_bit_cast(bf16x2_t, pair), scale, SEL);
  }
}

// Eight consecutive numbers as they lie in memory: four packed pairs (16-bit
// types) or eight words (fp32).
template <int DT>
struct MxPiece {
  static constexpr int WORDS = DT == QW_F32 ? 8 : 4;
  uint32_t w[WORDS];
};

// Piece of `p` (elements i .. i + 7, of which the first `valid` exist; the rest
// are zeros).  aligned: i starts on 16 bytes.
template <int DT>
__device__ __forceinline__ MxPiece<DT> mx_load_piece(const void* __restrict__ p, int64_t i, int valid, bool aligned) {
  MxPiece<DT> r;
  if (aligned && valid >= 8) {
    if constexpr (DT == QW_F32) {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
      const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i + 4);
      r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
      r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
      r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    }
    return r;
  }
  if constexpr (DT == QW_F32) {
#pragma unroll
    for (int k = 0; k < 8; ++k) r.w[k] = k < valid ? static_cast<const uint32_t*>(p)[i + k] : 0u;
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = 2 * k < valid ? h[2 * k] : 0u, hi = 2 * k + 1 < valid ? h[2 * k + 1] : 0u;
      r.w[k] = lo | (hi << 16);
    }
  }
  return r;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

// The largest magnitude of a piece: magnitude bits of a float type are ordered
// as whole numbers, infinities and NaNs above everything.  fp32 bits, or for the
// 16-bit types the larger half still to be taken (mx_top_bits).
template <int DT>
__device__ __forceinline__ uint32_t mx_piece_top(const MxPiece<DT>& v) {
  constexpr uint32_t MASK = DT == QW_F32 ? 0x7fffffffu : 0x7fff7fffu;
  uint32_t m = v.w[0] & MASK;
#pragma unroll
  for (int k = 1; k < MxPiece<DT>::WORDS; ++k) {
    const uint32_t o = v.w[k] & MASK;
    if constexpr (DT == QW_F32) m = max(m, o);
    else m = max_u16x2(m, o);
  }
  return m;
}
template <int DT>
__device__ __forceinline__ uint32_t mx_top_max(uint32_t a, uint32_t b) {
  if constexpr (DT == QW_F32) return max(a, b);
  else return max_u16x2(a, b);
}
// fp32 bits of the magnitude behind mx_piece_top.
template <int DT>
__device__ __forceinline__ uint32_t mx_top_bits(uint32_t m) {
  if constexpr (DT == QW_F32) return m;
  const uint32_t h = max(m & 0xffffu, m >> 16);
  if constexpr (DT == QW_BF16) return h << 16;
  else return __float_as_uint(f16_to_f32(static_cast<uint16_t>(h)));
}

// The eight codes of a piece under scale byte s.
template <int DT>
__device__ __forceinline__ uint32_t mx_piece_codes(const MxPiece<DT>& v, uint32_t s) {
  const float scale = mx_divisor(s);
  uint32_t r = 0;
  if constexpr (DT == QW_F32) {
    r = mx_pack_f32<0>(r, __uint_as_float(v.w[0]), __uint_as_float(v.w[1]), scale);
    r = mx_pack_f32<1>(r, __uint_as_float(v.w[2]), __uint_as_float(v.w[3]), scale);
    r = mx_pack_f32<2>(r, __uint_as_float(v.w[4]), __uint_as_float(v.w[5]), scale);
    r = mx_pack_f32<3>(r, __uint_as_float(v.w[6]), __uint_as_float(v.w[7]), scale);
  } else {
    r = mx_pack_half<DT, 0>(r, v.w[0], scale);
    r = mx_pack_half<DT, 1>(r, v.w[1], scale);
    r = mx_pack_half<DT, 2>(r, v.w[2], scale);
    r = mx_pack_half<DT, 3>(r, v.w[3], scale);
  }
  return s == kMxNan ? 0u : r;
}

// silu(g) * u of the fp32 accumulators; the product is rounded once, to its code.
__device__ __forceinline__ float mx_swiglu(float g, float u) { return silu_fast(g) * u; }

}  // namespace qw
