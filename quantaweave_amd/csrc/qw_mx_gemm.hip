// Microscaled products of many rows on the scaled matrix instruction.
//
// One workgroup (8 waves) owns a row chunk (up to 32 * SUBT rows of one group)
// and a tile of 256 stored weight rows: 256 columns of the result, or 128 gate
// rows with the matching 128 up rows for 128 hidden columns.  Operands move
// HBM/L2 -> LDS with global_load_lds in K slices of 256 columns (128 bytes of
// codes, two matrix steps, and eight scale bytes per row) through a ring of two
// or three stages, one barrier per slice, the next slices requested right after
// it.  A load of codes is eight whole 128-byte row segments.  Every wave issues
// the same loads per slice (rows past the end are clamped to a valid row, their
// results never stored), so a fixed vmcnt marks a slice as landed.
//
// LDS rows are 128 bytes; the eight 16-byte pieces of row r, each one block of 32
// columns, are stored XOR-swizzled by (r >> 1) & 7, so the sixteen rows of a
// fragment read hit distinct banks.  A lane's fragment of a step is one block
// (piece 4 * step + lane / 16 of its row) and its scale byte.
//
// Waves form a 2 x 4 grid: wave (wm, wn) multiplies row sub-tiles wm, wm + 2, ...
// (16 rows each) by its 64 weight rows; sub-tiles go in pairs, a pair past the
// rows is not multiplied.  The weights are the instruction's first operand, so a
// lane holds four consecutive columns of one row.  A wave's 32 hidden columns are
// one block of the hidden row: its largest magnitude goes round the four lanes
// that share the row, and silu(gate) * up leaves as codes, a quarter of the bytes
// of a 16-bit row and nothing rounded on the way.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qw_mx_product.h"

namespace qw {

namespace {

constexpr int MX_SLICE = 128;   // bytes of codes per row and slice: 256 columns
constexpr int MX_SROW = 8;      // scale bytes per row and slice
constexpr int MX_NB = 256;      // weight rows per workgroup
constexpr int MX_THREADS = 512;
constexpr int MX_WAVES = 8;
constexpr int MX_NT = 4;        // 16-column tiles per wave
constexpr int MX_LDS = 160 * 1024;
constexpr int64_t kCus = 256;

enum { MX_HIDDEN = -1 };        // epilogue: microscaled silu(gate) * up; else the output's dtype

constexpr int mx_stage(int subt) { return (32 * subt + MX_NB) * (MX_SLICE + MX_SROW); }
constexpr int mx_stages(int subt) { return MX_LDS / mx_stage(subt) >= 3 ? 3 : 2; }

__device__ __forceinline__ int mx_swz(int row, int piece) { return piece ^ ((row >> 1) & 7); }

// Workgroup -> tile.  Grouped rows (run > 0): the chunks that hold rows, found on
// the device and dealt to the XCDs in runs that share their weights
// (find_run_chunk), so that no bound on a group's rows can lose any.  One dense
// group (run 0): the tiles in blocks of 8 row chunks by all columns, cut into one
// contiguous part per XCD.
struct MxGrid {
  int n_tiles, run, row_chunks, per_xcd;
};

template <int EPI, int SUBT>
__global__ __launch_bounds__(MX_THREADS) void mx_gemm_kernel(
    const uint8_t* __restrict__ x_codes, const uint8_t* __restrict__ x_scales, const int32_t* __restrict__ row_index,
    const int32_t* __restrict__ offsets, int max_rows, int groups, MxMatrix wa, MxMatrix wb, int n, int k_padded,
    MxGrid grid, void* __restrict__ out, uint8_t* __restrict__ h_codes, uint8_t* __restrict__ h_scales) {
  constexpr bool GATEUP = EPI == MX_HIDDEN;
  constexpr int MCH = 32 * SUBT;
  constexpr int A_STAGE = MCH * MX_SLICE, B_STAGE = MX_NB * MX_SLICE;
  constexpr int AS_STAGE = MCH * MX_SROW, BS_STAGE = MX_NB * MX_SROW;
  constexpr int STAGE = A_STAGE + B_STAGE + AS_STAGE + BS_STAGE;
  constexpr int ST = mx_stages(SUBT), AHEAD = ST - 1;
  constexpr int AG = MCH / 8, AL = (AG + MX_WAVES - 1) / MX_WAVES;  // 8-row load groups
  constexpr int BL = MX_NB / 8 / MX_WAVES;
  constexpr int ASL = (AS_STAGE / 256 + MX_WAVES - 1) / MX_WAVES;   // 256-byte scale loads
  constexpr int BSL = BS_STAGE / 256 / MX_WAVES;
  constexpr int LOADS = AL + BL + ASL + BSL;
  static_assert(STAGE == mx_stage(SUBT) && ST * STAGE <= MX_LDS && AHEAD * LOADS < 64, "ring");
  static_assert(AG % MX_WAVES == 0, "every wave loads the same number of groups");
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  // ---- tile of this workgroup ----
  const int xcd = blockIdx.x % kXcds, j = blockIdx.x / kXcds;
  int nt, mc = 0, e = 0;
  int lo = 0, hi = max_rows;
  if (grid.run == 0) {
    const int t = xcd * grid.per_xcd + j;
    if (t >= grid.n_tiles * grid.row_chunks) return;
    const int block = 8 * grid.n_tiles, b0 = t / block * 8;
    const int high = min(8, grid.row_chunks - b0);
    const int r = t % block;
    mc = b0 + r % high;
    nt = r / high;
  } else {
    nt = j % grid.n_tiles;
    e = find_run_chunk(offsets, groups, max_rows, MCH, grid.run, xcd, j / grid.n_tiles, &mc);
    if (e < 0) return;
    lo = max(offsets[e], 0);
    hi = min(offsets[e + 1], max_rows);
  }
  const int r0 = lo + mc * MCH;
  const int count = min(hi - r0, MCH);
  if (count <= 0) return;

  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int wm = wave / 4, wn = wave % 4;
  const int l16 = lane % 16, lq = lane / 16;
  const int n0 = nt * (GATEUP ? MX_NB / 2 : MX_NB);
  const uint32_t cb = k_padded / 2, sb = k_padded / kMxBlock;  // bytes of a row
  const int KT = (k_padded + 255) / 256;
  const bool half = k_padded % 256 != 0;  // the last slice holds one step

  // ---- sources of this wave's loads ----
  // lane i of a code load writes LDS row 8g + i/8, physical piece i%8; g has the
  // wave's parity in every load, so the logical piece is one per lane
  const int piece = mx_swz(8 * (wave & 1) + lane / 8, lane % 8);
  const int back = piece >= 4 ? -64 : 0;  // in a half slice the second step's pieces reread the first's
  uint32_t a_src[AL];
#pragma unroll
  for (int q = 0; q < AL; ++q) {
    const int row = 8 * (wave + q * MX_WAVES) + lane / 8;
    const int rr = r0 + min(row, count - 1);
    a_src[q] = static_cast<uint32_t>(row_index ? row_index[rr] : rr) * cb + piece * 16;
  }
  auto weight_row = [&](int row) {
    return static_cast<uint32_t>(GATEUP ? min(n0 + row % (MX_NB / 2), n - 1) : min(n0 + row, n - 1));
  };
  // the weight rows of one load belong to one matrix: the first half of a wave's
  // loads (GATEUP) reads gate, the second up
  const uint8_t* const wa_c = wa.codes + static_cast<int64_t>(e) * n * cb;
  const uint8_t* const wb_c = wb.codes + static_cast<int64_t>(e) * n * cb;
  const uint8_t* const wa_s = wa.scales + static_cast<int64_t>(e) * n * sb;
  const uint8_t* const wb_s = wb.scales + static_cast<int64_t>(e) * n * sb;
  uint32_t b_src[BL];
#pragma unroll
  for (int q = 0; q < BL; ++q)
    b_src[q] = weight_row(8 * (wave + q * MX_WAVES) + lane / 8) * cb + piece * 16;
  // a scale load is 64 dwords: 32 rows, the two steps' four bytes each
  const int sback = lane % 2 ? -4 : 0;
  uint32_t as_src[ASL];
  int as_at[ASL];
#pragma unroll
  for (int q = 0; q < ASL; ++q) {
    const int g = min(wave + q * MX_WAVES, AS_STAGE / 256 - 1);  // the last ones repeat a load
    const int row = 32 * g + lane / 2;
    const int rr = r0 + min(row, count - 1);
    as_src[q] = static_cast<uint32_t>(row_index ? row_index[rr] : rr) * sb + lane % 2 * 4;
    as_at[q] = g * 256;
  }
  const uint32_t bs_src = weight_row(32 * wave + lane / 2) * sb + lane % 2 * 4;
  const uint8_t* const bs_base = GATEUP && __builtin_amdgcn_readfirstlane(wave) >= MX_WAVES / 2 ? wb_s : wa_s;
  static_assert(BSL == 1, "one scale load of weight rows per wave");
  auto issue = [&](int kt) {
    char* const st = smem + (kt % ST) * STAGE;
    const bool cut = half && kt == KT - 1;
    const uint32_t off = kt * MX_SLICE + (cut ? back : 0), soff = kt * MX_SROW + (cut ? sback : 0);
#pragma unroll
    for (int q = 0; q < AL; ++q)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(x_codes + (a_src[q] + off)),
                                       (lds_void*)(st + (wave + q * MX_WAVES) * 1024), 16, 0, 0);
#pragma unroll
    for (int q = 0; q < BL; ++q)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>((GATEUP && q >= BL / 2 ? wb_c : wa_c) + (b_src[q] + off)),
                                       (lds_void*)(st + A_STAGE + (wave + q * MX_WAVES) * 1024), 16, 0, 0);
#pragma unroll
    for (int q = 0; q < ASL; ++q)
      __builtin_amdgcn_global_load_lds(static_cast<const void*>(x_scales + (as_src[q] + soff)),
                                       (lds_void*)(st + A_STAGE + B_STAGE + as_at[q]), 4, 0, 0);
    __builtin_amdgcn_global_load_lds(static_cast<const void*>(bs_base + (bs_src + soff)),
                                     (lds_void*)(st + A_STAGE + B_STAGE + AS_STAGE + wave * 256), 4, 0, 0);
  };

  f32x4 acc[SUBT][MX_NT];
#pragma unroll
  for (int i = 0; i < SUBT; ++i)
#pragma unroll
    for (int t = 0; t < MX_NT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // this lane's fragment in a stage: its row of sub-tile wm, of weight tile 0, and their scales
  const int frag = l16 * MX_SLICE + mx_swz(l16, lq) * 16;
  const int b_row = wn * (GATEUP ? 32 : 64);
  const int a_lane = wm * 16 * MX_SLICE + frag, b_lane = b_row * MX_SLICE + frag;
  const int as_lane = (wm * 16 + l16) * MX_SROW + lq, bs_lane = (b_row + l16) * MX_SROW + lq;
  const int active_sub = (count + 15) / 16;

  for (int s = 0; s < AHEAD && s < KT; ++s) issue(s);

  // One slice: STEPS matrix steps for NPA pairs of sub-tiles.  Fragments of the
  // next unit (a step of a pair) are read right after the first instruction of
  // the current one.
  struct Frag {
    u32x4 v;
    uint32_t s;
  };
  auto slice = [&](auto npa, auto steps, const char* st, auto&& request) {
    constexpr int NPA = decltype(npa)::value, STEPS = decltype(steps)::value;
    // one address per step and operand, the rest are constant offsets: a row's swizzle
    // is that of its lane, and the second step's pieces lie 64 bytes across
    const char* const a0 = st + a_lane;
    const char* const a1 = st + (a_lane ^ 64);
    const char* const b0 = st + A_STAGE + b_lane;
    const char* const b1 = st + A_STAGE + (b_lane ^ 64);
    const char* const as = st + A_STAGE + B_STAGE + as_lane;
    const char* const bs = st + A_STAGE + B_STAGE + AS_STAGE + bs_lane;
    auto read_a = [&](int i, int ks) {
      Frag f;
      f.v = *reinterpret_cast<const u32x4*>((ks ? a1 : a0) + i * 32 * MX_SLICE);
      f.s = *reinterpret_cast<const uint8_t*>(as + i * 32 * MX_SROW + ks * 4);
      return f;
    };
    auto read_b = [&](int t, int ks) {
      const int row = GATEUP ? t / 2 * (MX_NB / 2) + t % 2 * 16 : t * 16;
      Frag f;
      f.v = *reinterpret_cast<const u32x4*>((ks ? b1 : b0) + row * MX_SLICE);
      f.s = *reinterpret_cast<const uint8_t*>(bs + row * MX_SROW + ks * 4);
      return f;
    };
    Frag w[2][MX_NT], xb[2][2];
#pragma unroll
    for (int t = 0; t < MX_NT; ++t) w[0][t] = read_b(t, 0);
    xb[0][0] = read_a(0, 0);
    xb[0][1] = read_a(1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * MX_NT + 4, 0);
    request();
#pragma unroll
    for (int u = 0; u < STEPS * NPA; ++u) {
      const int ks = u / NPA, p = u % NPA;
      const Frag x0 = xb[u & 1][0], x1 = xb[u & 1][1];
      acc[2 * p][0] = mx_mfma(w[ks][0].v, x0.v, acc[2 * p][0], w[ks][0].s, x0.s);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (u + 1 < STEPS * NPA) {
        const int ks1 = (u + 1) / NPA, p1 = (u + 1) % NPA;
        if (ks1 != ks) {
#pragma unroll
          for (int t = 0; t < MX_NT; ++t) w[ks1][t] = read_b(t, ks1);
          xb[(u + 1) & 1][0] = read_a(2 * p1, ks1);
          xb[(u + 1) & 1][1] = read_a(2 * p1 + 1, ks1);
          __builtin_amdgcn_sched_group_barrier(0x100, 2 * MX_NT + 4, 0);
        } else {
          xb[(u + 1) & 1][0] = read_a(2 * p1, ks1);
          xb[(u + 1) & 1][1] = read_a(2 * p1 + 1, ks1);
          __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        }
      }
#pragma unroll
      for (int t = 1; t < MX_NT; ++t) acc[2 * p][t] = mx_mfma(w[ks][t].v, x0.v, acc[2 * p][t], w[ks][t].s, x0.s);
#pragma unroll
      for (int t = 0; t < MX_NT; ++t)
        acc[2 * p + 1][t] = mx_mfma(w[ks][t].v, x1.v, acc[2 * p + 1][t], w[ks][t].s, x1.s);
      __builtin_amdgcn_sched_group_barrier(0x008, 2 * MX_NT - 1, 0);
    }
  };
  constexpr int NP = SUBT / 2;
  static_assert(SUBT % 2 == 0 && AHEAD >= 1 && AHEAD <= 2, "pairs; ring depth");
  auto k_loop = [&](auto npa) {
    using Two = std::integral_constant<int, 2>;
    using One = std::integral_constant<int, 1>;
    // slice kt has landed when only the slices requested after it may be in flight
    int kt = 0;
    for (; kt < KT - AHEAD; ++kt) {
      wait_vmcnt<(AHEAD - 1) * LOADS>();
      ring_barrier();
      slice(npa, Two{}, smem + (kt % ST) * STAGE, [&] { issue(kt + AHEAD); });
    }
    for (const int full = half ? KT - 1 : KT; kt < full; ++kt) {
      if (AHEAD == 2 && kt + 1 < KT) wait_vmcnt<LOADS>();
      else wait_vmcnt<0>();
      ring_barrier();
      slice(npa, Two{}, smem + (kt % ST) * STAGE, [] {});
    }
    if (half) {
      wait_vmcnt<0>();
      ring_barrier();
      slice(npa, One{}, smem + (kt % ST) * STAGE, [] {});
    }
  };
  const int wave_sub = active_sub > wm ? (active_sub - wm + 1) / 2 : 0;
  const int npa = __builtin_amdgcn_readfirstlane((wave_sub + 1) / 2);
  if constexpr (NP >= 4) {
    if (npa >= NP) k_loop(std::integral_constant<int, NP>{});
    else if (npa >= 3) k_loop(std::integral_constant<int, (NP > 4 ? 4 : 3)>{});
    else k_loop(std::integral_constant<int, 2>{});
  } else {
    k_loop(std::integral_constant<int, NP>{});
  }

  // ---- epilogue: lane holds row l16 of a sub-tile, columns 4 lq .. 4 lq + 3 of each tile ----
  if constexpr (GATEUP) {
    const int64_t np = (n + kMxStep - 1) / kMxStep * static_cast<int64_t>(kMxStep);
    const int c0 = n0 + wn * 32 + 4 * lq;
#pragma unroll
    for (int i = 0; i < SUBT; ++i) {
      const int s = wm + 2 * i;
      if (s >= active_sub) continue;  // wave-uniform
      const int row = s * 16 + l16;
      float h[2][4];
      uint32_t top = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          // padding columns of the hidden row are zero codes
          h[t][q] = c0 + t * 16 + q < n ? mx_swiglu(acc[i][t][q], acc[i][t + 2][q]) : 0.0f;
          top = max(top, __float_as_uint(h[t][q]) & 0x7fffffffu);
        }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
      const uint32_t sc = mx_scale_of(top);
      const float div = mx_divisor(sc);
      uint32_t code[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        code[t] = mx_pack_f32<0>(0u, h[t][0], h[t][1], div);
        code[t] = sc == kMxNan ? 0u : mx_pack_f32<1>(code[t], h[t][2], h[t][3], div);
      }
      if (row < count) {
        uint8_t* const o = h_codes + (r0 + row) * (np / 2) + c0 / 2;
        *reinterpret_cast<uint16_t*>(o) = static_cast<uint16_t>(code[0]);
        *reinterpret_cast<uint16_t*>(o + 8) = static_cast<uint16_t>(code[1]);
        if (lq == 0) h_scales[(r0 + row) * (np / kMxBlock) + c0 / kMxBlock] = static_cast<uint8_t>(sc);
      }
    }
  } else {
    const bool vec = n % 4 == 0;
#pragma unroll
    for (int i = 0; i < SUBT; ++i) {
      const int s = wm + 2 * i;
      if (s >= active_sub) continue;
      const int row = s * 16 + l16;
      if (row >= count) continue;
      const int64_t orow = static_cast<int64_t>(r0 + row) * n;
#pragma unroll
      for (int t = 0; t < MX_NT; ++t) {
        const int col = n0 + wn * 64 + t * 16 + 4 * lq;
        const float v[4] = {acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]};
        if (vec && col < n) {
          store_vec<EPI, 4>(out, orow + col, v);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (col + q < n) store_act<EPI>(out, orow + col + q, v[q]);
        }
      }
    }
  }
}

template <int EPI, int SUBT>
int launch_t(const MxProduct& p, hipStream_t stream) {
  constexpr int MCH = 32 * SUBT;
  constexpr bool GATEUP = EPI == MX_HIDDEN;
  MxGrid g;
  g.n_tiles = static_cast<int>(GATEUP ? ceil_div(p.n, MX_NB / 2) : ceil_div(p.n, MX_NB));
  g.row_chunks = static_cast<int>(ceil_div(p.rows, MCH));
  g.per_xcd = g.run = 0;
  int64_t chunks;
  if (p.offsets == nullptr) {
    const int64_t tiles = static_cast<int64_t>(g.n_tiles) * g.row_chunks;
    if (tiles > INT32_MAX / 16) return set_error(QW_ERR_UNSUPPORTED, "too many tiles for one microscaled product");
    g.per_xcd = static_cast<int>(ceil_div(tiles, kXcds));
    chunks = g.per_xcd;
  } else {
    const int run = loose_run(p.rows, p.groups, MCH);
    g.run = run;
    chunks = loose_chunks(p.rows, p.groups, MCH, run) * g.n_tiles;
  }
  const int64_t blocks = kXcds * chunks;
  if (blocks > INT32_MAX) return set_error(QW_ERR_UNSUPPORTED, "too many tiles for one microscaled product");
  constexpr int lds = mx_stages(SUBT) * mx_stage(SUBT);
  const hipError_t attr = reserve_lds<mx_gemm_kernel<EPI, SUBT>>(lds);
  if (attr != hipSuccess)
    return set_error(QW_ERR_HIP, "cannot reserve %d bytes of LDS: %s", lds, hipGetErrorString(attr));
  mx_gemm_kernel<EPI, SUBT><<<static_cast<unsigned>(blocks), MX_THREADS, lds, stream>>>(
      p.x_codes, p.x_scales, p.row_index, p.offsets, static_cast<int>(p.rows), static_cast<int>(p.groups), p.a, p.b,
      static_cast<int>(p.n), static_cast<int>(mx_padded(p.k)), g, p.out, p.h_codes, p.h_scales);
  QW_LAUNCH_CHECK("mx_gemm_kernel");
  return QW_OK;
}

template <int EPI>
int launch_sel(int subt, const MxProduct& p, hipStream_t stream) {
  switch (subt) {
    case 2: return launch_t<EPI, 2>(p, stream);
    case 4: return launch_t<EPI, 4>(p, stream);
    case 6: return launch_t<EPI, 6>(p, stream);
    case 8: return launch_t<EPI, 8>(p, stream);
    default: return launch_t<EPI, 10>(p, stream);
  }
}

// Sub-tile pairs of a workgroup.  Dense rows: the chunk height whose tiles cost
// the fewest rounds of the chip.  Grouped rows: the smallest chunk that holds the
// usual group (even routing and 3.5 standard deviations, within the bound).
int pick_subt(const MxProduct& p, bool gateup) {
  const int64_t n_tiles = gateup ? ceil_div(p.n, MX_NB / 2) : ceil_div(p.n, MX_NB);
  if (p.offsets == nullptr) {
    int best = 2;
    int64_t cost = INT64_MAX;
    for (int s : {2, 4, 6, 8, 10}) {
      // a tile costs its rows and its weight rows' loads
      const int64_t c = ceil_div(ceil_div(p.rows, 32 * s) * n_tiles, kCus) * (32 * s + 96);
      if (c <= cost) best = s, cost = c;
    }
    return best;
  }
  const int64_t avg = std::min(p.row_cap, ceil_div(p.rows, p.groups));
  const int64_t likely = std::min(p.row_cap, avg + static_cast<int64_t>(3.5 * std::sqrt(static_cast<double>(avg))));
  const int64_t rows = p.row_cap <= 320 && p.row_cap <= 2 * avg ? p.row_cap : likely;
  for (int s : {2, 4, 6, 8})
    if (rows <= 32 * s) return s;
  return 10;
}

}  // namespace

int launch_mx_gemm(const MxProduct& p, hipStream_t stream) {
  const bool gateup = p.h_codes != nullptr;
  // rows are addressed by 32-bit offsets from the matrix (or the rows') start
  if (std::max(p.rows, p.x_rows) * mx_code_bytes(p.k) > UINT32_MAX || p.n * mx_code_bytes(p.k) > UINT32_MAX)
    return launch_mx_rows(p, stream);
  const int subt = pick_subt(p, gateup);
  if (gateup) return launch_sel<MX_HIDDEN>(subt, p, stream);
  if (p.out_dtype == QW_F32) return launch_sel<QW_F32>(subt, p, stream);
  if (p.out_dtype == QW_F16) return launch_sel<QW_F16>(subt, p, stream);
  return launch_sel<QW_BF16>(subt, p, stream);
}

}  // namespace qw
