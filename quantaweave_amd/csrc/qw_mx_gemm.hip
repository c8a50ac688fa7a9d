// Microscaled products of many rows on the scaled matrix instruction.
//
// The chip holds one workgroup (8 waves) per compute unit, each with a list of
// tiles: a row chunk (up to 32 * SUBT rows of one group) by 256 stored weight
// rows, 256 columns of the result, or 128 gate rows with the matching 128 up rows
// for 128 hidden columns.  Operands move HBM/L2 -> LDS with global_load_lds in
// slices of one matrix step (128 columns: 64 bytes of codes and four scale bytes
// per row) through a ring of as many stages as the LDS holds (four at 320 rows,
// seven at 64).  The ring runs on across tiles: while a tile's last slices are
// multiplied and its result is stored, the first slices of the next are on their
// way, so that neither a start nor an epilogue leaves the memory idle.  One tile
// per workgroup, whose slices of 256 columns began anew with each, took for 16384
// rows of 64 experts (d 2048, f 1024) 65 us for gate and up and 51 us for down, now
// 66 and 42; for 4099 rows of popular experts (d 4096, f 1408) 149 and 95 us, now
// 139 and 76; a product of few tiles has nothing to run on into and loses (1023 x
// 1408 x 4096: 11.3 us, now 13.9).  Bound by the matrix instructions: 8192 x 2048 x
// 7168 in 80 us, 3.0 PFLOP/s; a slice of 320 rows takes about 2000 cycles of which
// its instructions issue in 1280.
// Every wave issues the same number of loads per slice (rows past the end are
// clamped to a valid row, their results never stored; past the last slice the
// last one is requested again), so a fixed vmcnt marks a slice as landed.
//
// LDS rows are 64 bytes, four 16-byte pieces, each one block of 32 columns; pieces
// are stored XOR-swizzled so that the sixteen rows that a quarter wave reads cover
// all banks.  Rows are stored ones in row order, their scales step by
// step: dword [step][row].
//
// Waves form a 2 x 4 grid: wave (wm, wn) multiplies row tiles wm, wm + 2, ... (32
// rows each) by its 64 weight rows, with the instruction of 32 x 32 rows and 64
// columns (the 16 x 16 one issues twice the instructions for the same reads: 1743
// against 1499 cycles a slice with every operand from LDS).  A lane's half h takes
// blocks 2h and 2h + 1 of the slice, in the two steps, so one 16-bit read holds
// both scales.  The weights are the instruction's first operand, so a lane holds
// columns of one row; weight rows are dealt to the instruction's rows so that its
// columns are consecutive: 32 of the result (whole 128-byte lines per row), or 16
// hidden ones.  A wave's 32 hidden columns are one block of the hidden row: its
// largest magnitude goes across the two lanes that share the row, and
// silu(gate) * up leaves as codes, a quarter of the bytes of a 16-bit row.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qw_mx_product.h"

namespace qw {

namespace {

constexpr int MX_ROWB = 64;     // bytes of codes per row and slice: 128 columns
constexpr int MX_NB = 256;      // weight rows per tile
constexpr int MX_THREADS = 512;
constexpr int MX_WAVES = 8;
constexpr int MX_LDS = 160 * 1024;
constexpr int kCus = 256;

enum { MX_HIDDEN = -1 };        // epilogue: microscaled silu(gate) * up; else the output's dtype

constexpr int mx_stage(int subt) { return (32 * subt + MX_NB) * (MX_ROWB + 4); }
constexpr int mx_stages(int subt) { return MX_LDS / mx_stage(subt) < 8 ? MX_LDS / mx_stage(subt) : 8; }

struct MxTiles {
  int n_tiles, row_chunks;  // row_chunks: of one dense group (chunk table NULL)
};

template <int EPI, int SUBT>
__global__ __launch_bounds__(MX_THREADS) void mx_gemm_kernel(
    const uint8_t* __restrict__ x_codes, const uint8_t* __restrict__ x_scales, int rows,
    const int4* __restrict__ table, MxMatrix wa, MxMatrix wb, int n, int k_padded, MxTiles grid,
    void* __restrict__ out, bool wide, uint8_t* __restrict__ h_codes, uint8_t* __restrict__ h_scales) {
  constexpr bool GATEUP = EPI == MX_HIDDEN;
  constexpr int MCH = 32 * SUBT;
  constexpr int AG = MCH / 16, CG = AG + MX_NB / 16;       // 16-row load groups of codes: rows, then weights
  constexpr int XG = MCH / 64, SG = XG + MX_NB / 64;       // 64-row load groups of scales
  constexpr int CL = (CG + MX_WAVES - 1) / MX_WAVES, SL = (SG + MX_WAVES - 1) / MX_WAVES, LOADS = CL + SL;
  constexpr int STAGE = mx_stage(SUBT), ST = mx_stages(SUBT), AHEAD = ST - 1;
  constexpr int B_AT = AG * 1024, XS_AT = CG * 1024, WS_AT = XS_AT + XG * 256;
  static_assert(SUBT % 2 == 0 && WS_AT + MX_NB * 4 == STAGE && AHEAD >= 2 && AHEAD * LOADS < 64, "ring");
  static_assert(CG % 4 == 0 && CL * MX_WAVES - CG <= 4 && AG % 4 == 0, "groups per wave and their swizzles");
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wm = wave / 4, wn = wave % 4;
  const uint32_t cb = k_padded / 2, sb = k_padded / kMxBlock;  // bytes of a row
  const int KT = k_padded / kMxStep;

  // ---- this workgroup's tiles: one run of all tiles per XCD, dealt to its units ----
  const int xcd = blockIdx.x % kXcds, unit = blockIdx.x / kXcds, units = gridDim.x / kXcds;
  const int64_t all = static_cast<int64_t>(table ? table[0].x : grid.row_chunks) * grid.n_tiles;
  const int first = static_cast<int>(all * xcd / kXcds), last = static_cast<int>(all * (xcd + 1) / kXcds);
  struct Tile {
    int e, r0, count, n0;
  };
  auto tile_at = [&](int t) {
    Tile r;
    int nt;
    if (table) {  // chunk by chunk: the tiles side by side share their rows
      const int4 c = table[1 + t / grid.n_tiles];
      nt = t % grid.n_tiles;
      r.e = c.x, r.r0 = c.y, r.count = c.z;
    } else {  // blocks of 8 row chunks by all columns
      const int block = 8 * grid.n_tiles, b0 = t / block * 8;
      const int high = min(8, grid.row_chunks - b0), q = t % block;
      nt = q / high;
      r.e = 0, r.r0 = (b0 + q % high) * MCH, r.count = min(rows - r.r0, MCH);
    }
    r.n0 = nt * (GATEUP ? MX_NB / 2 : MX_NB);
    return r;
  };
  int at = first + unit;
  if (at >= last) return;

  // ---- loads ----
  // Slot q of a wave is one load: of rows, or of weight rows (a wave-uniform fact).
  const uint32_t lane_c = lane / 4 * cb, lane_s = lane * sb;
  const uint32_t x_piece = ((lane % 4) ^ (lane / 16)) * 16;
  const uint32_t w_piece = ((lane % 4) ^ (((GATEUP ? wave : wave >> 1) & 1) | (lane / 16 & 1) << 1)) * 16;
  Tile req{0, 0, 0, 0};  // the tile whose slices are being requested; the first is set by the first advance
  int req_kt = KT, req_at = at - units, stage = 0;
  struct Slot {
    int64_t base;              // address of the slice in the slot's first row
    uint32_t row0, end;        // first row and last valid row, in bytes from there
  };
  Slot code_slot[CL], scale_slot[SL];
  // group of a wave's load q (past the last group four back: another wave's group, the same swizzle)
  auto code_group = [&](int q) {
    const int g = wave + q * MX_WAVES;
    return g >= CG ? g - 4 : g;
  };
  auto scale_group = [&](int q) { return min(wave + q * MX_WAVES, SG - 1); };
  auto set_slots = [&] {
    auto addr = [](const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); };
    const int64_t w_row0 = static_cast<int64_t>(req.e) * n + req.n0;
    // (the matrix's last row where the tile has it: bytes from the tile's first row, within 32 bits)
    const uint32_t x_end = req.count - 1, w_end = min(n - 1 - req.n0, MX_NB - 1);
#pragma unroll
    for (int q = 0; q < CL; ++q) {
      const int g = code_group(q), gw = g - AG;
      const bool up = GATEUP && gw >= MX_NB / 32;
      Slot& s = code_slot[q];
      s.base = gw < 0 ? addr(x_codes) + static_cast<int64_t>(req.r0) * cb
                      : addr(up ? wb.codes : wa.codes) + w_row0 * cb;
      s.row0 = 16 * (gw < 0 ? g : up ? gw - MX_NB / 32 : gw) * cb;
      s.end = (gw < 0 ? x_end : w_end) * cb;
    }
#pragma unroll
    for (int q = 0; q < SL; ++q) {
      const int g = scale_group(q), gw = g - XG;
      const bool up = GATEUP && gw >= MX_NB / 128;
      Slot& s = scale_slot[q];
      s.base = gw < 0 ? addr(x_scales) + static_cast<int64_t>(req.r0) * 4
                      : addr(up ? wb.scales : wa.scales) + w_row0 * sb;
      s.row0 = 64 * (gw < 0 ? g * 4 : (up ? gw - MX_NB / 128 : gw) * sb);
      s.end = gw < 0 ? x_end * 4 : w_end * sb;
    }
  };
  const int64_t xs_step = static_cast<int64_t>(rows) * 4;  // from step to step of the rows' scales
  auto request = [&] {
    char* const st = smem + stage;
#pragma unroll
    for (int q = 0; q < CL; ++q) {
      const int g = code_group(q);
      Slot& s = code_slot[q];
      const uint32_t off = min(s.row0 + lane_c, s.end) + (g < AG ? x_piece : w_piece);
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint8_t*>(static_cast<uintptr_t>(s.base)) + off,
                                       (lds_void*)(st + g * 1024), 16, 0, 0);
      s.base += MX_ROWB;
    }
#pragma unroll
    for (int q = 0; q < SL; ++q) {
      const int g = scale_group(q);
      Slot& s = scale_slot[q];
      const uint32_t off = min(s.row0 + (g < XG ? lane * 4u : lane_s), s.end);
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint8_t*>(static_cast<uintptr_t>(s.base)) + off,
                                       (lds_void*)(st + XS_AT + g * 256), 4, 0, 0);
      s.base += g < XG ? xs_step : 4;
    }
    stage = stage + STAGE == ST * STAGE ? 0 : stage + STAGE;
    ++req_kt;
  };
  // Before a request, where the tile's slices are all requested: the next tile.
  auto advance = [&] {
    if (req_kt < KT) return;
    if (req_at + units < last) {
      req_at += units;
      req = tile_at(req_at);
    }  // else nothing is left: the last tile's slices again, into stages that are not read
    req_kt = 0;
    set_slots();
  };

  // ---- fragments: one address per operand, the rest are constant offsets ----
  const int l32 = lane % 32, half = lane / 32;
  // instruction row 8j + 4h + c is weight row 4j + c of the lane half h's run
  const int w_run = (l32 >> 3) * 4 + (l32 & 3), w_half = l32 >> 2 & 1;
  const int w_row = GATEUP ? wn * 32 + w_half * 16 + w_run : wn * 64 + w_half * 32 + w_run;
  constexpr int W_TILE = GATEUP ? MX_NB / 2 : 16;  // from weight tile to weight tile: up's rows, or the run's other half
  const int a_lane = (wm * 32 + l32) * MX_ROWB + (((2 * half) ^ (l32 >> 2 & 3)) * 16);
  const int b_lane = B_AT + w_row * MX_ROWB + (((2 * half) ^ (w_half | (l32 >> 3 & 1) << 1)) * 16);
  const int as_lane = XS_AT + (wm * 32 + l32) * 4 + 2 * half, bs_lane = WS_AT + w_row * 4 + 2 * half;
  auto read_a = [&](const char* st, int i, int step) {
    return *reinterpret_cast<const u32x4*>(st + (a_lane ^ (step * 16)) + i * 64 * MX_ROWB);
  };
  auto read_as = [&](const char* st, int i) {
    return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(st + as_lane + i * 64 * 4));
  };
  auto read_b = [&](const char* st, int t, int step) {
    return *reinterpret_cast<const u32x4*>(st + (b_lane ^ (step * 16)) + t * W_TILE * MX_ROWB);
  };
  auto read_bs = [&](const char* st, int t) {
    return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(st + bs_lane + t * W_TILE * 4));
  };
  constexpr int NT = SUBT / 2;  // row tiles of a wave
  f32x16 acc[NT][2];

  // Fragments are read two units (a row tile in a step) ahead of their
  // instructions, across slices too: a slice starts with its first step's weight
  // fragments, both steps' weight scales and its first two units in registers.
  u32x4 w[2], x[2];
  uint32_t ws[2], xs[2];
  auto read_first = [&](const char* st, auto npa) {
    constexpr int NPA = decltype(npa)::value;
#pragma unroll
    for (int t = 0; t < 2; ++t) w[t] = read_b(st, t, 0), ws[t] = read_bs(st, t);
    x[0] = read_a(st, 0, 0), xs[0] = read_as(st, 0);
    x[1] = read_a(st, 1 % NPA, 1 / NPA), xs[1] = read_as(st, 1 % NPA);
  };
  auto slice = [&](auto npa, const char* st, const char* next) {
    constexpr int NPA = decltype(npa)::value, UNITS = 2 * NPA;
    u32x4 xq[UNITS + 2], w1[2], wn[2];
    uint32_t sq[UNITS + 2], wsn[2];  // the scale of a unit; both steps of a tile share it
    xq[0] = x[0], xq[1] = x[1], sq[0] = xs[0], sq[1] = xs[1];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (u == 1) request();
      const int i = u % NPA;
      auto multiply = [&](int t) {
        if (u < NPA) acc[i][t] = mx_mfma32<0>(w[t], xq[u], acc[i][t], ws[t], sq[u]);
        else acc[i][t] = mx_mfma32<1>(w1[t], xq[u], acc[i][t], ws[t], sq[u]);
      };
      multiply(0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      // two units ahead
      const int v = u + 2 < UNITS ? u + 2 : u + 2 - UNITS;
      xq[u + 2] = read_a(u + 2 < UNITS ? st : next, v % NPA, v / NPA);
      if (u + 2 < UNITS && v >= NPA) {
        sq[u + 2] = sq[v - NPA];
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      } else {
        sq[u + 2] = read_as(u + 2 < UNITS ? st : next, v % NPA);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      if (u == 0) {  // the second step's weights
        w1[0] = read_b(st, 0, 1), w1[1] = read_b(st, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      if (u == NPA) {  // the next slice's
        wn[0] = read_b(next, 0, 0), wn[1] = read_b(next, 1, 0);
        wsn[0] = read_bs(next, 0), wsn[1] = read_bs(next, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
      }
      multiply(1);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    x[0] = xq[UNITS], x[1] = xq[UNITS + 1], xs[0] = sq[UNITS], xs[1] = sq[UNITS + 1];
    w[0] = wn[0], w[1] = wn[1], ws[0] = wsn[0], ws[1] = wsn[1];
  };

#pragma unroll 1
  for (int s = 0; s < AHEAD; ++s) {
    advance();
    request();
  }
  wait_vmcnt<LOADS>();  // all but the newest slice
  ring_barrier();
  int read_at = 0;  // the stage that is multiplied
  Tile tile = tile_at(at);
  for (; at < last; at += units) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[i][t][q] = 0.f;
    const int tiles = __builtin_amdgcn_readfirstlane((tile.count + 31) / 32);  // row tiles holding valid rows
    auto k_loop = [&](auto npa) {
      read_first(smem + read_at, npa);
      for (int kt = 0; kt < KT; ++kt) {
        // the slice after this one has landed (a tile's first slices were waited for
        // before the stores of the tile before it) ...
        if (kt >= AHEAD - 2) wait_vmcnt<(AHEAD - 2) * LOADS>();
        ring_barrier();  // ... for every wave, and every wave is done with the slice before this one
        advance();       // ahead of the slice: its matrix instructions stay with its reads in one block
        const int next = read_at + STAGE == ST * STAGE ? 0 : read_at + STAGE;
        slice(npa, smem + read_at, smem + next);
        read_at = next;
      }
    };
    // a wave's row tiles wm, wm + 2, ... below `tiles` hold rows
    const int mine = tiles > wm ? (tiles - wm + 1) / 2 : 0;
    if constexpr (NT >= 2) {
      if (mine > (NT + 1) / 2) k_loop(std::integral_constant<int, NT>{});
      else k_loop(std::integral_constant<int, (NT + 1) / 2>{});
    } else {
      k_loop(std::integral_constant<int, NT>{});
    }
    const Tile done = tile;
    if (at + units < last) tile = tile_at(at + units);
    // the slices requested so far but the newest, before the stores go into the same queue
    wait_vmcnt<LOADS>();

    // ---- epilogue: lane holds row l32 of a tile ----
    const int r0 = done.r0;
    if constexpr (GATEUP) {
      const int64_t np = (n + kMxStep - 1) / kMxStep * static_cast<int64_t>(kMxStep);
      const int c0 = done.n0 + wn * 32 + 16 * half;
      uint8_t* const hs = h_scales + (static_cast<int64_t>(done.n0 / kMxStep) * rows + r0) * 4 + wn;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (wm + 2 * i >= tiles) continue;  // wave-uniform
        const int row = (wm + 2 * i) * 32 + l32;
        float h[16];
        uint32_t top = 0;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          // padding columns of the hidden row are zero codes
          h[q] = c0 + q < n ? mx_swiglu(acc[i][0][q], acc[i][1][q]) : 0.0f;
          top = max(top, __float_as_uint(h[q]) & 0x7fffffffu);
        }
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
        const uint32_t sc = mx_scale_of(top);
        const float div = mx_divisor(sc);
        uint32_t code[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          code[q] = mx_pack_f32<0>(0u, h[8 * q], h[8 * q + 1], div);
          code[q] = mx_pack_f32<1>(code[q], h[8 * q + 2], h[8 * q + 3], div);
          code[q] = mx_pack_f32<2>(code[q], h[8 * q + 4], h[8 * q + 5], div);
          code[q] = mx_pack_f32<3>(code[q], h[8 * q + 6], h[8 * q + 7], div);
          if (sc == kMxNan) code[q] = 0u;
        }
        if (row < done.count) {
          *reinterpret_cast<uint2*>(h_codes + (r0 + row) * (np / 2) + c0 / 2) = make_uint2(code[0], code[1]);
          if (half == 0) hs[row * 4] = static_cast<uint8_t>(sc);
        }
        __builtin_amdgcn_sched_barrier(0);  // tile by tile: the accumulators leave no registers for two
      }
    } else {
      // 16-bit results go through LDS, a row tile at a time in this wave's part of the
      // stage that the next request will fill (free once every wave is done with the
      // last slice), so that a store is eight whole 128-byte lines (a lane's own 16
      // bytes of 32 rows each: 320 x 256 results 12 us instead of 3.5 us).
      constexpr int PASSES = MX_WAVES * 32 * 128 <= STAGE ? 1 : 2;  // sixteen rows at a time in small stages
      constexpr int MINE = 32 * 128 / PASSES;
      static_assert(MX_WAVES * MINE <= STAGE, "the rows of every wave fit a stage");
      const int free_at = read_at == 0 ? (ST - 1) * STAGE : read_at - STAGE;
      char* const st = smem + free_at + wave * MINE;
      if (EPI != QW_F32 && wide) ring_barrier();
      const int col = done.n0 + wn * 64;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (wm + 2 * i >= tiles) continue;
        const int row0 = (wm + 2 * i) * 32;
        if (EPI != QW_F32 && wide) {
          // 16-byte chunk c of row r at chunk c ^ (r & 7): a lane writes chunks of one row, reads one of eight rows
          const int c = lane % 8;
#pragma unroll
          for (int pass = 0; pass < PASSES; ++pass) {
            constexpr int R = 32 / PASSES;
            if (PASSES == 1 || l32 / R == pass) {
#pragma unroll
              for (int q = 0; q < 32; q += 8) {
                u32x4 v;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  v[k] = pack_half2<EPI == QW_F16 ? QW_F16 : QW_BF16>(acc[i][q / 16][q % 16 + 2 * k],
                                                                      acc[i][q / 16][q % 16 + 2 * k + 1]);
                *reinterpret_cast<u32x4*>(st + l32 % R * 128 + (((half * 4 + q / 8) ^ (l32 & 7)) * 16)) = v;
              }
            }
            wave_lds_order();
            u32x4 v[R / 8];
#pragma unroll
            for (int q = 0; q < R / 8; ++q) {
              const int r = q * 8 + lane / 8;
              v[q] = *reinterpret_cast<const u32x4*>(st + r * 128 + ((c ^ (r & 7)) * 16));
            }
            wave_lds_order();
#pragma unroll
            for (int q = 0; q < R / 8; ++q) {
              const int row = row0 + pass * R + q * 8 + lane / 8;
              if (row < done.count && col + c * 8 < n)
                *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(out) + static_cast<int64_t>(r0 + row) * n + col +
                                          c * 8) = v[q];
            }
          }
        } else {
          const int row = row0 + l32, c0 = col + half * 32;
          if (row >= done.count) continue;
          const int64_t o = static_cast<int64_t>(r0 + row) * n + c0;
          if (wide && c0 + 32 <= n) {  // fp32
#pragma unroll
            for (int q = 0; q < 32; q += 4) {
              const float v[4] = {acc[i][q / 16][q % 16], acc[i][q / 16][q % 16 + 1], acc[i][q / 16][q % 16 + 2],
                                  acc[i][q / 16][q % 16 + 3]};
              store_vec<QW_F32, 4>(out, o + q, v);
            }
          } else {
#pragma unroll
            for (int q = 0; q < 32; ++q)
              if (c0 + q < n) store_act<EPI>(out, o + q, acc[i][q / 16][q % 16]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  wait_vmcnt<0>();  // the LDS is not given back while requests for it are on their way
}

template <int EPI, int SUBT>
int launch_t(const MxProduct& p, hipStream_t stream) {
  MxTiles g;
  g.n_tiles = static_cast<int>(EPI == MX_HIDDEN ? ceil_div(p.n, MX_NB / 2) : ceil_div(p.n, MX_NB));
  g.row_chunks = static_cast<int>(ceil_div(p.rows, 32 * SUBT));
  const int64_t chunks = p.table ? g.row_chunks + p.groups : g.row_chunks;
  if (chunks * g.n_tiles > INT32_MAX / 16)
    return set_error(QW_ERR_UNSUPPORTED, "too many tiles for one microscaled product");
  const int64_t units = std::min<int64_t>(kCus / kXcds, ceil_div(chunks * g.n_tiles, kXcds));
  constexpr int lds = mx_stages(SUBT) * mx_stage(SUBT);
  const hipError_t attr = reserve_lds<mx_gemm_kernel<EPI, SUBT>>(lds);
  if (attr != hipSuccess)
    return set_error(QW_ERR_HIP, "cannot reserve %d bytes of LDS: %s", lds, hipGetErrorString(attr));
  const int size = EPI == QW_F32 ? 4 : 2;
  const bool wide = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.n * size % 16 == 0;
  mx_gemm_kernel<EPI, SUBT><<<static_cast<unsigned>(units * kXcds), MX_THREADS, lds, stream>>>(
      p.x_codes, p.x_scales, static_cast<int>(p.rows), p.table, p.a, p.b, static_cast<int>(p.n),
      static_cast<int>(mx_padded(p.k)), g, p.out, wide, p.h_codes, p.h_scales);
  QW_LAUNCH_CHECK("mx_gemm_kernel");
  return QW_OK;
}

template <int EPI>
int launch_sel(const MxProduct& p, hipStream_t stream) {
  switch (p.chunk_rows) {
    case 64: return launch_t<EPI, 2>(p, stream);
    case 128: return launch_t<EPI, 4>(p, stream);
    case 192: return launch_t<EPI, 6>(p, stream);
    case 256: return launch_t<EPI, 8>(p, stream);
    default: return launch_t<EPI, 10>(p, stream);
  }
}

}  // namespace

// Dense rows: the chunk height whose tiles cost the fewest rounds of the chip.  A
// tile costs its rows and, as about 96 rows more, its start and its weight rows (a
// slice of 320 rows about 2000 cycles, the start and store of a tile as much as five).
int mx_dense_chunk(int64_t rows, int64_t n) {
  int best = 64;
  int64_t cost = INT64_MAX;
  for (int h : {64, 128, 192, 256, 320}) {
    const int64_t c = ceil_div(ceil_div(rows, h) * ceil_div(n, MX_NB), kCus) * (h + 96);
    if (c <= cost) best = h, cost = c;
  }
  return best;
}

// Grouped rows: the smallest chunk that holds the usual group (even routing and
// 3.5 standard deviations, within the bound).
int mx_group_chunk(int64_t rows, int64_t groups, int64_t cap) {
  const int64_t avg = std::min(cap, ceil_div(rows, groups));
  const int64_t likely = std::min(cap, avg + static_cast<int64_t>(3.5 * std::sqrt(static_cast<double>(avg))));
  const int64_t want = cap <= 320 && cap <= 2 * avg ? cap : likely;
  for (int h : {64, 128, 192, 256})
    if (want <= h) return h;
  return 320;
}

int launch_mx_gemm(const MxProduct& p, hipStream_t stream) {
  if (p.h_codes) return launch_sel<MX_HIDDEN>(p, stream);
  if (p.out_dtype == QW_F32) return launch_sel<QW_F32>(p, stream);
  if (p.out_dtype == QW_F16) return launch_sel<QW_F16>(p, stream);
  return launch_sel<QW_BF16>(p, stream);
}

}  // namespace qw
