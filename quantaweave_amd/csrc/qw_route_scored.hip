// Routing by scores: softmax or sigmoid scores, a balance bias that steers the
// choice alone, groups of experts of which the best are kept, top-k among them
// and renormalised weights; and its gradient.
//
//   s_e   = softmax(l)_e, or 1 / (1 + exp(-l_e))
//   c_e   = s_e + bias_e                        what the choice goes by
//   v_g   = sum of the group's `group_top` (1 or 2) highest c
//   kept  = the top_groups groups of highest v
//   idx   = the top_k highest c among the kept groups' experts, descending
//   w_j   = scale * s_idx_j / (sum_i s_idx_i + 1e-20), or scale * s_idx_j
//
// The choice is the one of 64-bit arithmetic: s, c and v are formed in double, so
// scores next to each other are told apart as the definition does, whatever
// fp32's exponential rounds to; equal values go to the lowest index, a NaN counts
// as -infinity.  A softmax row of -infinities has scores 0 (so weights 0).
#include "qw_common.h"

namespace qw {

int route_validate(int64_t T, int64_t E, int64_t K);

namespace {

constexpr double kRouteEps = 1e-20;
constexpr int kRouteWaves = 4;

// What a call fixes for all its tokens.
struct ScoredRule {
  int softmax, groups, top_groups, group_top, renormalize;
  float scale;
};

// Order-preserving key of a double; NaN as -infinity, -0 as 0.  Never 0: that
// marks an expert that is out (taken, or of a group not kept).
__device__ __forceinline__ uint64_t choice_key(double v) {
  if (v != v) v = -__builtin_inf();
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
  return (b >> 63) ? ~b : b | (1ull << 63);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// Largest value over the wave, in every lane and on the scalar side.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp_u32<kDppXor1>(v));
  v = max(v, dpp_u32<kDppXor2>(v));
  v = max(v, dpp_u32<kDppHalfMirror>(v));
  v = max(v, dpp_u32<kDppMirror>(v));
  const uint32_t a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31);
  const uint32_t c = __builtin_amdgcn_readlane(v, 47), d = __builtin_amdgcn_readlane(v, 63);
  return max(max(a, b), max(c, d));
}

// One wave per token; lane l owns experts l * EPL .. l * EPL + EPL - 1, so the
// lowest lane of a tie has the lowest expert.  A round of the top-k compares the
// upper halves of the 64-bit keys (sign, exponent, 20 bits): one instruction per
// step of the maximum; the lower halves are looked at in the rounds where two
// experts share the largest upper half.
// Bound by one wave's chain of steps, not by bytes: 1 token of 256 experts in 8
// groups, k 8: 7.4 us; 8192 tokens: 24.3 us (17 MB, 0.7 TB/s).
template <int EPL>
__global__ __launch_bounds__(kRouteWaves* kWave) void route_scored_kernel(
    const float* __restrict__ logits, int T, int E, int K, const float* __restrict__ bias, ScoredRule rule,
    float* __restrict__ scores, int32_t* __restrict__ top_idx, float* __restrict__ top_w) {
  __shared__ double choice[kRouteWaves][EPL * kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int t = blockIdx.x * kRouteWaves + wave;
  if (t >= T) return;  // no barrier below: a wave uses its own LDS only
  const int64_t base = static_cast<int64_t>(t) * E;
  float l[EPL];
  bool nan = false;
#pragma unroll
  for (int c = 0; c < EPL; ++c) {
    const int e = lane * EPL + c;
    l[c] = e < E ? logits[base + e] : -__builtin_inff();
    nan |= l[c] != l[c];
  }
  // ---- scores ----
  double s[EPL];
  if (rule.softmax) {
    float m = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < EPL; ++c) m = fmaxf(m, l[c]);
    m = wave_max(m);
    const bool none = m == -__builtin_inff() && !__any(nan);
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < EPL; ++c) {
      s[c] = lane * EPL + c < E && !none ? exp(static_cast<double>(l[c]) - static_cast<double>(m)) : 0.0;
      sum += s[c];
    }
    sum = wave_sum_d(sum);
    if (!none)
#pragma unroll
      for (int c = 0; c < EPL; ++c) s[c] = s[c] / sum;
  } else {
#pragma unroll
    for (int c = 0; c < EPL; ++c) s[c] = lane * EPL + c < E ? 1.0 / (1.0 + exp(-static_cast<double>(l[c]))) : 0.0;
  }
  double sel[EPL];
#pragma unroll
  for (int c = 0; c < EPL; ++c) {
    const int e = lane * EPL + c;
    sel[c] = s[c] + (bias != nullptr && e < E ? static_cast<double>(bias[e]) : 0.0);
    if (sel[c] != sel[c] || e >= E) sel[c] = -__builtin_inf();
    if (e < E) scores[base + e] = static_cast<float>(s[c]);
  }
  // ---- the groups that stay ----
  uint32_t hi[EPL], lo[EPL];
#pragma unroll
  for (int c = 0; c < EPL; ++c) {
    const uint64_t key = lane * EPL + c < E ? choice_key(sel[c]) : 0;
    hi[c] = static_cast<uint32_t>(key >> 32);
    lo[c] = static_cast<uint32_t>(key);
  }
  if (rule.top_groups < rule.groups) {
    const int per = E / rule.groups;
    double* const mine = choice[wave];
#pragma unroll
    for (int c = 0; c < EPL; ++c) mine[lane * EPL + c] = sel[c];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    // lane g (and g + 64, ...): the value of group g, kept at its first expert's place
    for (int g0 = 0; g0 < rule.groups; g0 += kWave) {
      const int g = g0 + lane;
      double a = -__builtin_inf(), b = -__builtin_inf();
      if (g < rule.groups)
        for (int i = 0; i < per; ++i) {
          const double v = mine[g * per + i];
          b = v > a ? a : (v > b ? v : b);
          a = v > a ? v : a;
        }
      double v = rule.group_top == 2 && per > 1 ? a + b : a;
      if (v != v) v = -__builtin_inf();
      if (g < rule.groups) mine[g * per] = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < EPL; ++c) {
      const int e = lane * EPL + c;
      if (e < E) {
        const int g = e / per;
        const double v = mine[g * per];
        int before = 0;
        for (int o = 0; o < rule.groups; ++o) {
          const double u = mine[o * per];
          before += u > v || (u == v && o < g);
        }
        if (before >= rule.top_groups) hi[c] = 0;
      }
    }
  }
  // ---- top-k ----
  int my_e = 0;
  double my_s = 0.0, total = 0.0;
  for (int j = 0; j < K; ++j) {
    uint32_t best = hi[0];
#pragma unroll
    for (int c = 1; c < EPL; ++c) best = max(best, hi[c]);
    best = wave_max_u32(best);
    int found = 0, at = 0, slot = 0;
#pragma unroll
    for (int c = EPL - 1; c >= 0; --c) {
      const unsigned long long mask = __ballot(hi[c] == best);
      found += __popcll(mask);
      if (mask) {
        at = __ffsll(static_cast<long long>(mask)) - 1;
        slot = c;
      }
    }
    if (found > 1) {  // the same upper half: the largest lower half, then the lowest expert
      uint32_t low = 0;
      bool any = false;
      int first = 0;
#pragma unroll
      for (int c = EPL - 1; c >= 0; --c)
        if (hi[c] == best && (!any || lo[c] >= low)) {
          low = lo[c];
          first = c;
          any = true;
        }
      const uint32_t top = wave_max_u32(any ? low : 0u);
      at = __ffsll(static_cast<long long>(__ballot(any && low == top))) - 1;
      slot = __builtin_amdgcn_readlane(first, at);
    }
    double picked = 0.0;
#pragma unroll
    for (int c = 0; c < EPL; ++c)
      if (c == slot) picked = s[c];
    picked = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(picked), at),
                              __builtin_amdgcn_readlane(__double2loint(picked), at));
    total += picked;
#pragma unroll
    for (int c = 0; c < EPL; ++c)
      if (lane == at && c == slot) hi[c] = 0;
    if (lane == j) {
      my_e = at * EPL + slot;
      my_s = picked;
    }
  }
  if (lane < K) {
    top_idx[static_cast<int64_t>(t) * K + lane] = my_e;
    // the quotient of the 64-bit scores: scores that fp32 holds as subnormals keep their digits
    top_w[static_cast<int64_t>(t) * K + lane] =
        static_cast<float>(rule.renormalize ? my_s / (total + kRouteEps) : my_s) * rule.scale;
  }
}

// One wave per token.  With g the gradient of w and idx_j the choices:
//   dp_j  = scale * (g_j - sum_i g_i s_idx_i / S) / S   (S the renormalising sum; scale * g_j without)
//   ds_e  = grad_scores_e + sum_{idx_j = e} dp_j
//   dl_e  = softmax: s_e (ds_e - sum ds s);  sigmoid: ds_e s_e (1 - s_e)
// An index outside [0, E) is skipped.  8192 tokens of 256 experts, k 8, with the
// gradients of both weights and scores: 9.8 us (25 MB, 2.6 TB/s; the choices are dealt
// to their lanes one after another).
template <int EPL>
__global__ __launch_bounds__(kRouteWaves* kWave) void route_scored_backward_kernel(
    const float* __restrict__ scores, const int32_t* __restrict__ top_idx, const float* __restrict__ grad_top_w,
    const float* __restrict__ grad_scores, int T, int E, int K, ScoredRule rule, float* __restrict__ out) {
  const int lane = threadIdx.x % kWave;
  const int t = blockIdx.x * kRouteWaves + threadIdx.x / kWave;
  if (t >= T) return;
  const int64_t base = static_cast<int64_t>(t) * E, krow = static_cast<int64_t>(t) * K;
  int idx = -1;
  float pj = 0.0f, gj = 0.0f;
  if (lane < K && grad_top_w != nullptr) {
    idx = top_idx[krow + lane];
    if (idx < 0 || idx >= E) idx = -1;
    if (idx >= 0) {
      pj = scores[base + idx];
      gj = grad_top_w[krow + lane] * rule.scale;
    }
  }
  float dpj = gj;
  if (rule.renormalize) {
    const float S = wave_sum_f(pj) + static_cast<float>(kRouteEps);
    dpj = (gj - wave_sum_f(gj * pj) / S) / S;
  }
  float s[EPL], ds[EPL];
#pragma unroll
  for (int c = 0; c < EPL; ++c) {
    const int e = lane * EPL + c;
    s[c] = e < E ? scores[base + e] : 0.0f;
    ds[c] = e < E && grad_scores ? grad_scores[base + e] : 0.0f;
  }
  for (int j = 0; j < K; ++j) {
    const int e = __builtin_amdgcn_readlane(idx, j);
    const float d = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(dpj), j));
#pragma unroll
    for (int c = 0; c < EPL; ++c)
      if (lane * EPL + c == e) ds[c] += d;
  }
  if (rule.softmax) {
    float d = 0.0f;
#pragma unroll
    for (int c = 0; c < EPL; ++c) d = __builtin_fmaf(ds[c], s[c], d);
    d = wave_sum_f(d);
#pragma unroll
    for (int c = 0; c < EPL; ++c) ds[c] = s[c] * (ds[c] - d);
  } else {
#pragma unroll
    for (int c = 0; c < EPL; ++c) ds[c] = ds[c] * s[c] * (1.0f - s[c]);
  }
#pragma unroll
  for (int c = 0; c < EPL; ++c) {
    const int e = lane * EPL + c;
    if (e < E) out[base + e] = ds[c];
  }
}

int check_rule(int64_t T, int64_t E, int64_t K, int score, int64_t groups, int64_t top_groups, int group_top,
               float scale) {
  const int st = route_validate(T, E, K);
  if (st) return st;
  QW_REQUIRE(K <= kWave, "top_k must be at most %d, got %lld", kWave, (long long)K);
  QW_REQUIRE(score == 0 || score == 1, "score must be 0 (softmax) or 1 (sigmoid), got %d", score);
  QW_REQUIRE(groups >= 1 && groups <= E && E % groups == 0, "groups must divide the experts (%lld, %lld)",
             (long long)groups, (long long)E);
  QW_REQUIRE(top_groups >= 1 && top_groups <= groups, "top_groups must be in [1, groups], got %lld",
             (long long)top_groups);
  QW_REQUIRE(K <= top_groups * (E / groups), "top_k %lld exceeds the experts of %lld groups", (long long)K,
             (long long)top_groups);
  QW_REQUIRE(group_top == 1 || group_top == 2, "group_top must be 1 or 2, got %d", group_top);
  QW_REQUIRE(scale == scale && scale - scale == 0.0f, "scale must be finite");
  return QW_OK;
}

}  // namespace

int route_scored(const float* logits, int64_t T, int64_t E, int64_t K, int score, const float* bias, int64_t groups,
                 int64_t top_groups, int group_top, int renormalize, float scale, float* scores, int32_t* top_idx,
                 float* top_w, hipStream_t stream) {
  const unsigned grid = static_cast<unsigned>(ceil_div(T, kRouteWaves));
  const ScoredRule rule{score == 0, static_cast<int>(groups), static_cast<int>(top_groups), group_top, renormalize,
                        scale};
  const int t = static_cast<int>(T), e = static_cast<int>(E), k = static_cast<int>(K);
  const int epl = static_cast<int>(ceil_div(E, kWave));
#define QW_RS(N)                                                                                                 \
  route_scored_kernel<N><<<grid, kRouteWaves * kWave, 0, stream>>>(logits, t, e, k, bias, rule, scores, top_idx, \
                                                                   top_w)
  if (epl <= 1) QW_RS(1);
  else if (epl <= 2) QW_RS(2);
  else if (epl <= 4) QW_RS(4);
  else if (epl <= 8) QW_RS(8);
  else QW_RS(16);
#undef QW_RS
  QW_LAUNCH_CHECK("route_scored_kernel");
  return QW_OK;
}

int route_scored_backward(const float* scores, const int32_t* top_idx, const float* grad_top_w,
                          const float* grad_scores, int64_t T, int64_t E, int64_t K, int score, int renormalize,
                          float scale, float* out, hipStream_t stream) {
  const unsigned grid = static_cast<unsigned>(ceil_div(T, kRouteWaves));
  const ScoredRule rule{score == 0, 1, 1, 1, renormalize, scale};
  const int t = static_cast<int>(T), e = static_cast<int>(E), k = static_cast<int>(K);
  const int epl = static_cast<int>(ceil_div(E, kWave));
#define QW_RS(N)                                                                                             \
  route_scored_backward_kernel<N><<<grid, kRouteWaves * kWave, 0, stream>>>(scores, top_idx, grad_top_w,     \
                                                                            grad_scores, t, e, k, rule, out)
  if (epl <= 1) QW_RS(1);
  else if (epl <= 2) QW_RS(2);
  else if (epl <= 4) QW_RS(4);
  else if (epl <= 8) QW_RS(8);
  else QW_RS(16);
#undef QW_RS
  QW_LAUNCH_CHECK("route_scored_backward_kernel");
  return QW_OK;
}

}  // namespace qw

using namespace qw;

extern "C" {

int qw_moe_route_scored_from_logits(const float* logits, int64_t tokens, int64_t experts, int64_t top_k, int score,
                                    const float* bias, int64_t groups, int64_t top_groups, int group_top,
                                    int renormalize, float scale, float* scores, int32_t* top_idx, float* top_w,
                                    void* stream) {
  clear_error();
  const int st = check_rule(tokens, experts, top_k, score, groups, top_groups, group_top, scale);
  if (st) return st;
  if (tokens == 0) return QW_OK;
  QW_REQUIRE(logits && scores && top_idx && top_w, "logits, scores, top_idx and top_w are required");
  return route_scored(logits, tokens, experts, top_k, score, bias, groups, top_groups, group_top, renormalize, scale,
                      scores, top_idx, top_w, as_stream(stream));
}

int qw_moe_route_scored_backward(const float* scores, const int32_t* top_idx, const float* grad_top_w,
                                 const float* grad_scores, int64_t tokens, int64_t experts, int64_t top_k, int score,
                                 int renormalize, float scale, float* grad_logits, void* stream) {
  clear_error();
  const int st = check_rule(tokens, experts, top_k, score, 1, 1, 1, scale);
  if (st) return st;
  if (tokens == 0) return QW_OK;
  QW_REQUIRE(scores && grad_logits, "scores and grad_logits are required");
  QW_REQUIRE(grad_top_w == nullptr || top_idx != nullptr, "grad_top_w needs top_idx");
  return route_scored_backward(scores, top_idx, grad_top_w, grad_scores, tokens, experts, top_k, score, renormalize,
                               scale, grad_logits, as_stream(stream));
}

}  // extern "C"
