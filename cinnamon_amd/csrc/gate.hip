// The experts' gate on gfx950: scores, group limits, top-k and weights of a router's logits, and
// the gradient of the logits (reference src/layers.py:122-126: sigmoid scores, a bias that only
// chooses, top-k, weights that sum to one).
//
//   s      = sigmoid(z) or softmax(z)                       over a token's E experts
//   choice = s + bias
//   group  = sum of the best one or two choices of each of G groups of E / G experts;
//            experts outside the best top_groups groups are left out
//   idx    = the k largest choices left, falling, ties to the lowest index
//   w_j    = scale * s[idx_j] / (sum_j s[idx_j] + 1e-9)     (or scale * s[idx_j])
// backward, with gw and gs the gradients of w and s:
//   ds     = gs;  ds[idx_j] += scale * (gw_j - sum_i gw_i s[idx_i] / total) / total
//   dz     = ds s (1 - s)  or  s (ds - sum_e ds_e s_e)
//
// Scores are ordered in 64 bits: neighbours in the order may differ by less than 32 bits hold.
// NaN counts as the greatest value, in a row and among groups.
//
// A token's experts lie over LANES lanes, EPL consecutive ones a lane, so that the order of the
// lanes is the order of the indices: the lowest of equal candidates is the first lane of a ballot.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "cin_common.h"
#include "cin_runtime.h"

using namespace cin;

namespace {

constexpr int kGateMaxExperts = 4096;
constexpr int kGateMaxTopK = 16;
constexpr int kGateMaxGroups = 64;
constexpr double kEps = 1e-9;

enum Score { kSigmoid = 0, kSoftmax = 1 };

struct GateArgs {
  const void* logits;
  int dtype;
  int64_t ldl;
  const float* bias;
  int64_t T;
  int E, k, score, groups, top_groups, group_top, renormalize;
  float scale;
};

// Keys that order as the values do, NaN above all; 0 is below every key (an expert left out).
__device__ inline uint64_t key_of(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // -0 counts as 0
  if (v != v) return ~0ull;
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ inline double value_of(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

template <int LANES, class V>
__device__ inline V lanes_max(V v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    const V u = __shfl_xor(v, o);
    v = u > v ? u : v;
  }
  return v;
}
template <int LANES, class V>
__device__ inline V lanes_sum(V v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// The first lane of this lane's token for which `mine` holds, or -1.
template <int LANES>
__device__ inline int first_lane(bool mine, int lane) {
  uint64_t m = __ballot(mine);
  if constexpr (LANES < 64) m = (m >> (lane & ~(LANES - 1))) & ((1ull << LANES) - 1);
  return m ? __builtin_ctzll(m) : -1;
}

// Scores of the token's experts, EPL a lane; z holds -inf past E.
template <int LANES, int EPL, class F>
__device__ inline void scores(int kind, const float (&z)[EPL], F (&s)[EPL]) {
  if (kind == kSigmoid) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = 1 / (1 + exp(-(F)z[j]));
  } else {
    F m = z[0];
#pragma unroll
    for (int j = 0; j < EPL; ++j) m = z[j] > m || z[j] != z[j] ? (F)z[j] : m;
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      const F u = __shfl_xor(m, o);
      m = u > m || u != u ? u : m;
    }
    F t = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) t += s[j] = exp((F)z[j] - m);
    t = lanes_sum<LANES>(t);
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] /= t;
  }
}

template <int EPL>
__device__ inline void load_logits(const GateArgs& a, int64_t t, int e0, float (&z)[EPL]) {
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    z[j] = e0 + j < a.E ? load_elem(a.logits, a.dtype, t * a.ldl + e0 + j) : -__builtin_inff();
}

// One token a wave: its keys through LDS for the groups, then k rounds of a maximum.
template <int LANES, int EPL, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_gate_fwd(GateArgs a, int64_t* __restrict__ idx, float* __restrict__ w,
                                                         float* __restrict__ all) {
  constexpr int kTokens = 64 / LANES * WAVES;
  __shared__ uint64_t sk[kTokens][LANES * EPL];
  const int lane = threadIdx.x & 63, sub = lane & (LANES - 1);
  const int slot = threadIdx.x / LANES;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens + slot;
  const bool live = t0 < a.T;
  const int64_t t = live ? t0 : a.T - 1;  // (a token past the end repeats the last one and stores nothing)
  const int e0 = sub * EPL;
  float z[EPL];
  double s[EPL];
  uint64_t key[EPL];
  load_logits(a, t, e0, z);
  scores<LANES, EPL>(a.score, z, s);
  if (all && live) {
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (e0 + j < a.E) all[t * a.E + e0 + j] = (float)s[j];
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    key[j] = e0 + j < a.E ? key_of(s[j] + (a.bias ? (double)a.bias[e0 + j] : 0.0)) : 0;
  if (a.groups > 1 && a.top_groups < a.groups) {
    const int n = a.E / a.groups;
#pragma unroll
    for (int j = 0; j < EPL; ++j) sk[slot][e0 + j] = key[j];
    __syncthreads();
    // lane g < G ranks group g (LANES >= G, or a lane takes several)
    uint64_t kept = 0;
    uint64_t best[kGateMaxGroups / LANES > 0 ? kGateMaxGroups / LANES : 1];
    constexpr int kPer = sizeof(best) / sizeof(best[0]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = sub * kPer + i;
      uint64_t k1 = 0, k2 = 0;
      if (g < a.groups)
        for (int e = 0; e < n; ++e) {
          const uint64_t v = sk[slot][g * n + e];
          k2 = v > k1 ? k1 : (v > k2 ? v : k2);
          k1 = v > k1 ? v : k1;
        }
      best[i] = g >= a.groups ? 0 : (a.group_top == 1 || n == 1 ? k1 : key_of(value_of(k1) + value_of(k2)));
    }
    for (int r = 0; r < a.top_groups; ++r) {
      uint64_t m = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) m = best[i] > m ? best[i] : m;
      const uint64_t top = lanes_max<LANES>(m);
      const int from = first_lane<LANES>(m == top, lane);
      int g = 0;
#pragma unroll
      for (int i = kPer - 1; i >= 0; --i) g = best[i] == top ? i : g;
      if (sub == from) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) best[i] = i == g ? 0 : best[i];
      }
      kept |= 1ull << __shfl(sub * kPer + g, (lane & ~(LANES - 1)) + from);
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (e0 + j < a.E && !(kept >> ((e0 + j) / n) & 1)) key[j] = 0;
  }
  // k rounds; lane j keeps the j-th expert and its score
  int my_e = 0;
  double my_s = 0;
  for (int r = 0; r < a.k; ++r) {
    uint64_t m = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) m = key[j] > m ? key[j] : m;
    const uint64_t top = lanes_max<LANES>(m);
    const int from = first_lane<LANES>(m == top, lane);
    int at = 0;
#pragma unroll
    for (int j = EPL - 1; j >= 0; --j) at = key[j] == top ? j : at;
    double sv = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      sv = j == at ? s[j] : sv;
      if (sub == from && j == at) key[j] = 0;
    }
    const int src = (lane & ~(LANES - 1)) + from;
    const int e = __shfl(e0 + at, src);
    sv = __shfl(sv, src);
    if (sub == r) {
      my_e = e;
      my_s = sv;
    }
  }
  if (sub >= a.k) my_s = 0;
  const double total = lanes_sum<LANES>(my_s) + kEps;
  if (live && sub < a.k) {
    idx[t * a.k + sub] = my_e;
    w[t * a.k + sub] = (float)((a.renormalize ? my_s / total : my_s) * (double)a.scale);
  }
}

// Gradient of the logits; gs null: no gradient of the scores.
template <int LANES, int EPL, int WAVES, int DT>
__global__ __launch_bounds__(64 * WAVES) void k_gate_bwd(GateArgs a, const int64_t* __restrict__ idx,
                                                         const float* __restrict__ gw, const float* __restrict__ gs,
                                                         void* __restrict__ dz) {
  constexpr int kTokens = 64 / LANES * WAVES;
  const int lane = threadIdx.x & 63, sub = lane & (LANES - 1);
  const int64_t t0 = (int64_t)blockIdx.x * kTokens + threadIdx.x / LANES;
  const bool live = t0 < a.T;
  const int64_t t = live ? t0 : a.T - 1;
  const int e0 = sub * EPL;
  float z[EPL], s[EPL], ds[EPL];
  load_logits(a, t, e0, z);
  scores<LANES, EPL>(a.score, z, s);
#pragma unroll
  for (int j = 0; j < EPL; ++j) ds[j] = gs && e0 + j < a.E ? gs[t * a.E + e0 + j] : 0.0f;
  if (gw) {
    // lane j of the token: the chosen expert j, its weight's gradient and its score
    const int my_e = sub < a.k ? (int)idx[t * a.k + sub] : -1;
    const float g = sub < a.k ? gw[t * a.k + sub] * a.scale : 0.0f;
    float my_s = 0.0f;
    for (int r = 0; r < a.k; ++r) {
      const int e = __shfl(my_e, (lane & ~(LANES - 1)) + r);
      float v = 0.0f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) v = e0 + j == e ? s[j] : v;
      const float got = __shfl(v, (lane & ~(LANES - 1)) + e / EPL);
      if (sub == r) my_s = got;
    }
    float d = g;
    if (a.renormalize) {
      const float total = lanes_sum<LANES>(my_s) + (float)kEps;
      d = (g - lanes_sum<LANES>(g * my_s) / total) / total;
    }
    for (int r = 0; r < a.k; ++r) {
      const int e = __shfl(my_e, (lane & ~(LANES - 1)) + r);
      const float v = __shfl(d, (lane & ~(LANES - 1)) + r);
#pragma unroll
      for (int j = 0; j < EPL; ++j) ds[j] += e0 + j == e ? v : 0.0f;
    }
  }
  if (a.score == kSoftmax) {
    float u = 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) u += e0 + j < a.E ? ds[j] * s[j] : 0.0f;
    u = lanes_sum<LANES>(u);
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] = s[j] * (ds[j] - u);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] = ds[j] * s[j] * (1.0f - s[j]);
  }
  if (!live) return;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    if (e0 + j >= a.E) continue;
    const int64_t at = t * a.E + e0 + j;
    if constexpr (DT == CIN_DT_F32)
      static_cast<float*>(dz)[at] = ds[j];
    else
      static_cast<uint16_t*>(dz)[at] = (uint16_t)f32_to_half_bits(DT, ds[j]);
  }
}

// launch(lanes, experts a lane, waves a workgroup)
template <class F>
void with_experts(int E, F launch) {
  using std::integral_constant;
  if (E <= 64)
    launch(integral_constant<int, 64>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (E <= 256)
    launch(integral_constant<int, 64>{}, integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (E <= 1024)
    launch(integral_constant<int, 64>{}, integral_constant<int, 16>{}, integral_constant<int, 2>{});
  else
    launch(integral_constant<int, 64>{}, integral_constant<int, 64>{}, integral_constant<int, 1>{});
}

int gate_args(const char* name, GateArgs& a, const void* logits, int dtype, int64_t ldl, const float* bias, int64_t T,
              int64_t E, int64_t k, int score, int64_t groups, int64_t top_groups, int group_top, int renormalize,
              float scale) {
  CIN_CHECK_ARG(dtype == CIN_DT_BF16 || dtype == CIN_DT_F32 || dtype == CIN_DT_F16, "%s: bad dtype %d", name, dtype);
  CIN_CHECK_ARG(T >= 0 && T < ((int64_t)1 << 31), "%s: T must be in [0, 2^31)", name);
  CIN_CHECK_ARG(E >= 1 && E <= kGateMaxExperts, "%s: 1 to %d experts", name, kGateMaxExperts);
  CIN_CHECK_ARG(k >= 1 && k <= kGateMaxTopK, "%s: top-k of 1 to %d", name, kGateMaxTopK);
  CIN_CHECK_ARG(score == kSigmoid || score == kSoftmax, "%s: bad score function %d", name, score);
  CIN_CHECK_ARG(groups >= 1 && groups <= kGateMaxGroups && E % groups == 0,
                "%s: 1 to %d groups that divide the experts", name, kGateMaxGroups);
  CIN_CHECK_ARG(top_groups >= 1 && top_groups <= groups, "%s: top_groups must be in [1, groups]", name);
  CIN_CHECK_ARG(k <= top_groups * (E / groups), "%s: the kept groups hold fewer than k experts", name);
  CIN_CHECK_ARG(group_top == 1 || group_top == 2, "%s: group_top must be 1 or 2", name);
  CIN_CHECK_ARG(ldl >= E, "%s: logits rows overlap", name);
  CIN_CHECK_ARG(T == 0 || logits, "%s: null pointer", name);
  a = GateArgs{logits, dtype, ldl, bias, T, (int)E, (int)k, score, (int)groups, (int)top_groups, group_top, renormalize, scale};
  return CIN_OK;
}

}  // namespace

extern "C" {

int cin_moe_gate(const void* logits, int dtype, int64_t ldl, const float* bias, int64_t T, int64_t E, int64_t k,
                 int score, int64_t groups, int64_t top_groups, int group_top, int renormalize, float scale,
                 int64_t* idx, float* weights, float* scores_out, void* stream) {
  GateArgs a;
  if (int rc = gate_args("moe_gate", a, logits, dtype, ldl, bias, T, E, k, score, groups, top_groups, group_top,
                         renormalize, scale))
    return rc;
  if (T == 0) return CIN_OK;
  CIN_CHECK_ARG(idx && weights, "moe_gate: null pointer");
  with_experts((int)E, [&](auto lanes, auto epl, auto waves) {
    constexpr int kTokens = 64 / lanes() * waves();
    hipLaunchKernelGGL((k_gate_fwd<lanes(), epl(), waves()>), (unsigned)cdiv(T, kTokens), 64 * waves(), 0,
                       static_cast<hipStream_t>(stream), a, idx, weights, scores_out);
  });
  return cin_check_launch("moe_gate");
}

int cin_moe_gate_backward(const void* logits, int dtype, int64_t ldl, int64_t T, int64_t E, int64_t k, int score,
                          int renormalize, float scale, const int64_t* idx, const float* gweights,
                          const float* gscores, void* dlogits, void* stream) {
  GateArgs a;
  if (int rc = gate_args("moe_gate_backward", a, logits, dtype, ldl, nullptr, T, E, k, score, 1, 1, 1, renormalize, scale))
    return rc;
  if (T == 0) return CIN_OK;
  CIN_CHECK_ARG(idx && dlogits, "moe_gate_backward: null pointer");
  with_experts((int)E, [&](auto lanes, auto epl, auto waves) {
    constexpr int kTokens = 64 / lanes() * waves();
    auto go = [&](auto dt) {
      hipLaunchKernelGGL((k_gate_bwd<lanes(), epl(), waves(), dt()>), (unsigned)cdiv(T, kTokens), 64 * waves(), 0,
                         static_cast<hipStream_t>(stream), a, idx, gweights, gscores, dlogits);
    };
    if (dtype == CIN_DT_F32)
      go(std::integral_constant<int, CIN_DT_F32>{});
    else if (dtype == CIN_DT_F16)
      go(std::integral_constant<int, CIN_DT_F16>{});
    else
      go(std::integral_constant<int, CIN_DT_BF16>{});
  });
  return cin_check_launch("moe_gate_backward");
}

}  // extern "C"
