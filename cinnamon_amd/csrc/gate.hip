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
// without the differences that cancel: s (1 - s) = t / (1 + t)^2 with t = e^-|z|, a softmax's ds less one
// of them, and the weights' term is scale * (1e-9 gw_j + sum_i (gw_j - gw_i) s[idx_i]) / total^2.
//
// Choices are ordered as they compare in 64 bits: neighbours in the order may differ by less than
// 32 bits hold.  A token is first ranked in 32 bits; where every difference that decides exceeds
// the error bound (or is one of equal logits and biases, a true tie), that is the order.  Where the
// chosen experts are sure and their order is not, they are sorted by their choices in 64 bits; else the
// wave ranks the token again in 64 bits (256 experts with biases in 8 groups, top-8, random logits: the
// order is in doubt in 1.3 tokens of a thousand, the choice in 0.2).  NaN counts as the greatest value,
// in a row and among groups.
//
// A token's experts lie over LANES lanes, EPL consecutive ones a lane, so that the order of the
// lanes is the order of the indices: the lowest of equal candidates is the first lane of a ballot.
// Up to 256 experts a token takes 16 lanes (a DPP row): maxima and sums need no LDS, and the rounds
// of the top k serve four tokens at once.  65536 tokens, 256 bf16 logits in 8 groups of which 4 stay,
// top-8, all scores out: 56 us, 1.9 TB/s, of which about 14 are the few waves that rank again in 64 bits
// (they end last); bound by VALU issue (1600 instructions a wave).  A wave per token with 64-bit keys
// throughout took 188 us.  The gradient, 23 us, 5.8 TB/s, is bound by HBM.
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
__device__ inline uint32_t key_of(float v) {  // (not for NaN)
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b >> 31 ? ~b : b | (1u << 31);
}
__device__ inline float value_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & ~(1u << 31) : ~k); }

template <int CTRL>
__device__ inline uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
// f over the token's lanes, every lane getting the result: within a DPP row by quad permutations,
// a half mirror and a mirror, across rows by swaps through LDS.
template <int LANES, class F>
__device__ inline uint32_t over_lanes(uint32_t v, F f) {
  static_assert(LANES == 16 || LANES == 64, "a DPP row or a wave");
  v = f(v, moved<0xB1>(v));
  v = f(v, moved<0x4E>(v));
  v = f(v, moved<0x141>(v));
  v = f(v, moved<0x140>(v));
  if constexpr (LANES == 64) {
    v = f(v, (uint32_t)__shfl_xor((int)v, 16));
    v = f(v, (uint32_t)__shfl_xor((int)v, 32));
  }
  return v;
}
template <int LANES>
__device__ inline uint32_t lanes_max(uint32_t v) {
  return over_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int LANES>
__device__ inline float lanes_sum(float v) {
  return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
// the maximum, NaN where there is one
template <int LANES>
__device__ inline float lanes_max_nan(float v) {
  return __uint_as_float(over_lanes<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    const float x = __uint_as_float(a), y = __uint_as_float(b);
    return y > x || y != y ? b : a;
  }));
}
template <int LANES>
__device__ inline uint64_t lanes_max(uint64_t v) {
  const uint32_t mine = (uint32_t)(v >> 32), hi = lanes_max<LANES>(mine);
  return (uint64_t)hi << 32 | lanes_max<LANES>(mine == hi ? (uint32_t)v : 0u);
}
template <int LANES>
__device__ inline double lanes_sum(double v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// Whether this lane is the first of its token for which `mine` holds.
template <int LANES>
__device__ inline bool is_first(bool mine, int lane) {
  const uint64_t m = __ballot(mine);
  if constexpr (LANES == 64) return lane == (int)__builtin_ctzll(m | (1ull << 63));
  const uint32_t w = lane & 32 ? (uint32_t)(m >> 32) : (uint32_t)m;
  const uint32_t row = (w >> (lane & 16)) & 0xffffu;
  return (lane & 15) == __builtin_ctz(row | 0x10000u);
}
// Whether `mine` holds on any lane of the token.
template <int LANES>
__device__ inline bool any_lane(bool mine, int lane) {
  const uint64_t m = __ballot(mine);
  if constexpr (LANES == 64) return m != 0;
  const uint32_t w = lane & 32 ? (uint32_t)(m >> 32) : (uint32_t)m;
  return ((w >> (lane & 16)) & 0xffffu) != 0;
}

// LDS written by lanes of a wave and read by others of the same wave: accesses of one wave are
// carried out in order, so only the compiler has to keep them so.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// EPL neighbours from any element's address, `other` past n.
template <int DT, int EPL>
__device__ __forceinline__ void load_row(const void* p, int64_t row, int e0, int n, float other, float (&v)[EPL]) {
  constexpr int es = DT == CIN_DT_F32 ? 4 : 2;
  const uint8_t* q = static_cast<const uint8_t*>(p) + (row + e0) * es;
  if (e0 + EPL <= n) {
    if constexpr (DT == CIN_DT_F32) {
      __builtin_memcpy(v, q, 4 * EPL);
    } else {
      uint16_t h[EPL];
      __builtin_memcpy(h, q, 2 * EPL);
#pragma unroll
      for (int j = 0; j < EPL; ++j) v[j] = half_bits_to_f32(DT, h[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) v[j] = e0 + j < n ? load_elem(q, DT, j) : other;
  }
}

// 1 / (1 + e^-z) and e^d in 32 bits within 8 roundings, below 1e-37 in absolute terms; NaN stays.  The
// exponential's argument is formed in two parts, as a rounded one is off by |d| of its last bits.
__device__ inline float exp_of(float d) {
  d = d > 88.7f ? 88.7f : d;
  d = d < -104.0f ? -104.0f : d;
  const float t = d * 1.44269504f, lo = __builtin_fmaf(d, 1.44269504f, -t) + d * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, lo * 0.693147182f, e);
}
__device__ inline float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-z)); }

// Scores of the token's experts; z holds -inf past E.  top: an upper bound of them (softmax).
template <int LANES, int EPL>
__device__ inline void scores(int kind, const float (&z)[EPL], float (&s)[EPL], float& top, float& zmax, float& inv) {
  top = 1.0f;
  zmax = 0.0f;
  inv = 1.0f;
  if (kind == kSigmoid) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] = sigmoid_of(z[j]);
  } else {
    float m = z[0], t = 0.0f;
#pragma unroll
    for (int j = 1; j < EPL; ++j) m = z[j] > m || z[j] != z[j] ? z[j] : m;
    m = lanes_max_nan<LANES>(m);
#pragma unroll
    for (int j = 0; j < EPL; ++j) t += s[j] = exp_of(z[j] - m);
    t = lanes_sum<LANES>(t);
    top = inv = 1.0f / t;
    zmax = m;
#pragma unroll
    for (int j = 0; j < EPL; ++j) s[j] *= inv;
  }
}
// Groups that stay, as a mask: lanes share a group's keys, `part` of `parts` each.  `margin` gets
// the difference between the last group that stays, `worst`, and the first that does not; where that is 0,
// `gap` the least difference between `worst` and a group, staying or not, that is not equal to it.
template <int LANES, class K, class F>
__device__ inline uint64_t keep_groups(const GateArgs& a, const K* keys, int lane, F& margin, F& worst, F& gap) {
  constexpr int kPer = kGateMaxGroups / LANES;  // groups of a lane
  const int sub = lane & (LANES - 1), n = a.E / a.groups;
  K best[kPer], all[kPer];
  // (differences are not negative: as integers they compare the same)
  const auto least_gap = [&] {
    gap = 0;
    if (!__ballot(margin == 0)) return;
    K far = 0;  // the complement of the least
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      F d = value_of(all[i]) - worst;
      d = d < 0 ? -d : d;
      if (sub + i * LANES < a.groups && d != 0) {
        const K c = ~__builtin_bit_cast(K, d);
        far = c > far ? c : far;
      }
    }
    far = lanes_max<LANES>(far);
    gap = far ? __builtin_bit_cast(F, (K)~far) : (F)__builtin_inff();
  };
#pragma unroll
  for (int i = 0; i < kPer; ++i) best[i] = 0;
  if (2 * a.groups <= LANES) {
    // 2, 4 or 8 lanes a group
    int parts = 2;
    while (2 * parts * a.groups <= LANES && parts < 8) parts *= 2;
    const int g = sub / parts, part = sub % parts;
    K k1 = 0, k2 = 0;
    if (g < a.groups)
      for (int e = part; e < n; e += parts) {
        const K v = keys[g * n + e];
        k2 = v > k1 ? k1 : (v > k2 ? v : k2);
        k1 = v > k1 ? v : k1;
      }
    for (int o = 1; o < parts; o <<= 1) {
      const K o1 = __shfl_xor(k1, o), o2 = __shfl_xor(k2, o);
      const K lo = k1 < o1 ? k1 : o1, hi2 = k2 > o2 ? k2 : o2;
      k1 = k1 > o1 ? k1 : o1;
      k2 = lo > hi2 ? lo : hi2;
    }
    // group sub's result to lane sub
    const int from = (lane & ~(LANES - 1)) + (sub * parts) % LANES;
    k1 = __shfl(k1, from);
    k2 = __shfl(k2, from);
    if (sub < a.groups) best[0] = a.group_top == 1 || n == 1 ? k1 : key_of(value_of(k1) + value_of(k2));
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = sub + i * LANES;
      K k1 = 0, k2 = 0;
      if (g < a.groups)
        for (int e = 0; e < n; ++e) {
          const K v = keys[g * n + e];
          k2 = v > k1 ? k1 : (v > k2 ? v : k2);
          k1 = v > k1 ? v : k1;
        }
      best[i] = g >= a.groups ? 0 : (a.group_top == 1 || n == 1 ? k1 : key_of(value_of(k1) + value_of(k2)));
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) all[i] = best[i];
  uint64_t kept = 0;
  K last = 0;
  if (a.groups <= LANES) {  // a group a lane
    for (int r = 0; r < a.top_groups; ++r) {
      last = lanes_max<LANES>(best[0]);
      const bool mine = is_first<LANES>(best[0] == last, lane);
      uint64_t m = __ballot(mine);
      if constexpr (LANES < 64) m = (m >> (lane & ~(LANES - 1))) & ((1ull << LANES) - 1);
      kept |= m;
      if (mine) best[0] = 0;
    }
    worst = value_of(last);
    margin = worst - value_of(lanes_max<LANES>(best[0]));
    least_gap();
    return kept;
  }
  for (int r = 0; r <= a.top_groups; ++r) {
    // the best group left, the lowest of equals: lane sub holds groups sub, sub + LANES, ..
    K m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) m = best[i] > m ? best[i] : m;
    const K top = lanes_max<LANES>(m);
    if (r == a.top_groups) {
      worst = value_of(last);
      margin = worst - value_of(top);
      break;
    }
    last = top;
    bool done = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      uint64_t mine = __ballot(!done && best[i] == top);
      if constexpr (LANES < 64) mine = (mine >> (lane & ~(LANES - 1))) & ((1ull << LANES) - 1);
      if (mine && !done) {
        const int at = (int)__builtin_ctzll(mine);
        kept |= 1ull << (at + i * LANES);
        if (sub == at) best[i] = 0;
        done = true;
      }
    }
  }
  least_gap();
  return kept;
}

// Keys with the place in the lane in their lowest bits, the first place largest: neighbours closer
// than EPL steps of a key count as equal from here on (an equal key's first place comes first).
template <int EPL>
constexpr uint32_t kPlace = EPL - 1;

// Bitonic sort of a lane's keys, the largest first.
template <int EPL>
__device__ inline void sort_keys(uint32_t (&key)[EPL]) {
#pragma unroll
  for (int size = 2; size <= EPL; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2)
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int o = i ^ step;
        if (o < i) continue;
        const uint32_t hi = key[i] > key[o] ? key[i] : key[o], lo = key[i] > key[o] ? key[o] : key[i];
        const bool down = (i & size) == 0 || size == EPL;
        key[i] = down ? hi : lo;
        key[o] = down ? lo : hi;
      }
}

// The k largest keys, the lowest index of equals: lane r's key, and the expert in chosen[r].  Each
// lane's keys are sorted once, so that a round is one maximum over the lanes' first keys and a shift in
// the lane that had it; keys left stay sorted.
template <int LANES, int EPL>
__device__ inline uint32_t top_k(int k, int lane, uint32_t (&key)[EPL], int* chosen) {
  const int sub = lane & (LANES - 1);
  sort_keys(key);
  uint32_t mine = 0;
  for (int r = 0; r < k; ++r) {
    const uint32_t head = key[0] & ~kPlace<EPL>;
    const uint32_t top = lanes_max<LANES>(head);
    mine = sub == r ? top : mine;
    if (is_first<LANES>(head == top, lane)) {
      chosen[r] = sub * EPL + (int)(kPlace<EPL> - (key[0] & kPlace<EPL>));
#pragma unroll
      for (int j = 0; j + 1 < EPL; ++j) key[j] = key[j + 1];
      key[EPL - 1] = 0;
    }
  }
  wave_sync();
  return mine;
}

// Token t's ranking in 64 bits by the whole wave, its keys in LDS: lane r < k gets the r-th expert
// and its score.
template <int DT>
__device__ inline void rank64(const GateArgs& a, int64_t t, int lane, uint64_t* keys, int& my_e, double& my_s) {
  const int64_t row = t * a.ldl;
  double m = -__builtin_inf(), total = 0;
  if (a.score == kSoftmax) {
    for (int e = lane; e < a.E; e += 64) {
      const double z = load_elem(a.logits, DT, row + e);
      m = z > m || z != z ? z : m;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_xor(m, o);
      m = u > m || u != u ? u : m;
    }
    for (int e = lane; e < a.E; e += 64) total += exp((double)load_elem(a.logits, DT, row + e) - m);
    total = lanes_sum<64>(total);
  }
  const auto score = [&](int e) {
    const double z = load_elem(a.logits, DT, row + e);
    return a.score == kSoftmax ? exp(z - m) / total : 1 / (1 + exp(-z));
  };
  wave_sync();
  for (int e = lane; e < a.E; e += 64) keys[e] = key_of(score(e) + (a.bias ? (double)a.bias[e] : 0.0));
  wave_sync();
  if (a.top_groups < a.groups) {
    double margin, worst, gap;
    const uint64_t kept = keep_groups<64, uint64_t, double>(a, keys, lane, margin, worst, gap);
    const int n = a.E / a.groups;
    wave_sync();
    for (int e = lane; e < a.E; e += 64)
      if (!(kept >> (e / n) & 1)) keys[e] = 0;
    wave_sync();
  }
  my_e = 0;
  for (int r = 0; r < a.k; ++r) {
    uint64_t best = 0;
    int at = 0;  // the lane's first expert with it
    for (int e = lane; e < a.E; e += 64) {
      const uint64_t v = keys[e];
      at = v > best ? e : at;
      best = v > best ? v : best;
    }
    const uint64_t top = lanes_max<64>(best);
    // (the lowest expert: the largest complement)
    const int e = (int)~lanes_max<64>(~(uint32_t)(best == top ? at : a.E));
    if (lane == r) my_e = e;
    if (lane == 0) keys[e] = 0;
    wave_sync();
  }
  my_s = lane < a.k ? score(my_e) : 0.0;
}

template <int LANES, int EPL, int WAVES, int DT>
__global__ __launch_bounds__(64 * WAVES, EPL <= 16 ? 4 : 1) void k_gate_fwd(GateArgs a, int64_t* __restrict__ idx,
                                                                               float* __restrict__ w,
                                                                               float* __restrict__ all) {
  constexpr int kTokens = 64 / LANES * WAVES;
  __shared__ uint64_t keys64[WAVES][LANES * EPL];   // of the token a wave ranks in 64 bits
  __shared__ uint32_t keys32[kTokens][LANES * EPL];
  __shared__ int chosen[kTokens][kGateMaxTopK];
  const int lane = threadIdx.x & 63, sub = lane & (LANES - 1);
  const int slot = threadIdx.x / LANES;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens + slot;
  const bool live = t0 < a.T;
  const int64_t t = live ? t0 : a.T - 1;  // (a token past the end repeats the last one and stores nothing)
  const int e0 = sub * EPL;
  const bool limited = a.top_groups < a.groups;
  float z[EPL], b[EPL], s[EPL];
  load_row<DT, EPL>(a.logits, t * a.ldl, e0, a.E, -__builtin_inff(), z);
  if (a.bias) {
    load_row<CIN_DT_F32, EPL>(a.bias, 0, e0, a.E, 0.0f, b);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) b[j] = 0.0f;
  }
  float top, zmax, inv;
  scores<LANES, EPL>(a.score, z, s, top, zmax, inv);
  if (all && live) {
    float* q = all + t * a.E + e0;
    if (e0 + EPL <= a.E) {
      __builtin_memcpy(q, s, 4 * EPL);
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (e0 + j < a.E) q[j] = s[j];
    }
  }
  // Without a bias, and with groups that count by one expert, the logits order as the choices do:
  // exactly, but where 64 bits cannot tell two scores apart (neighbours closer than 1e-10, sigmoids
  // above 10, scores under e^-600).  Else in 32 bits, u = 2^-24: a score is off by less than 8 u of
  // itself (a softmax's by 6 + EPL u more, its sum's), a choice by its rounding too, and ranked keys by
  // 2 EPL u (that of a 16-bit logit by nothing: those bits are 0).
  const bool direct = !a.bias && (!limited || a.group_top == 1);
  constexpr float kU = 5.9604644775390625e-8f, kC = (2 + 2 * EPL) * kU;
  const float kS = (a.score == kSoftmax ? 28 + 2 * EPL : 16) * kU;
  constexpr float kZ = DT == CIN_DT_F32 ? 2 * EPL * kU : 0.0f;
  const auto bound = [&](float c) {
    return direct ? 1e-10f + kZ * fabsf(c) : kS * (a.bias ? top : fabsf(c)) + kC * fabsf(c);
  };
  const auto blurred = [&](float c) { return direct && !(c - zmax > -600.0f && (a.score == kSoftmax || c < 10.0f)); };
  uint32_t key[EPL];
  bool doubt = false;
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const float c = direct ? z[j] : s[j] + b[j];
    key[j] = key_of(c);
    const bool there = e0 + EPL <= a.E || e0 + j < a.E;
    doubt |= there && !(c < __builtin_inff());  // NaN or infinite
    most = fmaxf(most, there ? fabsf(c) : 0.0f);
  }
  if (e0 + EPL > a.E) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) key[j] = e0 + j < a.E ? key[j] : 0;
  }
  if (limited) {
    uint32_t* keys = keys32[slot];
#pragma unroll
    for (int j = 0; j < EPL; ++j) keys[e0 + j] = key[j];
    wave_sync();
    float margin, worst, gap;
    const uint64_t kept = keep_groups<LANES, uint32_t, float>(a, keys, lane, margin, worst, gap);
    const int n = a.E / a.groups;
    int g = e0 / n;  // the group of e0 + j
    if (n % EPL == 0) {  // a lane's experts are of one group
      const bool stays = kept >> (g & 63) & 1;
#pragma unroll
      for (int j = 0; j < EPL; ++j) key[j] = stays ? key[j] : 0;
    } else {
      int left = n - (e0 - g * n);  // its experts from e0 + j on
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        if (!(kept >> (g & 63) & 1)) key[j] = 0;
        if (--left == 0) {
          ++g;
          left = n;
        }
      }
    }
    // two choices of up to `most` each on either side
    most = __uint_as_float(lanes_max<LANES>(__float_as_uint(most)));
    // (equal logits are a true tie, but not where others that 64 bits may not tell from them are near)
    const float sure = 2 * bound(most) + 8 * kU * most;
    doubt |= !(margin > sure || (direct && margin == 0.0f && gap > sure)) || blurred(worst);
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) key[j] = key[j] ? (key[j] & ~kPlace<EPL>) | (kPlace<EPL> - j) : 0;
  // lane r < k: the r-th expert, its choice, logit and bias (the lanes from k on as lane k - 1)
  float my_c = value_of(top_k<LANES, EPL>(a.k, lane, key, chosen[slot]));
  const int first = lane & ~(LANES - 1), last = first + a.k - 1;
  int my_e = chosen[slot][sub < a.k ? sub : a.k - 1];
  const auto z_of = [&](int e) { return load_elem(a.logits, DT, t * a.ldl + e); };
  const float my_z = z_of(my_e), my_b = a.bias ? a.bias[my_e] : 0.0f;
  float my_s = a.score == kSigmoid ? sigmoid_of(my_z) : exp_of(my_z - zmax) * inv;
  // in doubt: neighbours in the order that are near and no true tie, an expert not taken that is
  // near the last one taken, and scores that 32 bits hardly hold
  const int up = sub > 0 ? lane - 1 : lane;
  const float c1 = __shfl(my_c, up), z1 = __shfl(my_z, up), b1 = __shfl(my_b, up);
  const bool order = sub > 0 && sub < a.k && !(c1 - my_c > bound(fmaxf(fabsf(c1), fabsf(my_c)))) && !(z1 == my_z && b1 == my_b);
  doubt |= sub < a.k && (my_s < 1e-30f || !(fabsf(my_c) < __builtin_inff()) || blurred(my_c));
  const float cl = __shfl(my_c, last), zl = __shfl(my_z, last), bl = __shfl(my_b, last), least = cl - bound(cl);
  // (a key is 0 for an expert taken or left out: below that of any choice)
  const uint32_t near = least < __builtin_inff() ? key_of(least) & ~kPlace<EPL> : 1u;
  bool tied = false;  // an expert not taken that equals the last one taken
  if (key[0] >= near) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (key[j] < near || key[j] == 0) break;
      const int e = e0 + (int)(kPlace<EPL> - (key[j] & kPlace<EPL>));
      const bool same = z_of(e) == zl && (a.bias ? a.bias[e] : 0.0f) == bl;
      tied |= same;
      doubt |= !same;
    }
  }
  if (__ballot(order)) {
    if (a.score == kSigmoid) {
      // The experts taken are those, in another order perhaps: sorted by their choices in 64 bits.  (But
      // where one taken before the last may be less than the last, so may it be than the last one's equals.)
      doubt |= any_lane<LANES>(tied, lane) && order;
      double c = 1 / (1 + exp(-(double)my_z)) + (double)my_b;
      for (int pass = 0; pass < a.k; ++pass) {
        const int p = (sub ^ (pass & 1)) & 1 ? sub - 1 : sub + 1;  // odd and even neighbours in turn
        const bool pair = p >= 0 && p < a.k && sub < a.k;
        const double pc = __shfl(c, first + (pair ? p : sub));
        const int pe = __shfl(my_e, first + (pair ? p : sub));
        const bool ahead = c > pc || (c == pc && my_e < pe);
        if (pair && (sub < p) != ahead) {
          c = pc;
          my_e = pe;
        }
      }
      my_s = sigmoid_of(z_of(my_e));
    } else {
      doubt |= order;
    }
  }
  const float total = lanes_sum<LANES>(sub < a.k ? my_s : 0.0f) + (float)kEps;
  float wt = (a.renormalize ? my_s / total : my_s) * a.scale;
  const uint64_t doubts = __ballot(doubt);
#pragma unroll 1
  for (int q = 0; q < 64 / LANES; ++q) {
    if (!(doubts >> (q * LANES) & (LANES == 64 ? ~0ull : (1ull << LANES % 64) - 1))) continue;  // the whole wave
    int e;
    double v;
    rank64<DT>(a, __shfl(t, q * LANES), lane, keys64[threadIdx.x >> 6], e, v);
    const double sum = lanes_sum<64>(v) + kEps;
    const float wv = (float)((a.renormalize ? v / sum : v) * (double)a.scale);
    const int e_r = __shfl(e, sub);
    const float w_r = __shfl(wv, sub);
    if (lane / LANES == q) {
      my_e = e_r;
      wt = w_r;
    }
  }
  if (live && sub < a.k) {
    idx[t * a.k + sub] = my_e;
    w[t * a.k + sub] = wt;
  }
}

// Gradient of the logits; gw or gs null: no gradient of the weights, of the scores.  The chosen
// experts' terms go to their places through LDS.
template <int LANES, int EPL, int WAVES, int DT>
__global__ __launch_bounds__(64 * WAVES) void k_gate_bwd(GateArgs a, const int64_t* __restrict__ idx,
                                                         const float* __restrict__ gw, const float* __restrict__ gs,
                                                         void* __restrict__ dz) {
  constexpr int kTokens = 64 / LANES * WAVES;
  __shared__ float place[kTokens][LANES * EPL];
  const int lane = threadIdx.x & 63, sub = lane & (LANES - 1);
  const int slot = threadIdx.x / LANES;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens + slot;
  const bool live = t0 < a.T;
  const int64_t t = live ? t0 : a.T - 1;
  const int e0 = sub * EPL;
  const bool mine = gw && sub < a.k;
  const int64_t e = mine ? idx[t * a.k + sub] : 0;
  const bool there = mine && e >= 0 && e < a.E;
  const float ze = there ? load_elem(a.logits, DT, t * a.ldl + e) : 0.0f;
  const float g = there ? gw[t * a.k + sub] : 0.0f;
  float z[EPL], s[EPL], ds[EPL];
  load_row<DT, EPL>(a.logits, t * a.ldl, e0, a.E, -__builtin_inff(), z);
  if (gs) {
    load_row<CIN_DT_F32, EPL>(gs, t * a.E, e0, a.E, 0.0f, ds);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] = 0.0f;
  }
  float top, zmax = 0.0f, inv = 1.0f;
  if (a.score == kSoftmax) {
    scores<LANES, EPL>(kSoftmax, z, s, top, zmax, inv);
  } else {  // s (1 - s)
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float t = exp_of(-fabsf(z[j])), r = __builtin_amdgcn_rcpf(1.0f + t);
      s[j] = t * r * r;
    }
  }
  if (gw) {
    const float se = there ? (a.score == kSigmoid ? sigmoid_of(ze) : exp_of(ze - zmax) * inv) : 0.0f;
    float d = g * a.scale;
    if (a.renormalize) {
      const float total = lanes_sum<LANES>(se) + (float)kEps;
      const int first = lane & ~(LANES - 1);
      d = (float)kEps * g;
      for (int i = 0; i < a.k; ++i) d += (g - __shfl(g, first + i)) * __shfl(se, first + i);
      d = d / total / total * a.scale;
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) place[slot][e0 + j] = 0.0f;
    wave_sync();
    if (there) place[slot][e] = d;
    wave_sync();
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] += place[slot][e0 + j];
  }
  if (a.score == kSoftmax) {
    // less the largest score's ds, which the sum of the scores, 1, leaves the same: its own term cancels
    float c = -__builtin_inff(), u = 0.0f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) c = z[j] == zmax ? fmaxf(c, ds[j]) : c;
    c = lanes_max_nan<LANES>(c);
#pragma unroll
    for (int j = 0; j < EPL; ++j) u += e0 + j < a.E ? (ds[j] - c) * s[j] : 0.0f;
    u = lanes_sum<LANES>(u);
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] = s[j] * (ds[j] - c - u);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) ds[j] *= s[j];
  }
  if (!live) return;
  constexpr int es = DT == CIN_DT_F32 ? 4 : 2;
  uint8_t* q = static_cast<uint8_t*>(dz) + (t * a.E + e0) * es;
  if (e0 + EPL <= a.E) {
    if constexpr (DT == CIN_DT_F32) {
      __builtin_memcpy(q, ds, 4 * EPL);
    } else {
      uint16_t h[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) h[j] = (uint16_t)f32_to_half_bits(DT, ds[j]);
      __builtin_memcpy(q, h, 2 * EPL);
    }
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      if (e0 + j >= a.E) continue;
      if constexpr (DT == CIN_DT_F32)
        reinterpret_cast<float*>(q)[j] = ds[j];
      else
        reinterpret_cast<uint16_t*>(q)[j] = (uint16_t)f32_to_half_bits(DT, ds[j]);
    }
  }
}

// launch(lanes, experts a lane, waves a workgroup, dtype)
template <class F>
void with_experts(int E, int dtype, F launch) {
  using std::integral_constant;
  auto go = [&](auto lanes, auto epl, auto waves) {
    if (dtype == CIN_DT_F32)
      launch(lanes, epl, waves, integral_constant<int, CIN_DT_F32>{});
    else if (dtype == CIN_DT_F16)
      launch(lanes, epl, waves, integral_constant<int, CIN_DT_F16>{});
    else
      launch(lanes, epl, waves, integral_constant<int, CIN_DT_BF16>{});
  };
  const integral_constant<int, 16> row{};
  const integral_constant<int, 64> wave{};
  const integral_constant<int, 4> four{};
  const integral_constant<int, 1> one{};
  if (E <= 16)
    go(row, integral_constant<int, 1>{}, four);
  else if (E <= 32)
    go(row, integral_constant<int, 2>{}, four);
  else if (E <= 64)
    go(row, integral_constant<int, 4>{}, four);
  else if (E <= 128)
    go(row, integral_constant<int, 8>{}, four);
  else if (E <= 256)
    go(row, integral_constant<int, 16>{}, four);
  else if (E <= 1024)
    go(wave, integral_constant<int, 16>{}, one);
  else
    go(wave, integral_constant<int, 64>{}, one);
}

int gate_args(const char* name, GateArgs& a, const void* logits, int dtype, int64_t ldl, const float* bias, int64_t T,
              int64_t E, int64_t k, int score, int64_t groups, int64_t top_groups, int group_top, int renormalize,
              float scale) {
  CIN_CHECK_ARG(dtype == CIN_DT_BF16 || dtype == CIN_DT_F32 || dtype == CIN_DT_F16, "%s: bad dtype %d", name, dtype);
  CIN_CHECK_ARG(T >= 0, "%s: negative size", name);
  CIN_CHECK_ARG(E >= 1 && E <= kGateMaxExperts, "%s: 1 to %d experts", name, kGateMaxExperts);
  // (a launch has fewer than 2^32 threads: 16 a token up to 256 experts, 64 above)
  CIN_CHECK_ARG(T <= ((int64_t)1 << (E <= 256 ? 28 : 26)) - 16, "%s: too many tokens", name);
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
  with_experts((int)E, dtype, [&](auto lanes, auto epl, auto waves, auto dt) {
    constexpr int kTokens = 64 / lanes() * waves();
    hipLaunchKernelGGL((k_gate_fwd<lanes(), epl(), waves(), dt()>), (unsigned)cdiv(T, kTokens), 64 * waves(), 0,
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
  with_experts((int)E, dtype, [&](auto lanes, auto epl, auto waves, auto dt) {
    constexpr int kTokens = 64 / lanes() * waves();
    hipLaunchKernelGGL((k_gate_bwd<lanes(), epl(), waves(), dt()>), (unsigned)cdiv(T, kTokens), 64 * waves(), 0,
                       static_cast<hipStream_t>(stream), a, idx, gweights, gscores, dlogits);
  });
  return cin_check_launch("moe_gate_backward");
}

}  // extern "C"
