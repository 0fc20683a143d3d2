// A whole mixture-of-experts layer for a few tokens on gfx950 (reference src/layers.py:113-157 at generation):
// router, gate, SwiGLU experts and a shared expert, weighted sum.
//
//   z_t = x_t R^T;  idx, wt = the gate of z (as csrc/gate.hip: scores, bias, groups, top k, weights)
//   h_tj = wt_tj silu(W1_e x_t) * (W2_e x_t)            e = idx_tj
//   out_t = sum_j W3_e h_tj  (+ the shared expert's, of weight 1)
//
// What it has to read is the chosen experts' weights, once; a few tokens' products are far below the matrix
// units' rate, so the weights (e4m3 codes with a scale a 128 x 128 block, or bf16) go from memory straight to
// registers, are widened there to bf16 (exact for codes) and multiplied by the tokens' bf16 parts on the
// 16 x 16 x 32 units, 16 weight rows by up to 16 tokens at a time.  The tokens of an expert are gathered, so
// that no column is wasted; a block's scale multiplies its fp32 sum.
//
// Rounding: x is split into bf16 parts that hold it exactly (one for bf16, two for fp16, three for fp32); h is
// split into two parts (2^-17 of a value; three, 2^-25, where the output is fp32), as one bf16 part would add an error as
// large as the output's own rounding.  All sums are fp32.  Logits and the gate are in 64 bits: choices next to
// the border of the top k differ by less than 32 bits hold.
//
// Four launches: k_router (logits by slices of D on the fp64 matrix units, and x's parts), k_gate (a workgroup a
// token), k_up (a workgroup an expert and 16 or 32 of its hidden channels, the waves sharing D), k_down (a workgroup
// 16 or 32 output channels, the waves sharing the chosen experts' hidden channels; each wave's sums per token
// lie in LDS and are joined in a fixed order).  No atomics on results.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "cin_common.h"
#include "cin_runtime.h"

using namespace cin;

namespace {

constexpr int kMaxTokens = 128;
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 16;
constexpr int kMaxGroups = 64;
constexpr int kBlock = 128;        // of a scale, and a step of K
constexpr int kMaxAssigned = kMaxTokens * kMaxTopK;
constexpr int kLeastUnit = 32;
constexpr int kMaxUnits = kMaxExperts + kMaxAssigned / kLeastUnit;
constexpr int kRouterSlice = 512;  // channels of a k_router workgroup
constexpr int kUpWaves = 4, kDownWaves = 8;

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef double d4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Parts of x and of h for an input type.
template <int DT>
constexpr int kXParts = DT == CIN_DT_BF16 ? 1 : DT == CIN_DT_F16 ? 2 : 3;
template <int DT>
constexpr int kHParts = DT == CIN_DT_F32 ? 3 : 2;
// Tokens of an expert multiplied at once: what the registers hold of their parts.
constexpr int unit_tokens(int dtype) { return dtype == CIN_DT_F32 ? kLeastUnit : 64; }

struct Expert {  // stacked experts, or a shared one
  const uint8_t *w12, *w3;
  const float *s12, *s3;  // null for bf16
  int H;
};

struct LayerArgs {
  const void* x;
  int64_t ldx;
  int T, D, Dp, E, k;
  const void* router;
  int router_dtype;
  int64_t ldr;
  const float* bias;
  int score, groups, top_groups, group_top, renormalize;
  float scale;
  Expert experts, shared;
  int64_t* idx;
  float* weights;
  void* out;
  // workspace
  double* logits;  // [slices, T, E]
  int slices;
  uint16_t *xb, *hb, *hs;  // parts of x [P, T, Dp], of h [P, T k, H], of the shared expert's [P, T, Hs]
  int units;               // the most that the routed experts can have
};

// ---------------------------------------------------------------------------------------------
// Router and gate
// ---------------------------------------------------------------------------------------------
// 8 elements of a row at any element's address.
__device__ __forceinline__ void load8(const void* p, int dt, int64_t i, float (&v)[8]) {
  if (dt == CIN_DT_F32) {
    __builtin_memcpy(v, static_cast<const float*>(p) + i, 32);
  } else {
    uint16_t h[8];
    __builtin_memcpy(h, static_cast<const uint16_t*>(p) + i, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = half_bits_to_f32(dt, h[e]);
  }
}

// bf16 parts of 8 values: each the rounding of what the ones before leave; an infinity or NaN has one.
template <int P>
__device__ __forceinline__ void split8(const float (&v)[8], u4 (&part)[P]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int p = 0; p < P; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = f32x2_to_bf16x2_bits(r[2 * i], r[2 * i + 1]);
      part[p][i] = w;
      if (p + 1 < P) {
        const float lo = bf16_lo(w), hi = bf16_hi(w);
        r[2 * i] = __builtin_isfinite(lo) ? r[2 * i] - lo : 0.0f;
        r[2 * i + 1] = __builtin_isfinite(hi) ? r[2 * i + 1] - hi : 0.0f;
      }
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void k_router(LayerArgs a) {
  __shared__ double lds[4][4][64];
  constexpr int P = kXParts<DT>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int etiles = (a.E + 15) / 16;
  const int slice = blockIdx.x / etiles, etile = blockIdx.x - slice * etiles;
  const int e = etile * 16 + (lane & 15), t = blockIdx.y * 16 + (lane & 15);
  d4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int s = 0; s < kRouterSlice / 4 / 32; ++s) {
    const int d = slice * kRouterSlice + wave * (kRouterSlice / 4) + s * 32 + (lane >> 4) * 8;
    float w[8] = {}, x[8] = {};
    if (d < a.D) {
      if (e < a.E) load8(a.router, a.router_dtype, e * a.ldr + d, w);
      if (t < a.T) load8(a.x, DT, t * a.ldx + d, x);
    }
    if (etile == 0 && t < a.T && d < a.Dp) {
      u4 part[P];
      split8<P>(x, part);
#pragma unroll
      for (int p = 0; p < P; ++p) *reinterpret_cast<u4*>(a.xb + ((int64_t)p * a.T + t) * a.Dp + d) = part[p];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)w[i], (double)x[i], acc, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) lds[wave][i][lane] = acc[i];
  __syncthreads();
  // register i of a lane is expert 4 i + lane / 16, token lane % 16; the waves' sums in order
  const int i = wave, er = etile * 16 + 4 * i + (lane >> 4);
  const double z = ((lds[0][i][lane] + lds[1][i][lane]) + lds[2][i][lane]) + lds[3][i][lane];
  if (er < a.E && t < a.T) a.logits[((int64_t)slice * a.T + t) * a.E + er] = z;
}

// Keys that order as the values do, NaN above all; 0 is below every key.
__device__ inline uint64_t order_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // -0 counts as 0
  if (v != v) return ~0ull;
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ inline double of_key(uint64_t k) {
  if (k == ~0ull) return __builtin_nan("");
  return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}

__device__ inline double block_reduce(double v, bool maximum, double* lds) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_xor(v, o);
    v = maximum ? (u > v || u != u ? u : v) : v + u;
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = lds[0];
  for (int w = 1; w < 4; ++w) r = maximum ? (lds[w] > r || lds[w] != lds[w] ? lds[w] : r) : r + lds[w];
  __syncthreads();
  return r;
}

__global__ __launch_bounds__(256) void k_gate(LayerArgs a) {
  __shared__ double score[kMaxExperts], reduce[4];
  __shared__ uint64_t key[kMaxExperts], group_key[kMaxGroups];
  __shared__ int chosen[kMaxTopK], kept[kMaxGroups];
  constexpr int kOwn = kMaxExperts / 256;
  const int t = blockIdx.x, tid = threadIdx.x;
  double z[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid + o * 256;
    z[o] = -__builtin_inf();
    if (e < a.E) {
      const double* p = a.logits + (int64_t)t * a.E + e;
      double s = p[0];
#pragma unroll 8
      for (int i = 1; i < a.slices; ++i) s += p[(int64_t)i * a.T * a.E];
      z[o] = s;
    }
  }
  if (a.score == 1) {
    double m = z[0];
#pragma unroll
    for (int o = 1; o < kOwn; ++o) m = z[o] > m || z[o] != z[o] ? z[o] : m;
    m = block_reduce(m, true, reduce);
    double sum = 0.0;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      z[o] = tid + o * 256 < a.E ? exp(z[o] - m) : 0.0;
      sum += z[o];
    }
    sum = block_reduce(sum, false, reduce);
#pragma unroll
    for (int o = 0; o < kOwn; ++o) z[o] /= sum;
  } else {
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      if (tid + o * 256 < a.E) {
        const double q = exp(-fabs(z[o]));
        z[o] = z[o] < 0 ? q / (1.0 + q) : 1.0 / (1.0 + q);
      }
    }
  }
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid + o * 256;
    if (e < a.E) {
      score[e] = z[o];
      key[e] = order_key(a.bias ? z[o] + (double)a.bias[e] : z[o]);
    }
  }
  __syncthreads();
  if (a.groups > 1) {
    const int n = a.E / a.groups;
    if (tid < a.groups) {
      uint64_t best = 0, second = 0;
      for (int i = 0; i < n; ++i) {
        const uint64_t k = key[tid * n + i];
        if (k > best) {
          second = best;
          best = k;
        } else if (k > second) {
          second = k;
        }
      }
      group_key[tid] = a.group_top == 2 && n > 1 ? order_key(of_key(best) + of_key(second)) : best;
    }
    __syncthreads();
    if (tid < a.groups) {
      int rank = 0;
      const uint64_t mine = group_key[tid];
      for (int j = 0; j < a.groups; ++j) rank += group_key[j] > mine || (group_key[j] == mine && j < tid);
      kept[tid] = rank < a.top_groups;
    }
    __syncthreads();
    for (int e = tid; e < a.E; e += 256)
      if (!kept[e / n]) key[e] = 0;
    __syncthreads();
  }
  // an expert's place is the number of experts in front of it
  uint64_t mine[kOwn];
  int rank[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid + o * 256;
    mine[o] = e < a.E ? key[e] : 0;
    rank[o] = 0;
  }
  const int own = (a.E + 255) / 256;
#pragma unroll 8
  for (int j = 0; j < a.E; ++j) {
    const uint64_t other = key[j];
    rank[0] += other > mine[0] || (other == mine[0] && j < tid);
    if (own > 1) {
#pragma unroll
      for (int o = 1; o < kOwn; ++o) rank[o] += other > mine[o] || (other == mine[o] && j < tid + o * 256);
    }
  }
#pragma unroll
  for (int o = 0; o < kOwn; ++o)
    if (tid + o * 256 < a.E && rank[o] < a.k) chosen[rank[o]] = tid + o * 256;
  __syncthreads();
  if (tid < a.k) {
    double total = 0.0;
    for (int j = 0; j < a.k; ++j) total += score[chosen[j]];
    const double s = score[chosen[tid]];
    a.idx[(int64_t)t * a.k + tid] = chosen[tid];
    a.weights[(int64_t)t * a.k + tid] = (float)((double)a.scale * (a.renormalize ? s / (total + 1e-9) : s));
  }
}

// ---------------------------------------------------------------------------------------------
// Which expert multiplies which tokens
// ---------------------------------------------------------------------------------------------
// The assignments (t k + j) by expert, in units of up to unit_tokens of one expert.
struct Plan {
  int count[kMaxExperts];           // assignments of an expert, then where its next one goes
  uint32_t unit[kMaxUnits];         // expert, first entry
  uint8_t tokens[kMaxUnits];
  uint16_t list[kMaxAssigned];
  uint32_t waves[kDownWaves];
  int units;
};

// ALL: units begin at their place in the list of all experts, which follows: an expert's in the atomics' order, as it
// only decides which column of a product a token has, but in increasing order where the expert has several units, whose
// steps are summed apart.  Else units begin at their place among their expert's assignments.
template <int THREADS, int UNIT, bool ALL>
__device__ __forceinline__ void make_plan(Plan& p, const int64_t* idx, int n, int E) {
  constexpr int kOwn = kMaxExperts / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e < E; e += THREADS) p.count[e] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += THREADS) atomicAdd(&p.count[(int)idx[i]], 1);
  __syncthreads();
  // units (upper half) and assignments of the experts before this thread's
  uint32_t own = 0;
  int c[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid * kOwn + o;
    c[o] = e < E ? p.count[e] : 0;
    own += (uint32_t)((c[o] + UNIT - 1) / UNIT) << 16 | (uint32_t)c[o];
  }
  uint32_t s = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)s, o);
    if (lane >= o) s += u;
  }
  if (lane == 63) p.waves[wave] = s;
  __syncthreads();
  uint32_t at = s - own, all = 0;
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) at += p.waves[w];
    all += p.waves[w];
  }
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid * kOwn + o;
    if (e < E) p.count[e] = (int)(at & 0xffffu);
    for (int i = 0; i < c[o]; i += UNIT) {
      p.unit[at >> 16] = (uint32_t)e << 16 | ((ALL ? at & 0xffffu : 0u) + i);
      p.tokens[at >> 16] = (uint8_t)min(c[o] - i, UNIT);
      at += 1u << 16;
    }
    at += (uint32_t)c[o];
  }
  if (tid == 0) p.units = (int)(all >> 16);
  __syncthreads();
  if constexpr (ALL) {
    for (int i = tid; i < n; i += THREADS) p.list[atomicAdd(&p.count[(int)idx[i]], 1)] = (uint16_t)i;
    __syncthreads();
    for (int u = wave; u + 1 < p.units; u += THREADS / 64) {
      const uint32_t e = p.unit[u] >> 16;
      if (p.unit[u + 1] >> 16 != e || (u > 0 && p.unit[u - 1] >> 16 == e)) continue;
      uint32_t to = p.unit[u] & 0xffffu;
      for (int i0 = 0; i0 < n; i0 += 64) {
        const bool mine = i0 + lane < n && (uint32_t)idx[i0 + lane] == e;
        const uint64_t m = __ballot(mine);
        if (mine) p.list[to + (uint32_t)__builtin_popcountll(m & ((1ull << lane) - 1))] = (uint16_t)(i0 + lane);
        to += (uint32_t)__builtin_popcountll(m);
      }
    }
    __syncthreads();
  }
}

// The list of one expert in increasing order: workgroups that take its units each find the same.
template <int THREADS>
__device__ __forceinline__ void list_of(Plan& p, const int64_t* idx, int n, int expert) {
  constexpr int kWaves = THREADS / 64, kOwn = kMaxAssigned / THREADS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int each = (n + kWaves * 64 - 1) / (kWaves * 64);  // 64 assignments a round, a wave's one behind the other
  uint64_t mine[kOwn];
  uint32_t found = 0;
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int i = (wave * each + o) * 64 + lane;
    mine[o] = __ballot(o < each && i < n && (int)idx[i < n ? i : 0] == expert);
    found += (uint32_t)__builtin_popcountll(mine[o]);
  }
  if (lane == 0) p.waves[wave] = found;
  __syncthreads();
  uint32_t at = 0;
  for (int w = 0; w < wave; ++w) at += p.waves[w];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    if (mine[o] >> lane & 1)
      p.list[at + (uint32_t)__builtin_popcountll(mine[o] & ((1ull << lane) - 1))] = (uint16_t)((wave * each + o) * 64 + lane);
    at += (uint32_t)__builtin_popcountll(mine[o]);
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------
// Products of M times 16 weight rows with NC times 16 tokens
// ---------------------------------------------------------------------------------------------
// In a step of 128 of K a lane has row (or token) lane % 16 and the 32 neighbours from 32 (lane / 16) on; both
// operands take the same ones, so that their order in a product does not matter.
template <bool FP8, int M>
struct Weights {
  static constexpr int kWords = FP8 ? 2 : 4;   // of 16 bytes
  static constexpr int kEach = FP8 ? 16 : 8;   // elements of one
  u4 w[M][kWords];
  float scale[FP8 ? M : 1];
  // rows[m] + off: this lane's; left: elements of K from this lane's first on
  __device__ __forceinline__ void load(const uint8_t* const (&rows)[M], int64_t off, int left) {
    if (__builtin_expect(left >= 32, 1)) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < kWords; ++j) w[m][j] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(rows[m] + off) + j);
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          w[m][j] = u4{0, 0, 0, 0};
          if (j * kEach < left) w[m][j] = *(reinterpret_cast<const u4*>(rows[m] + off) + j);
        }
    }
  }
  // the q-th 8 elements of row m as bf16
  __device__ __forceinline__ bf8 frag(int m, int q) const {
    if constexpr (!FP8) {
      return __builtin_bit_cast(bf8, w[m][q]);
    } else {
      const uint32_t a = w[m][q >> 1][2 * (q & 1)], b = w[m][q >> 1][2 * (q & 1) + 1];
      const bf2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
      const bf2 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
      const bf2 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
      const bf2 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
      return bf8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
    }
  }
};

template <int NC, int P>
struct Tokens {
  u4 b[NC][P][4];
  // cols[c]: this lane's token's, null for none; parts `plane` elements apart
  __device__ __forceinline__ void load(const uint16_t* const (&cols)[NC], int64_t plane, int64_t off, int left) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          b[c][p][q] = u4{0, 0, 0, 0};
          if (cols[c] && q * 8 < left) b[c][p][q] = *(reinterpret_cast<const u4*>(cols[c] + p * plane + off) + q);
        }
  }
};

template <bool FP8, int M, int NC, int P>
__device__ __forceinline__ void multiply(f4 (&acc)[M][NC], const Weights<FP8, M>& w, const Tokens<NC, P>& x) {
  f4 sum[M][NC];
  if constexpr (FP8) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c) sum[m][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bf8 row = w.frag(m, q);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int p = P - 1; p >= 0; --p) {
          f4& s = FP8 ? sum[m][c] : acc[m][c];
          s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(row, __builtin_bit_cast(bf8, x.b[c][p][q]), s, 0, 0, 0);
        }
    }
  if constexpr (FP8) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][c][i] = __builtin_fmaf(w.scale[m], sum[m][c][i], acc[m][c][i]);
  }
}

// acc += rows[.., first : end : step steps of K] times the tokens; the next step's loads go out before a step's
// products (the tokens' too, where they are few registers; else theirs of this step go first, as loads are waited
// for in their order).
template <bool FP8, int M, int NC, int P>
__device__ __forceinline__ void sum_steps(f4 (&acc)[M][NC], const uint8_t* const (&rows)[M], const float* const (&scales)[M],
                                          const uint16_t* const (&cols)[NC], int64_t plane, int K, int first, int end,
                                          int step) {
  constexpr bool kAhead = NC * P <= 2;
  if (first >= end) return;
  const int mine = (threadIdx.x >> 4 & 3) * 32;
  Weights<FP8, M> w, next;
  Tokens<NC, P> x, ahead;
  auto load = [&](Weights<FP8, M>& to, int b) {
    to.load(rows, (int64_t)b * (FP8 ? kBlock : 2 * kBlock), K - b * kBlock - mine);
    if constexpr (FP8) {
#pragma unroll
      for (int m = 0; m < M; ++m) to.scale[m] = scales[m][b];
    }
  };
  auto tokens = [&](Tokens<NC, P>& to, int b) { to.load(cols, plane, (int64_t)b * kBlock, K - b * kBlock - mine); };
  load(w, first);
  if constexpr (kAhead) tokens(x, first);
  for (int b = first; b < end; b += 2 * step) {
    if constexpr (!kAhead) tokens(x, b);
    if (b + step < end) {
      load(next, b + step);
      if constexpr (kAhead) tokens(ahead, b + step);
    }
    multiply<FP8, M, NC, P>(acc, w, x);
    if (b + step >= end) break;
    if constexpr (!kAhead) tokens(x, b + step);
    if (b + 2 * step < end) {
      load(w, b + 2 * step);
      if constexpr (kAhead) tokens(x, b + 2 * step);
    }
    multiply<FP8, M, NC, P>(acc, next, kAhead ? ahead : x);
  }
}

// ---------------------------------------------------------------------------------------------
// Up: h = weight * silu(W1 x) * (W2 x)
// ---------------------------------------------------------------------------------------------
template <int R>
struct UpShared {
  Plan plan;
  f4 sum[kUpWaves][2 * R][64];
};

template <int DT, bool FP8, int R, int NC, class LDS>
__device__ __forceinline__ void up_unit(const LayerArgs& a, LDS& lds, const Expert w, int expert, int h0, int first, int n,
                                        bool shared) {
  constexpr int M = 2 * R, P = kXParts<DT>, PH = kHParts<DT>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int H = w.H, KB = (a.D + kBlock - 1) / kBlock, RB = (2 * H + kBlock - 1) / kBlock;
  const int64_t pitch = (int64_t)a.D * (FP8 ? 1 : 2);
  const uint8_t* rows[M];
  const float* scales[M];
  const uint16_t* cols[NC];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int row = (m < R ? 0 : H) + h0 + 16 * (m < R ? m : m - R);
    rows[m] = w.w12 + ((int64_t)expert * 2 * H + row + r) * pitch + g * (FP8 ? 32 : 64);
    scales[m] = FP8 ? w.s12 + ((int64_t)expert * RB + row / kBlock) * KB : nullptr;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = c * 16 + r;
    cols[c] = nullptr;
    if (i < n) {
      const int t = shared ? first + i : lds.plan.list[first + i] / a.k;
      cols[c] = a.xb + (int64_t)t * a.Dp + g * 32;
    }
  }
  f4 acc[M][NC];
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[m][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  sum_steps<FP8, M, NC, P>(acc, rows, scales, cols, (int64_t)a.T * a.Dp, a.D, wave, KB, kUpWaves);
  const int64_t plane = (int64_t)(shared ? a.T : a.T * a.k) * H;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c * 16 >= n) break;
    if (c) __syncthreads();  // (the readers before)
#pragma unroll
    for (int m = 0; m < M; ++m) lds.sum[wave][m][lane] = acc[m][c];
    __syncthreads();
    // (four neighbouring channels of one token each)
    const int m = wave, at = c * 16 + r;
    if (m >= R || at >= n) continue;
    f4 h1 = lds.sum[0][m][lane], h2 = lds.sum[0][m + R][lane];
#pragma unroll
    for (int v = 1; v < kUpWaves; ++v) {
      h1 += lds.sum[v][m][lane];
      h2 += lds.sum[v][m + R][lane];
    }
    const int row = shared ? first + at : lds.plan.list[first + at];
    const float weight = shared ? 1.0f : a.weights[row];
    float h[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[e] = weight * (h1[e] / (1.0f + expf(-h1[e])) * h2[e]);
      h[4 + e] = 0.0f;
    }
    u4 part[PH];
    split8<PH>(h, part);
    uint16_t* to = (shared ? a.hs : a.hb) + (int64_t)row * H + h0 + 16 * m + 4 * g;
#pragma unroll
    for (int p = 0; p < PH; ++p) {
      const uint2 v = {part[p][0], part[p][1]};
      *reinterpret_cast<uint2*>(to + p * plane) = v;
    }
  }
}

template <int DT, bool FP8, int R, bool FEW>
__global__ __launch_bounds__(64 * kUpWaves) void k_up(LayerArgs a) {
  constexpr int UNIT = unit_tokens(DT);
  __shared__ UpShared<R> lds;
  const int tiles = (a.experts.H + 16 * R - 1) / (16 * R);
  const int routed = a.units * tiles;
  const bool shared = (int)blockIdx.x >= routed;
  int expert = 0, tile, first, n, H;
  if (!shared) {
    const int u = blockIdx.x / tiles;
    tile = blockIdx.x - u * tiles;
    make_plan<64 * kUpWaves, UNIT, false>(lds.plan, a.idx, a.T * a.k, a.E);
    if (u >= lds.plan.units) return;
    expert = (int)(lds.plan.unit[u] >> 16);
    first = (int)(lds.plan.unit[u] & 0xffffu);
    n = lds.plan.tokens[u];
    list_of<64 * kUpWaves>(lds.plan, a.idx, a.T * a.k, expert);
    H = a.experts.H;
  } else {
    H = a.shared.H;
    const int i = blockIdx.x - routed, per = (H + 16 * R - 1) / (16 * R);
    tile = i % per;
    first = i / per * UNIT;
    n = min(a.T - first, UNIT);
  }
  const Expert w = shared ? a.shared : a.experts;
  const int h0 = tile * 16 * R;
  auto run = [&](auto rows, auto columns) {
    up_unit<DT, FP8, decltype(rows)::value, decltype(columns)::value>(a, lds, w, expert, h0, first, n, shared);
  };
  auto with = [&](auto rows) {
    if (FEW || n <= 16)
      run(rows, std::integral_constant<int, 1>{});
    else if (UNIT == 32 || n <= 32)
      run(rows, std::integral_constant<int, FEW ? 1 : 2>{});
    else
      run(rows, std::integral_constant<int, FEW ? 1 : UNIT / 16>{});
  };
  if (R == 1 || h0 + 16 * R <= H)
    with(std::integral_constant<int, R>{});
  else
    with(std::integral_constant<int, 1>{});  // the last 16 channels of an odd number of them
}

// ---------------------------------------------------------------------------------------------
// Down: out = sum W3 h
// ---------------------------------------------------------------------------------------------
template <int R>
constexpr int kDownPitch = 16 * R + 4;  // floats of a token's sums in LDS

template <int DT, bool FP8, int R, int NC>
__device__ __forceinline__ void down_unit(const LayerArgs& a, const Plan& plan, float* sums, const Expert w, int expert, int d0,
                                          int first, int n, bool shared, int kb0, int kb1) {
  constexpr int P = kHParts<DT>;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int H = w.H, KB = (H + kBlock - 1) / kBlock, RB = (a.D + kBlock - 1) / kBlock;
  const int64_t pitch = (int64_t)H * (FP8 ? 1 : 2);
  const uint8_t* rows[R];
  const float* scales[R];
  const uint16_t* cols[NC];
  int token[NC];
#pragma unroll
  for (int m = 0; m < R; ++m) {
    const int row = d0 + 16 * m;
    rows[m] = w.w3 + ((int64_t)expert * a.D + row + r) * pitch + g * (FP8 ? 32 : 64);
    scales[m] = FP8 ? w.s3 + ((int64_t)expert * RB + row / kBlock) * KB : nullptr;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = c * 16 + r;
    cols[c] = nullptr;
    token[c] = -1;
    if (i < n) {
      const int at = shared ? first + i : plan.list[first + i];
      token[c] = shared ? at : at / a.k;
      cols[c] = (shared ? a.hs : a.hb) + (int64_t)at * H + g * 32;
    }
  }
  f4 acc[R][NC];
#pragma unroll
  for (int m = 0; m < R; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[m][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  sum_steps<FP8, R, NC, P>(acc, rows, scales, cols, (int64_t)(shared ? a.T : a.T * a.k) * H, H, kb0, kb1, 1);
  // (a token has an expert once, so a wave adds to a value once a unit)
#pragma unroll
  for (int c = 0; c < NC; ++c)
    if (token[c] >= 0) {
#pragma unroll
      for (int m = 0; m < R; ++m) {
        f4* to = reinterpret_cast<f4*>(sums + token[c] * kDownPitch<R> + 16 * m + 4 * g);
        *to += acc[m][c];
      }
    }
}

template <int DT, bool FP8, int R, bool FEW>
__global__ __launch_bounds__(64 * kDownWaves) void k_down(LayerArgs a) {
  constexpr int UNIT = unit_tokens(DT);
  __shared__ Plan plan;
  extern __shared__ f4 joined[];  // [waves][T][kDownPitch] floats
  float* const sums = reinterpret_cast<float*>(joined);
  const int wave = threadIdx.x >> 6;
  const int d0 = blockIdx.x * 16 * R;
  const bool half = R == 2 && d0 + 32 > a.D;  // the last 16 channels of an odd number of them
  make_plan<64 * kDownWaves, UNIT, true>(plan, a.idx, a.T * a.k, a.E);
  const int each = a.T * kDownPitch<R>;
  for (int i = threadIdx.x; i < kDownWaves * each; i += 64 * kDownWaves) sums[i] = 0.0f;
  __syncthreads();
  // the waves share the steps of all units, the shared expert's behind the others'
  const int KB = (a.experts.H + kBlock - 1) / kBlock;
  const int routed = plan.units * KB;
  const int KS = a.shared.w12 ? (a.shared.H + kBlock - 1) / kBlock : 0;
  const int all = routed + (KS ? (a.T + UNIT - 1) / UNIT * KS : 0);
  int at = (int)((int64_t)all * wave / kDownWaves);
  const int end = (int)((int64_t)all * (wave + 1) / kDownWaves);
  while (at < end) {
    const bool shared = at >= routed;
    const int per = shared ? KS : KB, from = shared ? at - routed : at;
    const int u = from / per, kb0 = from - u * per, kb1 = min(per, kb0 + end - at);
    const int expert = shared ? 0 : (int)(plan.unit[u] >> 16);
    const int first = shared ? u * UNIT : (int)(plan.unit[u] & 0xffffu);
    const int n = shared ? min(a.T - first, UNIT) : plan.tokens[u];
    const Expert w = shared ? a.shared : a.experts;
    auto run = [&](auto columns) {
      constexpr int NC = decltype(columns)::value;
      if (half) {
        // rows past D would lie outside: one fragment, its sums at the same pitch
        down_unit<DT, FP8, 1, NC>(a, plan, sums + wave * each, w, expert, d0, first, n, shared, kb0, kb1);
      } else {
        down_unit<DT, FP8, R, NC>(a, plan, sums + wave * each, w, expert, d0, first, n, shared, kb0, kb1);
      }
    };
    if (FEW || n <= 16)
      run(std::integral_constant<int, 1>{});
    else if (UNIT == 32 || n <= 32)
      run(std::integral_constant<int, FEW ? 1 : 2>{});
    else
      run(std::integral_constant<int, FEW ? 1 : UNIT / 16>{});
    at += kb1 - kb0;
  }
  __syncthreads();
  const int width = half ? 16 : 16 * R, row_pitch = half ? kDownPitch<1> : kDownPitch<R>;
  for (int i = threadIdx.x; i < a.T * width; i += 64 * kDownWaves) {
    const int t = i / width, d = i - t * width;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < kDownWaves; ++v) s += sums[v * each + t * row_pitch + d];
    const int64_t o = (int64_t)t * a.D + d0 + d;
    if constexpr (DT == CIN_DT_F32)
      static_cast<float*>(a.out)[o] = s;
    else
      static_cast<uint16_t*>(a.out)[o] = (uint16_t)f32_to_half_bits(DT, s);
  }
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
constexpr int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Bytes of the workspace; fills its pointers where `base` is given.
int64_t layout(LayerArgs& a, int dtype, char* base) {
  const int64_t px = dtype == CIN_DT_BF16 ? 1 : dtype == CIN_DT_F16 ? 2 : 3, ph = dtype == CIN_DT_F32 ? 3 : 2;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = base ? base + at : nullptr;
    at += padded(bytes);
    return p;
  };
  a.logits = reinterpret_cast<double*>(take(8LL * a.slices * a.T * a.E));
  a.xb = reinterpret_cast<uint16_t*>(take(2 * px * a.T * a.Dp));
  a.hb = reinterpret_cast<uint16_t*>(take(2 * ph * a.T * a.k * a.experts.H));
  a.hs = reinterpret_cast<uint16_t*>(take(2 * ph * a.T * a.shared.H));
  return at;
}

bool sizes_ok(int dtype, int64_t T, int64_t D, int64_t E, int64_t k, int64_t H, int64_t Hs) {
  return (dtype == CIN_DT_BF16 || dtype == CIN_DT_F16 || dtype == CIN_DT_F32) && T >= 0 && T <= kMaxTokens && D >= 16 &&
         D <= 65536 && D % 16 == 0 && E >= 1 && E <= kMaxExperts && k >= 1 && k <= kMaxTopK && k <= E && H >= 16 && H <= 65536 &&
         H % 16 == 0 && Hs >= 0 && Hs <= 65536 && Hs % 16 == 0;
}
const char* const kSizes =
    "dtype must be bf16, fp16 or fp32, T <= 128, E <= 1024, k <= min(16, E), D, H and the shared expert's H multiples of 16 up to 65536";

void set_sizes(LayerArgs& a, int dtype, int64_t T, int64_t D, int64_t E, int64_t k, int64_t H, int64_t Hs) {
  a.T = (int)T;
  a.D = (int)D;
  a.Dp = (int)(cdiv(D, kBlock) * kBlock);
  a.E = (int)E;
  a.k = (int)k;
  a.experts.H = (int)H;
  a.shared.H = (int)Hs;
  a.slices = (int)cdiv(a.Dp, kRouterSlice);
  const int64_t n = T * k;
  a.units = (int)((n < E ? n : E) + n / unit_tokens(dtype));
}

// FEW: at most 16 tokens, RD times 16 rows a workgroup of k_down.
template <int DT, bool FP8, bool FEW>
void launch_products(const LayerArgs& a, hipStream_t stream) {
  constexpr int RU = 1, RD = FEW ? 1 : 2;
  const int per = (a.experts.H + 16 * RU - 1) / (16 * RU), unit = unit_tokens(DT);
  const int shared = a.shared.w12 ? (a.shared.H + 16 * RU - 1) / (16 * RU) * ((a.T + unit - 1) / unit) : 0;
  hipLaunchKernelGGL((k_up<DT, FP8, RU, FEW>), dim3(a.units * per + shared), dim3(64 * kUpWaves), 0, stream, a);
  const size_t lds = sizeof(float) * kDownWaves * a.T * kDownPitch<RD>;
  if (lds + sizeof(Plan) > 65536)
    (void)hipFuncSetAttribute((const void*)k_down<DT, FP8, RD, FEW>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((k_down<DT, FP8, RD, FEW>), dim3((a.D + 16 * RD - 1) / (16 * RD)), dim3(64 * kDownWaves), lds, stream, a);
}

template <int DT>
void launch(const LayerArgs& a, bool fp8, hipStream_t stream) {
  hipLaunchKernelGGL((k_router<DT>), dim3(a.slices * ((a.E + 15) / 16), (a.T + 15) / 16), dim3(256), 0, stream, a);
  hipLaunchKernelGGL(k_gate, dim3(a.T), dim3(256), 0, stream, a);
  if (fp8 && a.T <= 16)
    launch_products<DT, true, true>(a, stream);
  else if (fp8)
    launch_products<DT, true, false>(a, stream);
  else if (a.T <= 16)
    launch_products<DT, false, true>(a, stream);
  else
    launch_products<DT, false, false>(a, stream);
}

}  // namespace

extern "C" {

int64_t cin_moe_decode_workspace(int dtype, int64_t T, int64_t D, int64_t E, int64_t k, int64_t H, int64_t shared_H) {
  if (!sizes_ok(dtype, T, D, E, k, H, shared_H)) {
    cin_set_error(CIN_ERR_ARG, "cin_moe_decode_workspace: %s", kSizes);
    return -1;
  }
  LayerArgs a = {};
  set_sizes(a, dtype, T, D, E, k, H, shared_H);
  return layout(a, dtype, nullptr);
}

int cin_moe_decode(const void* x, int dtype, int64_t ldx, int64_t T, int64_t D, const void* router, int router_dtype,
                   int64_t ldr, int64_t E, const float* bias, int64_t k, int score, int64_t groups, int64_t top_groups,
                   int group_top, int renormalize, float scale, int weights_fp8, const void* w12, const float* s12,
                   const void* w3, const float* s3, int64_t H, const void* shared_w12, const float* shared_s12,
                   const void* shared_w3, const float* shared_s3, int64_t shared_H, void* out, int64_t* idx, float* weights,
                   void* workspace, int64_t workspace_bytes, void* stream) {
  CIN_CHECK_ARG(sizes_ok(dtype, T, D, E, k, H, shared_H), "cin_moe_decode: %s", kSizes);
  CIN_CHECK_ARG(router_dtype == CIN_DT_BF16 || router_dtype == CIN_DT_F16 || router_dtype == CIN_DT_F32,
                "cin_moe_decode: router_dtype must be bf16, fp16 or fp32");
  CIN_CHECK_ARG((score == 0 || score == 1) && groups >= 1 && groups <= kMaxGroups && E % groups == 0 && top_groups >= 1 &&
                    top_groups <= groups && (group_top == 1 || group_top == 2) && k <= top_groups * (E / groups),
                "cin_moe_decode: bad gate options");
  CIN_CHECK_ARG(ldx >= D && ldr >= D, "cin_moe_decode: row stride below D");
  if (T == 0) return CIN_OK;
  CIN_CHECK_ARG(x && router && w12 && w3 && out && idx && weights && workspace, "cin_moe_decode: null pointer");
  CIN_CHECK_ARG((shared_H != 0) == (shared_w12 != nullptr) && (shared_H != 0) == (shared_w3 != nullptr),
                "cin_moe_decode: the shared expert's weights go with its H");
  CIN_CHECK_ARG((!weights_fp8 || (s12 && s3)) && (!weights_fp8 || !shared_H || (shared_s12 && shared_s3)),
                "cin_moe_decode: codes need their scales");
  CIN_CHECK_ARG(((uintptr_t)w12 | (uintptr_t)w3 | (uintptr_t)shared_w12 | (uintptr_t)shared_w3 | (uintptr_t)workspace) % 16 == 0,
                "cin_moe_decode: weights and workspace must lie on 16 bytes");
  CIN_CHECK_ARG(workspace_bytes >= cin_moe_decode_workspace(dtype, T, D, E, k, H, shared_H),
                "cin_moe_decode: workspace below cin_moe_decode_workspace bytes");
  LayerArgs a = {};
  set_sizes(a, dtype, T, D, E, k, H, shared_H);
  layout(a, dtype, static_cast<char*>(workspace));
  a.x = x;
  a.ldx = ldx;
  a.router = router;
  a.router_dtype = router_dtype;
  a.ldr = ldr;
  a.bias = bias;
  a.score = score;
  a.groups = (int)groups;
  a.top_groups = (int)top_groups;
  a.group_top = group_top;
  a.renormalize = renormalize;
  a.scale = scale;
  a.experts = {static_cast<const uint8_t*>(w12), static_cast<const uint8_t*>(w3), s12, s3, (int)H};
  a.shared = {static_cast<const uint8_t*>(shared_w12), static_cast<const uint8_t*>(shared_w3), shared_s12, shared_s3,
              (int)shared_H};
  a.out = out;
  a.idx = idx;
  a.weights = weights;
  if (dtype == CIN_DT_BF16)
    launch<CIN_DT_BF16>(a, weights_fp8 != 0, (hipStream_t)stream);
  else if (dtype == CIN_DT_F16)
    launch<CIN_DT_F16>(a, weights_fp8 != 0, (hipStream_t)stream);
  else
    launch<CIN_DT_F32>(a, weights_fp8 != 0, (hipStream_t)stream);
  return cin_check_launch("cin_moe_decode");
}

}  // extern "C"
