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
// Rounding: x is split into bf16 parts that hold it exactly (one for bf16, two for fp16, three for fp32); h, formed in
// fp32, into three (2^-25 of a value): two parts' 2^-17 would show wherever an output's terms cancel, in 16 bits too
// (one token 84.8 us with two, 85.6 with three, 64 tokens 308 and 327, 128 tokens 411 and 479).  All sums are fp32.  Logits and the gate are in 64 bits: choices next to
// the border of the top k differ by less than 32 bits hold.
//
// Five launches: k_router (logits by slices of D on the fp64 matrix units, and x's parts), k_gate (a workgroup a
// token, and the shared expert's h where that is little work), the products up to h and down to each expert's output
// rows, and k_join (a token's rows in the order of top k).  The products take a workgroup an expert's tokens and some
// of its rows:
//   k_few, up to 16 tokens and where the others would leave CUs idle: 16 rows of W1 and W2, or 32 of W3, the waves
//   sharing K;
//   k_products: as many rows a wave; the tokens' parts go through LDS once for all waves, as they
//   would be more bytes than the weights.
// No atomics on results.
//
// Bound by the weights' bytes.  32 experts of 7168 x 2048 in codes, 8 a token, and a shared one: one token 80 us (0.40 GB,
// 5.0 TB/s: up 40, down 24), 64 tokens 327 (1.46 GB, 4.5: up 163-180, down 131-146), 128 tokens 481.  16 experts of
// 1024 x 1024, one token: 26, the latency of five launches.
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
constexpr int kUnitTokens = 32;    // of an expert, multiplied at once, or twice as many (unit_tokens)
constexpr int kRouterSlice = 256;  // channels of a k_router workgroup
constexpr int kFewWaves = 4, kTileWaves = 4;
constexpr int kFewTokens = 16;

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef double d4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Parts of x for its type, and of h.
template <int DT>
constexpr int kXParts = DT == CIN_DT_BF16 ? 1 : DT == CIN_DT_F16 ? 2 : 3;
constexpr int kHParts = 3;

struct Expert {  // stacked experts, or a shared one
  const uint8_t *w12, *w3;
  const float *s12, *s3;  // null for bf16
  int H;
};

// A unit: up to kUnitTokens or twice as many tokens of one expert, as assignments t k + j.
struct UnitPlan {
  uint32_t expert, tokens;  // no tokens: no such unit
  uint16_t list[2 * kUnitTokens];
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
  float* y;                // the experts' outputs [T k, D], the shared one's [T, D]
  UnitPlan* plans;         // [units]
  int unit, units;         // tokens of a unit, and the most units that the routed experts can have
};

// Scales, the same for all lanes and nowhere written here: scalar loads.
typedef const __attribute__((address_space(4))) float* floats_at;

// 16 bytes at an offset into a buffer; zeros from kNothing on.  No load of k_products is behind a branch: one
// that may not have been issued would have to be counted as issued last, and all before it waited for.
constexpr uint32_t kNothing = 0x80000000u;
template <int AUX = 0>
__device__ __forceinline__ u4 load16(__amdgpu_buffer_rsrc_t from, uint32_t at) {
  return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, AUX));
}
constexpr int kStream = 2;  // read once: not kept in the caches

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

// bf16 parts of 8 values: each the rounding of what the ones before leave, kept finite for a finite value; an infinity has
// one.
template <int P>
__device__ __forceinline__ void split8(const float (&v)[8], u4 (&part)[P]) {
  float r[8];
  bool far = false;  // a value that rounds to infinity, or is one
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    r[e] = v[e];
    far |= fabsf(v[e]) >= 0x1.ffp127f;
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (P > 1 && far) {
        const uint32_t lo = take_part(r[2 * i]);
        part[p][i] = lo | take_part(r[2 * i + 1]) << 16;
      } else {
        part[p][i] = f32x2_to_bf16x2_bits(r[2 * i], r[2 * i + 1]);
        r[2 * i] -= bf16_lo(part[p][i]);
        r[2 * i + 1] -= bf16_hi(part[p][i]);
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

template <int WAVES>
__device__ inline double block_reduce(double v, bool maximum, double* lds) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_xor(v, o);
    v = maximum ? (u > v || u != u ? u : v) : v + u;
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = lds[0];
  for (int w = 1; w < WAVES; ++w) r = maximum ? (lds[w] > r || lds[w] != lds[w] ? lds[w] : r) : r + lds[w];
  __syncthreads();
  return r;
}

// A token's experts and weights, by one workgroup.
template <int WAVES>
__device__ __forceinline__ void choose(const LayerArgs& a, int t) {
  __shared__ double score[kMaxExperts], reduce[WAVES];
  __shared__ uint64_t key[kMaxExperts], group_key[kMaxGroups];
  __shared__ int chosen[kMaxTopK], kept[kMaxGroups];
  constexpr int kThreads = 64 * WAVES, kOwn = kMaxExperts / kThreads;
  const int tid = threadIdx.x;
  double z[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid + o * kThreads;
    z[o] = -__builtin_inf();
    if (e < a.E) {
      const double* p = a.logits + (int64_t)t * a.E + e;
      double s = 0.0;
      for (int i = 0; i < a.slices; i += 16) {
        double v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = p[(int64_t)min(i + j, a.slices - 1) * a.T * a.E];
#pragma unroll
        for (int j = 0; j < 16; ++j) s += i + j < a.slices ? v[j] : 0.0;
      }
      z[o] = s;
    }
  }
  if (a.score == 1) {
    double m = z[0];
#pragma unroll
    for (int o = 1; o < kOwn; ++o) m = z[o] > m || z[o] != z[o] ? z[o] : m;
    m = block_reduce<WAVES>(m, true, reduce);
    double sum = 0.0;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      z[o] = tid + o * kThreads < a.E ? exp(z[o] - m) : 0.0;
      sum += z[o];
    }
    sum = block_reduce<WAVES>(sum, false, reduce);
#pragma unroll
    for (int o = 0; o < kOwn; ++o) z[o] /= sum;
  } else {
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      if (tid + o * kThreads < a.E) {
        const double q = exp(-fabs(z[o]));
        z[o] = z[o] < 0 ? q / (1.0 + q) : 1.0 / (1.0 + q);
      }
    }
  }
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid + o * kThreads;
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
    for (int e = tid; e < a.E; e += kThreads)
      if (!kept[e / n]) key[e] = 0;
    __syncthreads();
  }
  // an expert's place is the number of experts in front of it
  uint64_t mine[kOwn];
  int rank[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int e = tid + o * kThreads;
    mine[o] = e < a.E ? key[e] : 0;
    rank[o] = 0;
  }
  const int own = (a.E + kThreads - 1) / kThreads;
#pragma unroll 8
  for (int j = 0; j < a.E; ++j) {
    const uint64_t other = key[j];
    rank[0] += other > mine[0] || (other == mine[0] && j < tid);
    if (own > 1) {
#pragma unroll
      for (int o = 1; o < kOwn; ++o) rank[o] += other > mine[o] || (other == mine[o] && j < tid + o * kThreads);
    }
  }
#pragma unroll
  for (int o = 0; o < kOwn; ++o)
    if (tid + o * kThreads < a.E && rank[o] < a.k) chosen[rank[o]] = tid + o * kThreads;
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
// One unit: up to UNIT tokens of one expert.  The assignments (t k + j) are counted by expert, and the experts' units
// follow each other; the unit's list holds its expert's assignments in increasing order, so that the workgroups that take
// the expert's units each find the same.
template <int THREADS, int UNIT, int MOST>
struct OneUnit {
  int count[kMaxExperts];  // assignments of an expert
  uint32_t waves[THREADS / 64];
  uint32_t unit;           // expert, first entry of the list
  int tokens;
  uint16_t expert[MOST], list[kMaxTokens];

  // false where there is no unit u
  __device__ __forceinline__ bool make(const int64_t* idx, int T, int k, int E, int u) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = T * k;
    if (T == 1) {  // every assignment is a unit
      if (tid == 0) {
        unit = (uint32_t)idx[u] << 16;
        tokens = 1;
        list[0] = (uint16_t)u;
      }
      __syncthreads();
      return true;
    }
    for (int e = tid; e < E; e += THREADS) count[e] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      const int e = (int)idx[i];
      expert[i] = (uint16_t)e;
      atomicAdd(&count[e], 1);
    }
    __syncthreads();
    // units of the experts before this thread's
    constexpr int kOwn = kMaxExperts / THREADS;
    int own = 0, c[kOwn];
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      c[o] = tid * kOwn + o < E ? count[tid * kOwn + o] : 0;
      own += (c[o] + UNIT - 1) / UNIT;
    }
    int s = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(s, o);
      if (lane >= o) s += v;
    }
    if (lane == 63) waves[wave] = (uint32_t)s;
    __syncthreads();
    int at = s - own, all = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) at += (int)waves[w];
      all += (int)waves[w];
    }
    if (u >= all) return false;
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
      for (int i = 0; i < c[o]; i += UNIT, ++at)
        if (at == u) {
          unit = (uint32_t)(tid * kOwn + o) << 16 | (uint32_t)i;
          tokens = min(c[o] - i, UNIT);
        }
    __syncthreads();
    const int mine = (int)(unit >> 16);
    constexpr int kWaves = THREADS / 64;
    const int each = (n + kWaves * 64 - 1) / (kWaves * 64);  // rounds of 64 assignments, a wave's one behind the other
    uint32_t found = 0;
    for (int o = 0; o < each; ++o) {
      const int i = (wave * each + o) * 64 + lane;
      found += (uint32_t)__builtin_popcountll(__ballot(i < n && expert[i < n ? i : 0] == mine));
    }
    if (lane == 0) waves[wave] = found;
    __syncthreads();
    uint32_t to = 0;
    for (int w = 0; w < wave; ++w) to += waves[w];
    for (int o = 0; o < each; ++o) {
      const int i = (wave * each + o) * 64 + lane;
      const bool here = i < n && expert[i < n ? i : 0] == mine;
      const uint64_t m = __ballot(here);
      if (here) list[to + (uint32_t)__builtin_popcountll(m & ((1ull << lane) - 1))] = (uint16_t)i;
      to += (uint32_t)__builtin_popcountll(m);
    }
    __syncthreads();
    return true;
  }
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What a workgroup of the products keeps of its unit: the first product finds it from the chosen experts, and leaves it for
// the second.
template <bool UP, int THREADS, int UNIT, int MOST>
struct Unit : OneUnit<THREADS, UNIT, MOST> {};
template <int THREADS, int UNIT, int MOST>
struct Unit<false, THREADS, UNIT, MOST> {
  uint16_t list[UNIT];
};
// False where there is no unit u; else its expert and n tokens, list[first] and on.
template <int THREADS, int UNIT, int MOST>
__device__ __forceinline__ bool find_unit(const LayerArgs& a, Unit<true, THREADS, UNIT, MOST>& plan, int u, bool leave, int& expert,
                                          int& first, int& n) {
  const bool there = plan.make(a.idx, a.T, a.k, a.E, u);
  expert = there ? uniform((int)(plan.unit >> 16)) : 0;
  first = there ? uniform((int)(plan.unit & 0xffffu)) : 0;
  n = there ? uniform(plan.tokens) : 0;
  if (leave) {
    UnitPlan& p = a.plans[u];
    if (threadIdx.x == 0) {
      p.expert = (uint32_t)expert;
      p.tokens = (uint32_t)n;
    }
    if ((int)threadIdx.x < n) p.list[threadIdx.x] = plan.list[first + threadIdx.x];
  }
  return there;
}
template <int THREADS, int UNIT, int MOST>
__device__ __forceinline__ bool find_unit(const LayerArgs& a, Unit<false, THREADS, UNIT, MOST>& plan, int u, bool, int& expert,
                                          int& first, int& n) {
  const UnitPlan& p = a.plans[u];
  expert = uniform((int)p.expert);
  first = 0;
  n = uniform((int)p.tokens);
  if (n == 0) return false;
  if ((int)threadIdx.x < UNIT) plan.list[threadIdx.x] = p.list[threadIdx.x];
  __syncthreads();
  return true;
}

// ---------------------------------------------------------------------------------------------
// Products of 16 weight rows with 16 tokens
// ---------------------------------------------------------------------------------------------
// In a step of 128 of K a lane multiplies row (or token) lane % 16, and of it four times 8 elements, the q-th from
// k_of(q, lane / 16) on.  Both operands take the same elements, so their order in a product does not matter.
//
// A load takes 8 rows' 128 adjacent bytes (lane: row lane % 8, 16 bytes from 16 (lane / 8) on), a whole line of each,
// streamed past the caches where rows begin on lines: 969 MB of codes in rows of 7168 arrive at 6.2 TB/s, against 4.8
// with 64 bytes of 16 rows a load and 5.5 with those kept in the caches (linear reads: 7.0).  Two loads, of rows 0-7 and
// 8-15, then hold every lane's two words, half of them in the lane 8 further in its row of 16: settle() swaps those.
template <bool FP8>
__device__ __forceinline__ constexpr int k_of(int q, int g) {
  return FP8 ? g * 32 + q * 8 : (q >> 1) * 64 + g * 16 + (q & 1) * 8;
}
template <bool FP8, bool STREAM, int M>
struct Weights {
  static constexpr int kWords = FP8 ? 2 : 4;  // of 16 bytes
  u4 w[M][kWords];
  float scale[FP8 ? M : 1];
  // step b of 8 rows[m][i] from this lane's offset on, scaled by scales[m]
  __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t (&rows)[M][2], uint32_t mine, const floats_at (&scales)[M], int b,
                                       int K) {
    const uint32_t off = mine + (uint32_t)b * (FP8 ? kBlock : 2 * kBlock);
    const int left = K - b * kBlock, c = threadIdx.x >> 3 & 7;
#pragma unroll
    for (int j = 0; j < kWords / 2; ++j) {
      const uint32_t at = (FP8 ? c * 16 : j * 64 + c * 8) < left ? off + 128 * j : kNothing;
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) w[m][2 * j + i] = load16<STREAM ? kStream : 0>(rows[m][i], at);
    }
    if constexpr (FP8) {
#pragma unroll
      for (int m = 0; m < M; ++m) scale[m] = scales[m][left > 0 ? b : 0];  // (past the end: any)
    }
  }
  // from the loads' order to the lanes' rows: lanes 0-7 of 16 keep the first load's word and take the other's from
  // 8 lanes on, lanes 8-15 the other way round
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int j = 0; j < kWords; j += 2)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int a = (int)w[m][j][d], b = (int)w[m][j + 1][d];
          w[m][j][d] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x128, 0xF, 0xC, false);      // row_ror:8
          w[m][j + 1][d] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x128, 0xF, 0x3, false);
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

// 16 rows of an expert's stacked weights from `row` on, a lane's offset into their halves, and their blocks' scales.
template <bool FP8>
__device__ __forceinline__ void rows_at(__amdgpu_buffer_rsrc_t (&rows)[2], const uint8_t* w, int64_t row, int K) {
  const int64_t pitch = (int64_t)K * (FP8 ? 1 : 2);
#pragma unroll
  for (int i = 0; i < 2; ++i) rows[i] = make_rsrc(w + (row + 8 * i) * pitch, 8 * pitch);
}
template <bool FP8>
__device__ __forceinline__ uint32_t offset_in_rows(int K) {
  const int lane = threadIdx.x & 63;
  return (uint32_t)((lane & 7) * K * (FP8 ? 1 : 2) + (lane >> 3) * 16);
}
__device__ __forceinline__ floats_at scales_at(const float* s, int64_t expert, int64_t row, int rows, int K) {
  return (floats_at)(uintptr_t)s + (expert * ((rows + kBlock - 1) / kBlock) + row / kBlock) * ((K + kBlock - 1) / kBlock);
}

template <bool FP8, int M, int NC>
__device__ __forceinline__ void clear(f4 (&acc)[M][NC]) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[m][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
}
// A step's sums join the others by their block's scale (16 rows share it).
template <bool FP8, bool STREAM, int M, int NC>
__device__ __forceinline__ void join_step(f4 (&acc)[M][NC], const f4 (&sum)[M][NC], const Weights<FP8, STREAM, M>& w) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][c][i] = __builtin_fmaf(w.scale[m], sum[m][c][i], acc[m][c][i]);
}

// h = weight silu(h1) h2 of four neighbouring channels, its parts stored `plane` elements apart.
template <int PH>
__device__ __forceinline__ void store_h(uint16_t* to, int64_t plane, f4 h1, f4 h2, float weight) {
  float h[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = weight * (h1[e] / (1.0f + expf(-h1[e])) * h2[e]);
    h[4 + e] = 0.0f;
  }
  u4 part[PH];
  split8<PH>(h, part);
#pragma unroll
  for (int p = 0; p < PH; ++p) {
    const uint2 v = {part[p][0], part[p][1]};
    *reinterpret_cast<uint2*>(to + p * plane) = v;
  }
}

// What a lane has of a row (an assignment's, or a shared expert's token's): four h, or four outputs of each 16 rows.
template <int DT, bool UP>
__device__ __forceinline__ void leave_rows(const LayerArgs& a, bool shared, int at, int row, bool both, f4 first, f4 second) {
  if constexpr (UP) {
    const int H = shared ? a.shared.H : a.experts.H;
    store_h<kHParts>((shared ? a.hs : a.hb) + (int64_t)at * H + row, (int64_t)(shared ? a.T : a.T * a.k) * H, first, second,
                         shared ? 1.0f : a.weights[at]);
  } else {
    float* y = a.y + (int64_t)(shared ? a.T * a.k + at : at) * a.D + row;
    *reinterpret_cast<f4*>(y) = first;
    if (both) *reinterpret_cast<f4*>(y + 16) = second;
  }
}

// ---------------------------------------------------------------------------------------------
// Few tokens
// ---------------------------------------------------------------------------------------------
template <bool FP8, int P, int NC>
struct Tokens {
  u4 b[NC][P][4];
  // a step of this lane's tokens, which begin at token[c] of parts[p] (kNothing for none)
  __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t (&parts)[P], const uint32_t (&token)[NC], int step, int K) {
    const int left = K - step * kBlock, g = threadIdx.x >> 4 & 3;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = k_of<FP8>(q, g);
        const uint32_t at = k < left ? token[c] + (uint32_t)(step * kBlock + k) * 2 : kNothing;
#pragma unroll
        for (int p = 0; p < P; ++p) b[c][p][q] = load16(parts[p], at);
      }
  }
};

template <bool FP8, bool STREAM, int M, int P, int NC>
__device__ __forceinline__ void multiply(f4 (&acc)[M][NC], Weights<FP8, STREAM, M>& w, const Tokens<FP8, P, NC>& x) {
  w.settle();
  f4 sum[M][NC];
  if constexpr (FP8) clear<FP8, M, NC>(sum);
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const bf8 row = w.frag(m, q);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int p = P - 1; p >= 0; --p) {
          f4& s = FP8 ? sum[m][c] : acc[m][c];
          s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(row, __builtin_bit_cast(bf8, x.b[c][p][q]), s, 0, 0, 0);
        }
    }
  if constexpr (FP8) join_step<FP8, STREAM, M, NC>(acc, sum, w);
}

// acc += rows[.., steps first : end : step of K] times the tokens; the loads of the next step go out before a step's
// products.
template <bool FP8, bool STREAM, int M, int P, int NC>
__device__ __forceinline__ void sum_steps(f4 (&acc)[M][NC], const __amdgpu_buffer_rsrc_t (&rows)[M][2],
                                          const floats_at (&scales)[M], const __amdgpu_buffer_rsrc_t (&parts)[P],
                                          const uint32_t (&token)[NC], int K, int first, int end, int step) {
  if (first >= end) return;
  const uint32_t mine = offset_in_rows<FP8>(K);
  Weights<FP8, STREAM, M> w, next;
  Tokens<FP8, P, NC> x, ahead;
  w.load(rows, mine, scales, first, K);
  x.load(parts, token, first, K);
  for (int b = first; b < end; b += 2 * step) {
    const int b1 = b + step, b2 = b1 + step;
    if (b1 < end) {
      next.load(rows, mine, scales, b1, K);
      ahead.load(parts, token, b1, K);
    }
    multiply<FP8, STREAM, M, P, NC>(acc, w, x);
    if (b1 >= end) break;
    if (b2 < end) {
      w.load(rows, mine, scales, b2, K);
      x.load(parts, token, b2, K);
    }
    multiply<FP8, STREAM, M, P, NC>(acc, next, ahead);
  }
}

template <bool UP>
constexpr int kFewRows = UP ? 16 : 32;  // of a workgroup

// kFewRows rows times n <= 16 NC tokens: the shared expert's from `first` on, or the assignments of a list.
template <int DT, bool FP8, bool UP, bool STREAM, int NC, int WAVES>
__device__ __forceinline__ void few_rows(const LayerArgs& a, const uint16_t* list, int expert, int tile, int first, int n, bool shared) {
  constexpr int P = UP ? kXParts<DT> : kHParts;
  __shared__ f4 sum[WAVES][2][NC][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int H = shared ? a.shared.H : a.experts.H, K = UP ? a.D : H, KB = (K + kBlock - 1) / kBlock;
  const int row0 = tile * kFewRows<UP>, stacked = UP ? 2 * H : a.D;
  const bool both = UP || row0 + 16 < a.D;  // else the second 16 rows are the first ones again and not stored
  const uint8_t* w = UP ? (shared ? a.shared.w12 : a.experts.w12) : (shared ? a.shared.w3 : a.experts.w3);
  const float* s = UP ? (shared ? a.shared.s12 : a.experts.s12) : (shared ? a.shared.s3 : a.experts.s3);
  __amdgpu_buffer_rsrc_t rows[2][2], parts[P];
  floats_at scales[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int row = row0 + (UP ? m * H : m && both ? 16 : 0);
    rows_at<FP8>(rows[m], w, (int64_t)expert * stacked + row, K);
    scales[m] = scales_at(s, expert, row, stacked, K);
  }
  const int pitch = UP ? a.Dp : H;
  const int64_t plane = (int64_t)(UP || shared ? a.T : a.T * a.k) * pitch;
#pragma unroll
  for (int p = 0; p < P; ++p) parts[p] = make_rsrc((UP ? a.xb : shared ? a.hs : a.hb) + p * plane, 2 * plane);
  int at[NC];
  uint32_t token[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = c * 16 + r;
    at[c] = i < n ? (shared ? first + i : list[i]) : 0;
    token[c] = i < n ? (uint32_t)(UP && !shared ? at[c] / a.k : at[c]) * (uint32_t)pitch * 2 : kNothing;
  }
  f4 acc[2][NC];
  clear<FP8, 2, NC>(acc);
  sum_steps<FP8, STREAM, 2, P, NC>(acc, rows, scales, parts, token, K, uniform(wave), KB, WAVES);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) sum[wave][m][c][lane] = acc[m][c];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (wave != c || c * 16 + r >= n) continue;
    f4 v[2] = {sum[0][0][c][lane], sum[0][1][c][lane]};
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
      v[0] += sum[i][0][c][lane];
      v[1] += sum[i][1][c][lane];
    }
    leave_rows<DT, UP>(a, shared, at[c], row0 + 4 * g, both, v[0], v[1]);
  }
}

// The gate, a workgroup a token, and the shared expert's h, which needs no gate (its workgroups read their tokens
// from the cache, each for itself: see early_shared).  With up to 16 tokens the waves have fewer steps each to wait for.
template <int NC>
constexpr int kGateWaves = NC == 1 ? 8 : 4;
template <int DT, bool FP8, bool STREAM, int NC>
__global__ __launch_bounds__(64 * kGateWaves<NC>) void k_gate(LayerArgs a) {
  if ((int)blockIdx.x < a.T) return choose<kGateWaves<NC>>(a, blockIdx.x);
  const int i = blockIdx.x - a.T, units = (a.T + 16 * NC - 1) / (16 * NC), tile = i / units, first = (i - tile * units) * 16 * NC;
  few_rows<DT, FP8, true, STREAM, NC, kGateWaves<NC>>(a, nullptr, 0, tile, first, min(a.T - first, 16 * NC), true);
}

template <int DT, bool FP8, bool UP, bool STREAM>
__global__ __launch_bounds__(64 * kFewWaves) void k_few(LayerArgs a) {
  __shared__ Unit<UP, 64 * kFewWaves, kFewTokens, kFewTokens * kMaxTopK> plan;
  const int tiles = ((UP ? a.experts.H : a.D) + kFewRows<UP> - 1) / kFewRows<UP>, routed = a.units * tiles;
  const bool shared = (int)blockIdx.x >= routed;
  int expert = 0, tile = blockIdx.x - routed, first = 0, n = a.T;
  if (!shared) {
    const int u = blockIdx.x / tiles;
    tile = blockIdx.x - u * tiles;
    if (!find_unit(a, plan, u, tile == 0, expert, first, n)) return;
  }
  few_rows<DT, FP8, UP, STREAM, 1, kFewWaves>(a, plan.list, expert, tile, 0, n, shared);
}

// ---------------------------------------------------------------------------------------------
// More tokens
// ---------------------------------------------------------------------------------------------
constexpr int kTokenPitch = kBlock + 8;  // elements of a token's step in LDS: 16 lanes' 16 bytes on all banks

// Elements of a step's parts in LDS, and the steps that lie there: two, or one where two would leave a CU one workgroup.
template <int P, int NC>
constexpr int kTokenStep = P * NC * 16 * kTokenPitch;
template <int P, int NC>
constexpr int kStepsInLds = P * NC > 8 ? 1 : 2;

// Rows of a workgroup: 16 hidden channels (of W1 and W2 each) a wave, or 32 output channels.
template <bool UP>
constexpr int kTileRows = kTileWaves * (UP ? 16 : 32);

template <bool UP, int UNIT>
using TilePlan = Unit<UP, 64 * kTileWaves, UNIT, kMaxAssigned>;

template <int DT, bool FP8, bool UP, bool STREAM, int NC, class Plan>
__device__ __forceinline__ void tile_unit(const LayerArgs& a, const Plan& plan, uint16_t* lds, int expert, int tile, int first, int n,
                                          bool shared) {
  constexpr int P = UP ? kXParts<DT> : kHParts;
  constexpr int kChunks = NC * 16 * P * (kBlock / 8), kThreads = 64 * kTileWaves;  // of 16 bytes, a step
  constexpr int kOwn = (kChunks + kThreads - 1) / kThreads, kInLds = kStepsInLds<P, NC>;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int H = shared ? a.shared.H : a.experts.H, K = UP ? a.D : H, KB = (K + kBlock - 1) / kBlock;
  const int row0 = tile * kTileRows<UP> + wave * (UP ? 16 : 32), rows_all = UP ? H : a.D;
  const bool active = row0 < rows_all, both = UP || row0 + 16 < rows_all;
  // this lane's weight rows; those past the end are the first ones again and not stored
  __amdgpu_buffer_rsrc_t rows[2][2];
  floats_at scales[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int row = UP ? (active ? row0 : 0) + m * H : (!active ? 0 : row0 + (m && both ? 16 : 0));
    const uint8_t* w = UP ? (shared ? a.shared.w12 : a.experts.w12) : (shared ? a.shared.w3 : a.experts.w3);
    const float* s = UP ? (shared ? a.shared.s12 : a.experts.s12) : (shared ? a.shared.s3 : a.experts.s3);
    const int stacked = UP ? 2 * H : a.D;
    rows_at<FP8>(rows[m], w, (int64_t)expert * stacked + row, K);
    scales[m] = scales_at(s, expert, row, stacked, K);
  }
  // this thread's 16 bytes of the tokens' parts (of all of them at most 128 x 16 x 65536 x 3 x 2 bytes)
  const int pitch = UP ? a.Dp : H;
  const int64_t plane = (int64_t)(UP ? a.T : shared ? a.T : a.T * a.k) * pitch;
  const __amdgpu_buffer_rsrc_t parts = make_rsrc(UP ? a.xb : shared ? a.hs : a.hb, 2 * P * plane);
  uint32_t from[kOwn], to[kOwn];
#pragma unroll
  for (int o = 0; o < kOwn; ++o) {
    const int q = threadIdx.x + o * kThreads, chunk = q & 15, i = (q >> 4) % (NC * 16), p = (q >> 4) / (NC * 16);
    from[o] = kNothing;
    to[o] = (uint32_t)((p * NC * 16 + i) * kTokenPitch + chunk * 8);
    if (q < kChunks && i < n) {
      const int at = shared ? first + i : plan.list[first + i];
      from[o] = (uint32_t)(2 * (p * plane + (int64_t)(UP && !shared ? at / a.k : at) * pitch + chunk * 8));
    }
  }
  const int end = pitch - (int)(threadIdx.x & 15) * 8;
  u4 part[kOwn];
  auto fetch = [&](int b) {
    const bool there = b * kBlock < end;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) part[o] = load16(parts, there ? from[o] + (uint32_t)b * 2 * kBlock : kNothing);
  };
  auto leave = [&](int b) {
    uint16_t* tile_b = lds + b % kInLds * kTokenStep<P, NC>;
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
      if (kChunks % kThreads == 0 || threadIdx.x + o * kThreads < kChunks) *reinterpret_cast<u4*>(tile_b + to[o]) = part[o];
  };
  f4 acc[2][NC];
  clear<FP8, 2, NC>(acc);
  const uint32_t mine = offset_in_rows<FP8>(K);
  // The weights of two steps are on their way while one is multiplied; the next step's tokens go out before the latter
  // of them, as loads are waited for in their order.  Two steps' tokens lie in LDS, so that a step has one barrier.
  // (bf16 weights, of twice the bytes a step: one step's)
  constexpr int kSteps = FP8 ? 2 : 1;
  Weights<FP8, STREAM, 2> w[kSteps + 1];
  fetch(0);
  w[0].load(rows, mine, scales, 0, K);
  if constexpr (kSteps == 2) w[1].load(rows, mine, scales, 1, K);  // (past the end: zeros)
  leave(0);
  __syncthreads();
  auto one_step = [&](int b, Weights<FP8, STREAM, 2>& now, Weights<FP8, STREAM, 2>& later) {
    fetch(b + 1);
    later.load(rows, mine, scales, b + kSteps, K);
    if (active) {
      now.settle();
      const uint16_t* tile_b = lds + b % kInLds * kTokenStep<P, NC>;
      f4 sum[2][NC];
      if constexpr (FP8) clear<FP8, 2, NC>(sum);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bf8 f[2] = {now.frag(0, q), now.frag(1, q)};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int p = P - 1; p >= 0; --p) {
            const bf8 x = *reinterpret_cast<const bf8*>(tile_b + (p * NC * 16 + c * 16 + r) * kTokenPitch + k_of<FP8>(q, g));
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              f4& s = FP8 ? sum[m][c] : acc[m][c];
              s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[m], x, s, 0, 0, 0);
            }
          }
      }
      if constexpr (FP8) join_step<FP8, STREAM, 2, NC>(acc, sum, now);
    }
    if constexpr (kInLds == 1) __syncthreads();  // (this step's readers)
    leave(b + 1);
    __syncthreads();
  };
  for (int b = 0; b < KB; b += kSteps + 1) {
    one_step(b, w[0], w[kSteps]);
    if (b + 1 >= KB) break;
    one_step(b + 1, w[1], w[0]);
    if constexpr (kSteps == 2) {
      if (b + 2 >= KB) break;
      one_step(b + 2, w[2], w[1]);
    }
  }
  if (!active) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = c * 16 + r;
    if (i >= n) continue;
    const int at = shared ? first + i : plan.list[first + i];
    leave_rows<DT, UP>(a, shared, at, row0 + 4 * g, both, acc[0][c], acc[1][c]);
  }
}

// The units of a tile are neighbours: those of one expert read its weights at the same time, from the cache.
template <int DT, bool FP8, bool UP, bool STREAM, int UNIT>
__global__ __launch_bounds__(64 * kTileWaves, UNIT > kUnitTokens ? 2 : FP8 && UP && DT == CIN_DT_BF16 ? 4 : 3) void k_products(LayerArgs a) {
  constexpr int ROWS = kTileRows<UP>;
  __shared__ TilePlan<UP, UNIT> plan;
  extern __shared__ u4 tokens[];  // [parts, columns][kTokenPitch] of 16 bits
  const int tiles = ((UP ? a.experts.H : a.D) + ROWS - 1) / ROWS, routed = a.units * tiles;
  const bool shared = (int)blockIdx.x >= routed;
  int expert = 0, tile, first, n;
  if (!shared) {
    tile = blockIdx.x / a.units;
    const int u = blockIdx.x - tile * a.units;
    if (!find_unit(a, plan, u, tile == 0, expert, first, n)) return;
  } else {
    const int i = blockIdx.x - routed, units = (a.T + UNIT - 1) / UNIT;
    tile = i / units;
    first = (i - tile * units) * UNIT;
    n = min(a.T - first, UNIT);
  }
  uint16_t* lds = reinterpret_cast<uint16_t*>(tokens);
  if (n <= 16)
    tile_unit<DT, FP8, UP, STREAM, 1>(a, plan, lds, expert, tile, first, n, shared);
  else if (UNIT == 32 || n <= 32)
    tile_unit<DT, FP8, UP, STREAM, 2>(a, plan, lds, expert, tile, first, n, shared);
  else
    tile_unit<DT, FP8, UP, STREAM, UNIT / 16>(a, plan, lds, expert, tile, first, n, shared);
}

// out = the sum of a token's rows of y, in the order of its experts, the shared one's last.
template <int DT>
__global__ __launch_bounds__(256) void k_join(LayerArgs a) {
  const int per = a.D / 4, i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.T * per) return;
  const int t = i / per, d = (i - t * per) * 4;
  const float* y = a.y + (int64_t)t * a.k * a.D + d;
  f4 s = {0.0f, 0.0f, 0.0f, 0.0f}, last = s;
  if (a.shared.H) last = *reinterpret_cast<const f4*>(a.y + (int64_t)(a.T * a.k + t) * a.D + d);
  for (int j = 0; j < a.k; j += 8) {
    f4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const f4*>(y + (int64_t)min(j + i, a.k - 1) * a.D);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < a.k) s += v[i];
  }
  s += last;
  const int64_t o = (int64_t)t * a.D + d;
  if constexpr (DT == CIN_DT_F32) {
    *reinterpret_cast<f4*>(static_cast<float*>(a.out) + o) = s;
  } else {
    const uint2 v = {f32x2_to_half2_bits<DT>(s[0], s[1]), f32x2_to_half2_bits<DT>(s[2], s[3])};
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) = v;
  }
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
constexpr int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Bytes of the workspace; fills its pointers where `base` is given.
int64_t layout(LayerArgs& a, int dtype, char* base) {
  const int64_t px = dtype == CIN_DT_BF16 ? 1 : dtype == CIN_DT_F16 ? 2 : 3, ph = kHParts;
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
  a.y = reinterpret_cast<float*>(take(4LL * a.T * (a.k + 1) * a.D));
  a.plans = reinterpret_cast<UnitPlan*>(take((int64_t)sizeof(UnitPlan) * a.units));
  return at;
}

bool sizes_ok(int dtype, int64_t T, int64_t D, int64_t E, int64_t k, int64_t H, int64_t Hs) {
  return (dtype == CIN_DT_BF16 || dtype == CIN_DT_F16 || dtype == CIN_DT_F32) && T >= 0 && T <= kMaxTokens && D >= 16 &&
         D <= 65536 && D % 16 == 0 && E >= 1 && E <= kMaxExperts && k >= 1 && k <= kMaxTopK && k <= E && H >= 16 && H <= 65536 &&
         H % 16 == 0 && Hs >= 0 && Hs <= 65536 && Hs % 16 == 0;
}
const char* const kSizes =
    "dtype must be bf16, fp16 or fp32, T <= 128, E <= 1024, k <= min(16, E), D, H and the shared expert's H multiples of 16 up to 65536";

// Tokens of a unit.  A second unit of an expert reads its weights again, from the cache at best; more tokens at once
// cost the registers of a third workgroup a CU, and with the parts of an fp32 x the LDS of a second.  8 of 32 experts of
// 7168 x 2048 and a shared one: 80 tokens with units of 32 350 us, of 64 411; 96 408 and 436; 112 458 and 450; 96 tokens, 6
// of 8 experts 284 and 262; 64 tokens, 8 of 16 in bf16 518 and 330; 96 fp32 tokens 520 and 722.
int64_t unit_tokens(int dtype, int64_t T, int64_t E, int64_t k) {
  return dtype != CIN_DT_F32 && T > kUnitTokens && T * k > 24 * E ? 2 * kUnitTokens : kUnitTokens;
}

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
  a.unit = (int)unit_tokens(dtype, T, E, k);
  a.units = (int)((n < E ? n : E) + n / a.unit);
}

// Whether the waves share K: where k_products would have fewer than one and a half workgroups a CU.  One token, 8 of 32
// experts of 7168 x 2048 and a shared one: up, 256 of them, 40 us against 52, down, 504, 35 against 24; 2 of 16 experts of
// 1024 x 1024 and a shared one: up, 32, 5.5 against 9.5, down, 24, 9.8 against 26; 16 tokens of these, 272 and 144: 51
// against 60 a call.
bool splits_k(const LayerArgs& a, bool up) {
  const int64_t rows = up ? kTileRows<true> : kTileRows<false>;
  const int64_t groups = a.units * cdiv(up ? a.experts.H : a.D, rows) + (!up && a.shared.H ? cdiv(a.D, rows) : 0);
  return a.T <= kFewTokens && 2 * groups < 3 * cin_device_cus();
}

template <int DT, bool FP8, bool UP, bool STREAM>
void launch_tiles(const LayerArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int P = UP ? kXParts<DT> : kHParts;
  constexpr size_t lds = 2 * sizeof(uint16_t) * kTokenStep<P, kUnitTokens / 16>;
  if (DT == CIN_DT_F32 || a.unit == kUnitTokens) {
    hipLaunchKernelGGL((k_products<DT, FP8, UP, STREAM, kUnitTokens>), grid, dim3(64 * kTileWaves), lds, stream, a);
    return;
  }
  if constexpr (DT != CIN_DT_F32) {
    constexpr size_t more = lds * kStepsInLds<P, 2 * kUnitTokens / 16>;  // (twice the tokens, in one or two steps)
    auto kernel = k_products<DT, FP8, UP, STREAM, 2 * kUnitTokens>;
    if (more + sizeof(TilePlan<UP, 2 * kUnitTokens>) > 65536)
      (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)more);
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kTileWaves), more, stream, a);
  }
}

// Whether the shared expert's h is formed beside the gate: where its workgroups among the products, which come last and
// are waited for, would leave most CUs idle, and while the tokens' parts that each 16 rows read for themselves are few.
// Gate and up together, 32 experts of 7168 x 2048 and a shared one: one bf16 token 50 us, 52 with it among the products;
// 16 163 and 177; 64 190 and 201; with 64 tokens in fp16 248 and 229, with a shared one of 8192 243 and 225.
template <int DT>
bool early_shared(const LayerArgs& a) {
  return a.T * kXParts<DT> <= 64 && 2 * cdiv(a.shared.H, kTileRows<true>) * cdiv(a.T, a.unit) <= cin_device_cus();
}

template <int DT, bool FP8, bool UP, bool STREAM>
void launch_products(const LayerArgs& a, hipStream_t stream) {
  const bool few = splits_k(a, UP);
  const int64_t rows = few ? kFewRows<UP> : kTileRows<UP>, units = few ? 1 : cdiv(a.T, a.unit);
  const int64_t routed = a.units * cdiv(UP ? a.experts.H : a.D, rows);
  const int64_t shared = a.shared.H && !(UP && early_shared<DT>(a)) ? units * cdiv(UP ? a.shared.H : a.D, rows) : 0;
  const dim3 grid((uint32_t)(routed + shared));
  if (few) {
    hipLaunchKernelGGL((k_few<DT, FP8, UP, STREAM>), grid, dim3(64 * kFewWaves), 0, stream, a);
  } else {
    launch_tiles<DT, FP8, UP, STREAM>(a, grid, stream);
  }
}

// Rows that begin on lines of 128 bytes are streamed: a load takes whole lines, and none need be kept.  Else a line's
// parts are of two steps (17 tokens, rows of 7152 codes: streamed 419 us a call, kept 341; 64 tokens, rows of 7168: 323 and 336).
template <int DT, bool FP8, bool UP>
void launch_products(const LayerArgs& a, bool on_lines, hipStream_t stream) {
  constexpr int line = FP8 ? 128 : 64;
  const bool whole = UP ? a.D % line == 0 : a.experts.H % line == 0 && a.shared.H % line == 0;
  if (on_lines && whole)
    launch_products<DT, FP8, UP, true>(a, stream);
  else
    launch_products<DT, FP8, UP, false>(a, stream);
}

template <int DT, bool FP8, bool STREAM, int NC>
void launch_gate(const LayerArgs& a, hipStream_t stream) {
  const int64_t shared = early_shared<DT>(a) ? cdiv(a.shared.H, kFewRows<true>) * cdiv(a.T, 16 * NC) : 0;
  hipLaunchKernelGGL((k_gate<DT, FP8, STREAM, NC>), dim3((uint32_t)(a.T + shared)), dim3(64 * kGateWaves<NC>), 0, stream, a);
}
template <int DT, bool FP8, bool STREAM>
void launch_gate(const LayerArgs& a, hipStream_t stream) {
  if (a.T <= 16)
    launch_gate<DT, FP8, STREAM, 1>(a, stream);
  else
    launch_gate<DT, FP8, STREAM, 2>(a, stream);
}

template <int DT, bool FP8>
void launch_experts(const LayerArgs& a, hipStream_t stream) {
  const bool on_lines =
      ((uintptr_t)a.experts.w12 | (uintptr_t)a.experts.w3 | (uintptr_t)a.shared.w12 | (uintptr_t)a.shared.w3) % 128 == 0;
  if (on_lines && a.D % (FP8 ? 128 : 64) == 0)
    launch_gate<DT, FP8, true>(a, stream);
  else
    launch_gate<DT, FP8, false>(a, stream);
  launch_products<DT, FP8, true>(a, on_lines, stream);
  launch_products<DT, FP8, false>(a, on_lines, stream);
  hipLaunchKernelGGL((k_join<DT>), dim3((a.T * (a.D / 4) + 255) / 256), dim3(256), 0, stream, a);
}

template <int DT>
void launch(const LayerArgs& a, bool fp8, hipStream_t stream) {
  hipLaunchKernelGGL((k_router<DT>), dim3(a.slices * ((a.E + 15) / 16), (a.T + 15) / 16), dim3(256), 0, stream, a);
  if (fp8)
    launch_experts<DT, true>(a, stream);
  else
    launch_experts<DT, false>(a, stream);
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
