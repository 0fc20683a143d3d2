// Drafted tokens against the target's probabilities on gfx950, from given random numbers: what a step with
// draft heads (the reference trains them, src/layers.py:215-241) does with their tokens.
//
//   position i keeps its token x_i while u_i q_i(x_i) < p_i(x_i); at the first that does not, or past the
//   last draft, with n tokens kept, the token is drawn from
//     rest(v) = max(p_n(v) - q_n(v), 0)  (max(p_n(v), 0) past the last draft, or where no rest is left)
//   as the first v whose sum rest(0) + .. + rest(v) exceeds u_K times the whole sum.
//
// Everything that decides is in 64 bits: the products of two fp32 values are exact there, and on which
// side of a border among 131072 a number falls is lost in 32 (their sum is off by up to 1e-6, a border lies
// within that of the number in one draw of ten), while 64-bit sums in another order move a border by 1e-15.
//
// Two launches.  k_verify_sums: every workgroup finds n from the K products (2 K loads, in two steps), then sums its
// part of row n.  k_verify_pick: a workgroup a sequence finds the part in which the number falls, reads it
// again and finds the token.  Of the K + 1 rows of a sequence only one is read: the bytes are one row of
// p and one of q.  64 sequences of 131072 fp32 probabilities: 14 us (67 MB, 4.9 TB/s) and 7, four dependent reads;
// one sequence of 32000 4 and 6, latency.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cin_common.h"
#include "cin_runtime.h"

using namespace cin;

namespace {

constexpr int kSumThreads = 256;
constexpr int kPickThreads = 512;
constexpr int kMaxDrafts = 64;    // a wave decides
constexpr int kMaxParts = 1024;   // of a row
constexpr int kLeastPart = 2048;  // channels: 8 a thread

struct VerifyArgs {
  const int64_t* tokens;
  int64_t stb, stk;
  const void *q, *p;
  int64_t sqb, sqk, spb, spk;
  const void* u;
  int u64;
  int64_t sub, suk;
  const int64_t* counts;
  int64_t scb;
  int64_t B, V, part;
  int K, parts;
  double* sums;  // [B, parts, 2]: of rest and of max(p, 0)
  int* kept;     // [B]
  int64_t *out, *accepted;
};

__device__ inline double uniform(const VerifyArgs& a, int64_t b, int64_t i) {
  const int64_t at = b * a.sub + i * a.suk;
  return a.u64 ? static_cast<const double*>(a.u)[at] : (double)static_cast<const float*>(a.u)[at];
}

__device__ inline int limit_of(const VerifyArgs& a, int64_t b) {
  if (!a.counts) return a.K;
  const int64_t n = a.counts[b * a.scb];
  return n < 0 ? 0 : n > a.K ? a.K : (int)n;
}

// Tokens kept of sequence b: the lanes take a position each.
template <int DT>
__device__ inline int kept_of(const VerifyArgs& a, int64_t b) {
  const int i = threadIdx.x & 63;
  bool ok = false;
  if (i < limit_of(a, b)) {
    const int64_t x = a.tokens[b * a.stb + i * a.stk];
    if (x >= 0 && x < a.V) {
      const double p = (double)load_elem(a.p, DT, b * a.spb + i * a.spk + x);
      const double q = a.q ? (double)load_elem(a.q, DT, b * a.sqb + i * a.sqk + x) : 1.0;
      ok = uniform(a, b, i) * q < p;
    }
  }
  return (int)__builtin_ctzll(~__ballot(ok) | (1ull << 63));
}

// The row that the new token is drawn from.
template <int DT>
struct Row {
  const uint8_t *p, *q;  // q null past the last draft, and for drafts without probabilities
  int64_t without;       // the token that has all of the draft's probability, or -1
  __device__ Row(const VerifyArgs& a, int64_t b, int n) {
    constexpr int es = DT == CIN_DT_F32 ? 4 : 2;
    p = static_cast<const uint8_t*>(a.p) + (b * a.spb + n * a.spk) * es;
    const bool drafted = n < limit_of(a, b);
    q = drafted && a.q ? static_cast<const uint8_t*>(a.q) + (b * a.sqb + n * a.sqk) * es : nullptr;
    without = drafted && !a.q ? a.tokens[b * a.stb + n * a.stk] : -1;
  }
  // rest and max(p, 0) of 8 neighbours, of which cnt are there; NaN stays NaN
  __device__ __forceinline__ void get(int64_t v, int cnt, double (&rest)[8], double (&whole)[8]) const {
    float pv[8], qv[8];
    load(p, v, cnt, pv);
    if (q) {
      load(q, v, cnt, qv);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) qv[e] = v + e == without ? 1.0f : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double w = (double)pv[e], d = w - (double)qv[e];
      whole[e] = w < 0 ? 0.0 : w;
      rest[e] = d < 0 || (v + e == without && d == d) ? 0.0 : d;
    }
  }
  static __device__ __forceinline__ void load(const uint8_t* row, int64_t v, int cnt, float (&f)[8]) {
    if constexpr (DT == CIN_DT_F32) {
      if (cnt == 8) {
        __builtin_memcpy(f, row + v * 4, 32);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < cnt ? reinterpret_cast<const float*>(row)[v + e] : 0.0f;
      }
    } else {
      uint16_t h[8];
      if (cnt == 8) {
        __builtin_memcpy(h, row + v * 2, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = e < cnt ? reinterpret_cast<const uint16_t*>(row)[v + e] : (uint16_t)0;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = half_bits_to_f32(DT, h[e]);
    }
  }
};

__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

template <int DT>
__global__ __launch_bounds__(kSumThreads) void k_verify_sums(VerifyArgs a) {
  const int64_t b = blockIdx.x / a.parts;
  const int c = (int)(blockIdx.x - b * a.parts);
  const int n = kept_of<DT>(a, b);
  const Row<DT> row(a, b, n);
  const int64_t end = min((int64_t)(c + 1) * a.part, a.V);
  double s[2] = {0.0, 0.0};
  for (int64_t v = (int64_t)c * a.part + threadIdx.x * 8; v < end; v += kSumThreads * 8) {
    double rest[8], whole[8];
    row.get(v, (int)min(end - v, (int64_t)8), rest, whole);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[0] += rest[e];
      s[1] += whole[e];
    }
  }
  __shared__ double lds[2][kSumThreads / 64];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const double t = wave_sum(s[k]);
    if ((threadIdx.x & 63) == 0) lds[k][threadIdx.x >> 6] = t;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double t = 0.0;
    for (int w = 0; w < kSumThreads / 64; ++w) t += lds[threadIdx.x][w];
    a.sums[(b * a.parts + c) * 2 + threadIdx.x] = t;
  }
  if (c == 0 && threadIdx.x == 0) a.kept[b] = n;
}

// Sum of v over the threads before this one; `total` of all.  Ends with every thread past its reads of lds.
__device__ inline double before(double v, double& total, double* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(s, o);
    if (lane >= o) s += t;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  double base = 0.0, all = 0.0;
  for (int w = 0; w < kPickThreads / 64; ++w) {
    if (w < wave) base += lds[w];
    all += lds[w];
  }
  total = all;
  __syncthreads();
  return base + (s - v);
}

__device__ inline int block_min(int v, int* lds) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = min(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  int m = lds[0];
  for (int w = 1; w < kPickThreads / 64; ++w) m = min(m, lds[w]);
  __syncthreads();
  return m;
}

template <int DT>
__global__ __launch_bounds__(kPickThreads) void k_verify_pick(VerifyArgs a) {
  __shared__ double lds[kPickThreads / 64];
  __shared__ int ids[kPickThreads / 64];
  __shared__ double found_base;
  constexpr int kNone = 0x7fffffff;
  const int64_t b = blockIdx.x;
  const int n = a.kept[b];
  const Row<DT> row(a, b, n);
  constexpr int kOwn = kMaxParts / kPickThreads;  // parts of a thread
  double part[2][kOwn], mine[2] = {0.0, 0.0};
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int c = (int)threadIdx.x * kOwn + k;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      part[w][k] = c < a.parts ? a.sums[(b * a.parts + c) * 2 + w] : 0.0;
      mine[w] += part[w][k];
    }
  }
  double total[2], base[2];
  base[0] = before(mine[0], total[0], lds);
  base[1] = before(mine[1], total[1], lds);
  const int which = total[0] == 0.0 ? 1 : 0;  // nothing of p lies above q: all of p
  const double target = uniform(a, b, a.K) * total[which];
  int64_t token = -1;
  if (total[which] > 0.0 && total[which] < __builtin_inf()) {
    // the part: the first with a sum that passes the target; if rounding leaves none, the last with any
    int first = kNone, last = kNone;
    double s = base[which], first_base = 0.0, last_base = 0.0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int c = (int)threadIdx.x * kOwn + k;
      if (part[which][k] > 0.0) {
        last = -c;
        last_base = s;
        if (first == kNone && s + part[which][k] > target) {
          first = c;
          first_base = s;
        }
      }
      s += part[which][k];
    }
    int c = block_min(first, ids);
    if (c != kNone) {
      if (first == c) found_base = first_base;
    } else {
      c = -block_min(last, ids);
      if (last == -c) found_base = last_base;
    }
    __syncthreads();
    double sum = found_base;
    const int64_t end = min((int64_t)(c + 1) * a.part, a.V);
    int64_t last_any = -1;
    for (int64_t at = (int64_t)c * a.part; at < end && token < 0; at += kPickThreads * 8) {
      const int64_t v = at + threadIdx.x * 8;
      double rest[8], whole[8], own = 0.0;
      const int cnt = (int)max((int64_t)0, min(end - v, (int64_t)8));
      row.get(cnt > 0 ? v : at, cnt, rest, whole);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (which) rest[e] = whole[e];
        if (e >= cnt) rest[e] = 0.0;
        own += rest[e];
      }
      double all;
      double run = sum + before(own, all, lds);
      int hit = kNone, any = kNone;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        run += rest[e];
        if (rest[e] > 0.0) {
          any = -(int)(v + e - at);
          if (hit == kNone && run > target) hit = (int)(v + e - at);
        }
      }
      hit = block_min(hit, ids);
      any = block_min(any, ids);
      if (hit != kNone) token = at + hit;
      if (any != kNone) last_any = at - any;
      sum += all;
    }
    if (token < 0) token = last_any;
  }
  if (threadIdx.x <= a.K) {
    const int i = threadIdx.x;
    a.out[b * (a.K + 1) + i] = i < n ? a.tokens[b * a.stb + i * a.stk] : i == n ? token : -1;
  }
  if (threadIdx.x == 0) a.accepted[b] = n;
}

// Channels of a part: about eight workgroups a CU, whole steps of a workgroup.
int64_t part_of(int64_t B, int64_t V) {
  const int64_t want = cdiv(B * V, (int64_t)cin_device_cus() * 8);
  const int64_t least = cdiv(V, kMaxParts);
  const int64_t most = 4 * kLeastPart;
  int64_t part = want < kLeastPart ? kLeastPart : want > most ? most : want;
  if (part < least) part = least;
  return cdiv(part, kLeastPart) * kLeastPart;
}

template <int DT>
void launch(const VerifyArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((k_verify_sums<DT>), dim3((uint32_t)(a.B * a.parts)), dim3(kSumThreads), 0, stream, a);
  hipLaunchKernelGGL((k_verify_pick<DT>), dim3((uint32_t)a.B), dim3(kPickThreads), 0, stream, a);
}

bool sizes_ok(int64_t B, int64_t K, int64_t V) {
  return B >= 0 && B <= 65536 && K >= 0 && K < kMaxDrafts && V >= 1 && V < (1LL << 30) &&
         B * cdiv(V, part_of(B, V)) < (1LL << 32) / kSumThreads;  // threads of a launch
}
const char* const kSizes = "B must be in [0, 65536], K in [0, 63], V in [1, 2^30) and B V below 2^37";

}  // namespace

extern "C" {

int64_t cin_verify_drafts_workspace(int64_t B, int64_t K, int64_t V) {
  if (!sizes_ok(B, K, V)) {
    cin_set_error(CIN_ERR_ARG, "cin_verify_drafts_workspace: %s", kSizes);
    return -1;
  }
  return B * (16 * cdiv(V, part_of(B, V)) + 8);
}

int cin_verify_drafts(const int64_t* tokens, int64_t stb, int64_t stk, const void* q, int64_t sqb, int64_t sqk, const void* p,
                      int64_t spb, int64_t spk, int dtype, int64_t B, int64_t K, int64_t V, const void* u, int u_double,
                      int64_t sub, int64_t suk, const int64_t* counts, int64_t scb, int64_t* out, int64_t* accepted,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  CIN_CHECK_ARG(dtype == CIN_DT_BF16 || dtype == CIN_DT_F16 || dtype == CIN_DT_F32, "cin_verify_drafts: dtype must be bf16, fp16 or fp32");
  CIN_CHECK_ARG(sizes_ok(B, K, V), "cin_verify_drafts: %s", kSizes);
  if (B == 0) return CIN_OK;
  CIN_CHECK_ARG((tokens || K == 0) && p && u && out && accepted && workspace, "cin_verify_drafts: null pointer");
  CIN_CHECK_ARG((uintptr_t)workspace % 16 == 0 && workspace_bytes >= cin_verify_drafts_workspace(B, K, V),
                "cin_verify_drafts: workspace below cin_verify_drafts_workspace bytes or not on 16");
  VerifyArgs a = {};
  a.tokens = tokens;
  a.stb = stb;
  a.stk = stk;
  a.q = q;
  a.p = p;
  a.sqb = sqb;
  a.sqk = sqk;
  a.spb = spb;
  a.spk = spk;
  a.u = u;
  a.u64 = u_double;
  a.sub = sub;
  a.suk = suk;
  a.counts = counts;
  a.scb = scb;
  a.B = B;
  a.V = V;
  a.K = (int)K;
  a.part = part_of(B, V);
  a.parts = (int)cdiv(V, a.part);
  a.sums = static_cast<double*>(workspace);
  a.kept = reinterpret_cast<int*>(a.sums + 2 * B * a.parts);
  a.out = out;
  a.accepted = accepted;
  if (dtype == CIN_DT_BF16)
    launch<CIN_DT_BF16>(a, (hipStream_t)stream);
  else if (dtype == CIN_DT_F16)
    launch<CIN_DT_F16>(a, (hipStream_t)stream);
  else
    launch<CIN_DT_F32>(a, (hipStream_t)stream);
  return cin_check_launch("cin_verify_drafts");
}

}  // extern "C"
