// Rotary positions on gfx950: pairs of channels of queries and keys turned by the angle of their
// position (reference src/attention.py:9-128).
//
//   y0 = x0 cos - x1 sin      pairs (2i, 2i + 1) of the rotated channels, or (i, i + rot / 2)
//   y1 = x0 sin + x1 cos      with cos and sin [P, rot / 2] read at the token's position
//
// Channels outside [start, start + rot) are copied.  inverse turns back (-sin): the gradient.
// A token at a negative position is copied as it is (padding), one past the table gives NaN.
// Products and the sum are fp32, each output rounded once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "cin_common.h"
#include "cin_runtime.h"

using namespace cin;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxUnits = 2;
constexpr uint32_t kMagicLimit = 60000;      // (kThreads kMaxUnits + d) d < 2^32: see div_by

// Units a thread, their loads in flight together.  One is as fast for 16-byte units of 16-bit elements or
// faster (64 x 1024 x 17 heads of 64: 54 us, with two 58; 16 x 1024: 14.9 and 15.5; 1 x 32767 x 32 heads of 192
// in the half layout: 169 and 177, interleaved 179 and 177; of 193: 244 and 251); two for single channels (842
// and 785) and, by a little, for fp32 (1 x 32767 x 32 heads of 192: interleaved 350 and 331, half layout 314 and
// 320, of 193 416 and 406; 64 x 1024 x 17 heads of 64: 112 and 117).  Four needed half as many registers again.
template <int DT, int E>
constexpr int kUnitsOf = DT != CIN_DT_F32 && E > 1 ? 1 : kMaxUnits;

// One of the two tensors, [B, L, heads, D] with unit channel stride.
struct Side {
  const void* x;
  void* y;
  int64_t xb, xl, xh, yb, yl, yh;
};

struct RotaryArgs {
  Side q, k;
  int qheads;
  int64_t n, L;            // units in all, tokens of a sequence
  int64_t base;            // workgroups of the launches before this one
  const float *cos, *sin;
  int64_t P, ldt;
  int rot, start, turned;  // units of a head that turn: the first ones
  int before, after;       // channels copied before and after them
  uint32_t units, row;     // units of a head, of a token's heads
  uint32_t munits, mrow;   // ceil(2^32 / d) of the two, 0 for plain division
  uint64_t wrow, wL;       // ceil(2^64 / d) of row and L
  const int64_t* positions;
  int64_t pb, pl;
  int interleaved, inverse;
};

// i / d by m = ceil(2^32 / d) = (2^32 + e) / d, e < d: exact while i e < 2^32.
__device__ __forceinline__ uint32_t div_by(uint32_t i, uint32_t d, uint32_t m) {
  return d == 1 ? i : (m ? __umulhi(i, m) : i / d);
}

// The same in 64 bits, exact while i d < 2^64.
__device__ __forceinline__ int64_t div_by(int64_t i, int64_t d, uint64_t m) {
  return d == 1 ? i : (int64_t)__umul64hi((uint64_t)i, m);
}

template <int DT>
constexpr int kEs = DT == CIN_DT_F32 ? 4 : 2;

// E adjacent elements as they lie in memory: 16 bytes at any element's address, or one.
template <int DT, int E>
struct Chunk {
  uint32_t w[E > 1 ? 4 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (E > 1)
      __builtin_memcpy(w, static_cast<const uint8_t*>(p) + i * kEs<DT>, 16);
    else if constexpr (DT == CIN_DT_F32)
      w[0] = static_cast<const uint32_t*>(p)[i];
    else
      w[0] = static_cast<const uint16_t*>(p)[i];
  }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    if constexpr (E > 1)
      __builtin_memcpy(static_cast<uint8_t*>(p) + i * kEs<DT>, w, 16);
    else if constexpr (DT == CIN_DT_F32)
      static_cast<uint32_t*>(p)[i] = w[0];
    else
      static_cast<uint16_t*>(p)[i] = (uint16_t)w[0];
  }
  __device__ __forceinline__ void widen(float (&v)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (DT == CIN_DT_F32)
        v[e] = __uint_as_float(w[e]);
      else
        v[e] = half_bits_to_f32(DT, (uint16_t)(w[e / 2] >> (16 * (e & 1))));
    }
  }
  __device__ __forceinline__ void round(const float (&v)[E]) {
    if constexpr (DT == CIN_DT_F32) {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = __float_as_uint(v[e]);
    } else if constexpr (E == 1) {
      w[0] = f32_to_half_bits(DT, v[0]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = f32x2_to_half2_bits<DT>(v[2 * e], v[2 * e + 1]);
    }
  }
};

// N neighbours of a table's row, which start on their own size (up to 16 bytes).
template <int N>
__device__ __forceinline__ void load_pairs(const float* p, float (&v)[N]) {
  __builtin_memcpy(v, __builtin_assume_aligned(p, N >= 4 ? 16 : 4 * N), 4 * N);
}

// A unit is 16 bytes of a head's channels (E elements) or one channel (E = 1), and where it turns
// whole pairs: with the half layout the unit rot / 2 further comes with it, and single interleaved
// channels come in twos.  The last 16 bytes of the copied channels before or after the turning ones
// may overlap the ones in front of them (the same values twice); fewer go one by one.
// Bound by HBM: each element is read and written once; the tables' rows are shared by a token's heads
// through the caches.  A workgroup takes neighbouring units; their token, head, channel and offsets
// follow from the first one's in 32 bits (with 64-bit divisions and products the vector units bound it:
// 1 x 32767 x 32 heads of 192, fp16, half layout, 355 us).  That call now takes 169 us, 4.8 TB/s, its
// interleaved form 179 (4.5), 64 x 1024 x 17 heads of 64 in bf16 54 us, 5.3 TB/s.  Stores that bypass
// the caches took a quarter less there, and the next reader of the result as much more.
template <int DT, int E, bool INTER>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs a) {
  constexpr int kPairs = INTER ? (E > 1 ? E / 2 : 1) : E;  // pairs of a turning unit
  constexpr bool kTwo = !INTER || E == 1;                  // ... which lie in two chunks
  constexpr int kUnits = kUnitsOf<DT, E>;
  const int64_t first = (a.base + blockIdx.x) * (kThreads * kUnits);
  const int64_t tok0 = div_by(first, (int64_t)a.row, a.wrow);
  const uint32_t rem0 = (uint32_t)(first - tok0 * a.row);
  const int64_t b0 = div_by(tok0, a.L, a.wL), l0 = tok0 - b0 * a.L;
  const int64_t left = a.L - l0;  // tokens of this sequence
  const int64_t inq = b0 * a.q.xb + l0 * a.q.xl, ink = b0 * a.k.xb + l0 * a.k.xl;
  const int64_t outq = b0 * a.q.yb + l0 * a.q.yl, outk = b0 * a.k.yb + l0 * a.k.yl;
  Chunk<DT, E> c0[kUnits], c1[kUnits];
  int64_t out[kUnits];
  int at0[kUnits], at1[kUnits];
  float cs[kUnits][kPairs], sn[kUnits][kPairs];
  bool live[kUnits], turns[kUnits], second[kUnits], still[kUnits];  // still: padding, kept bit for bit
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    const uint32_t local = j * kThreads + threadIdx.x;
    live[j] = first + local < a.n;
    turns[j] = still[j] = false;
    if (!live[j]) continue;
    const uint32_t i = rem0 + local, dt = div_by(i, a.row, a.mrow), r = i - dt * a.row;
    const uint32_t h = div_by(r, a.units, a.munits), u = r - h * a.units;
    const bool of_k = (int)h >= a.qheads;
    const int hh = of_k ? (int)h - a.qheads : (int)h;
    // (the host checks that token and head strides fit in 32 bits: one multiply-add each)
    auto at = [&](int64_t base, int64_t qs, int64_t ks, int i) { return base + (int64_t)(int)(of_k ? ks : qs) * i; };
    int64_t in = at(at(of_k ? ink : inq, a.q.xl, a.k.xl, (int)dt), a.q.xh, a.k.xh, hh);
    out[j] = at(at(of_k ? outk : outq, a.q.yl, a.k.yl, (int)dt), a.q.yh, a.k.yh, hh);
    int64_t pos = (int64_t)dt * a.pl, l = l0 + dt;
    if (dt >= left) {  // in a following sequence
      const int64_t more = div_by(l, a.L, a.wL), back = more * a.L;
      l -= back;
      in += more * (of_k ? a.k.xb : a.q.xb) - back * (of_k ? a.k.xl : a.q.xl);
      out[j] += more * (of_k ? a.k.yb : a.q.yb) - back * (of_k ? a.k.yl : a.q.yl);
      pos += more * a.pb - back * a.pl;
    }
    const void* x = of_k ? a.k.x : a.q.x;
    second[j] = of_k;
    turns[j] = (int)u < a.turned;
    if (turns[j]) {
      at0[j] = a.start + (int)u * (INTER && E == 1 ? 2 : E);
    } else {
      int c = ((int)u - a.turned) * E, lo = 0, n = a.before;
      if (c >= n) {
        c -= (n + E - 1) / E * E;
        lo = a.start + a.rot;
        n = a.after;
      }
      at0[j] = lo + (c + E <= n ? c : n - E);
      if (n < E) {
        Chunk<DT, 1> one[E];
#pragma unroll
        for (int e = 0; e + 1 < E; ++e)
          if (e < n) one[e].load(x, in + lo + e);
#pragma unroll
        for (int e = 0; e + 1 < E; ++e)
          if (e < n) one[e].store(of_k ? a.k.y : a.q.y, out[j] + lo + e);
        live[j] = false;
        continue;
      }
    }
    at1[j] = at0[j] + (INTER ? 1 : a.rot / 2);
    c0[j].load(x, in + at0[j]);
    if (!turns[j]) continue;
    if constexpr (kTwo) c1[j].load(x, in + at1[j]);
    const int64_t p = a.positions ? a.positions[b0 * a.pb + l0 * a.pl + pos] : l;
    still[j] = p < 0;
    if (p >= 0 && p < a.P) {
      load_pairs(a.cos + p * a.ldt + (int)u * kPairs, cs[j]);
      load_pairs(a.sin + p * a.ldt + (int)u * kPairs, sn[j]);
    } else {
#pragma unroll
      for (int e = 0; e < kPairs; ++e) cs[j][e] = sn[j][e] = __builtin_nanf("");
    }
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    if (!live[j]) continue;
    void* y = second[j] ? a.k.y : a.q.y;
    if (turns[j] && !still[j]) {
      float v0[E], v1[E];
      c0[j].widen(v0);
      if constexpr (kTwo) c1[j].widen(v1);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        const float s = a.inverse ? -sn[j][e] : sn[j][e];
        float& x0 = kTwo ? v0[e] : v0[2 * e];
        float& x1 = kTwo ? v1[e] : v0[(2 * e + 1) % E];
        const float y0 = x0 * cs[j][e] - x1 * s, y1 = x0 * s + x1 * cs[j][e];
        x0 = y0;
        x1 = y1;
      }
      c0[j].round(v0);
      if constexpr (kTwo) c1[j].round(v1);
    }
    if constexpr (kTwo) {
      if (turns[j]) c1[j].store(y, out[j] + at1[j]);
    }
    c0[j].store(y, out[j] + at0[j]);
  }
}

}  // namespace

extern "C" {

int cin_rotary(const void* q, int64_t sqb, int64_t sql, int64_t sqh, void* q_out, int64_t soqb, int64_t soql,
               int64_t soqh, int64_t H, const void* k, int64_t skb, int64_t skl, int64_t skh, void* k_out,
               int64_t sokb, int64_t sokl, int64_t sokh, int64_t Hk, int dtype, int64_t B, int64_t L, int64_t D,
               const float* cos, const float* sin, int64_t P, int64_t ldt, int64_t rot, int64_t start,
               const int64_t* positions, int64_t spb, int64_t spl, int interleaved, int inverse, void* stream) {
  CIN_CHECK_ARG(dtype == CIN_DT_BF16 || dtype == CIN_DT_F32 || dtype == CIN_DT_F16, "rotary: bad dtype %d", dtype);
  CIN_CHECK_ARG(B >= 0 && L >= 0 && H >= 0 && Hk >= 0 && D >= 1 && P >= 0, "rotary: negative size");
  CIN_CHECK_ARG(rot >= 2 && rot % 2 == 0 && start >= 0 && rot <= D && start <= D - rot && D < (1 << 20),
                "rotary: the rotated channels [start, start + rot) must be pairs within the head");
  CIN_CHECK_ARG(ldt >= rot / 2, "rotary: table rows overlap");
  CIN_CHECK_ARG(positions || L <= P, "rotary: L = %lld positions, the tables hold %lld", (long long)L, (long long)P);
  const int64_t heads = H + Hk;
  if (B == 0 || L == 0 || heads == 0) return CIN_OK;
  CIN_CHECK_ARG((H == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)) && (P == 0 || (cos && sin)),
                "rotary: null pointer");
  CIN_CHECK_ARG((double)B * L * heads * D < 9e15, "rotary: too many elements");
  const int es = dtype == CIN_DT_F32 ? 4 : 2;
  RotaryArgs a{{q, q_out, sqb, sql, sqh, soqb, soql, soqh}, {k, k_out, skb, skl, skh, sokb, sokl, sokh}, (int)H, 0, L, 0, cos, sin,
               P, ldt, (int)rot, (int)start, 0, 0, 0, 0, 0, 0, 0, 0, 0, positions, spb, spl, interleaved, inverse};
  // 16 bytes at a time where they hold turning or copied channels only, whatever their alignment:
  // 1 x 32767 x 32 heads, fp16, rot 64: 169 us with heads of 192 channels, 244 with 193 (one
  // channel at a time 785).
  const int64_t e16 = 16 / es;
  const bool odd = (interleaved ? rot : rot / 2) % e16 || ((uintptr_t)cos | (uintptr_t)sin) % 16 || ldt % 4;
  const int64_t E = odd ? 1 : e16;
  a.before = (int)start;
  a.after = (int)(D - rot - start);
  const int64_t turned = interleaved ? rot / (E > 1 ? E : 2) : rot / 2 / E, units = turned + cdiv(a.before, E) + cdiv(a.after, E);
  CIN_CHECK_ARG(heads * units < ((int64_t)1 << 30), "rotary: too many elements in a token");
  a.turned = (int)turned;
  a.units = (uint32_t)units;
  a.row = (uint32_t)(heads * units);
  a.n = B * L * heads * units;
  auto magic = [](uint32_t d) { return d < kMagicLimit ? (uint32_t)((((uint64_t)1 << 32) + d - 1) / d) : 0u; };
  a.munits = a.row < kMagicLimit ? magic(a.units) : 0;
  a.mrow = magic(a.row);
  auto magic64 = [](uint64_t d) { return d < 2 ? 0ull : ~0ull / d + 1; };
  a.wrow = magic64(a.row);
  a.wL = magic64((uint64_t)L);
  CIN_CHECK_ARG((double)a.n * a.row < 9e18 && (double)B * L * L < 9e18,
                "rotary: too many elements");
  for (int64_t st : {sql, sqh, soql, soqh, skl, skh, sokl, sokh})
    CIN_CHECK_ARG(st < ((int64_t)1 << 31) && st > -((int64_t)1 << 31), "rotary: token and head strides must fit in 32 bits");
  // (a launch has fewer than 2^32 threads)
  constexpr int64_t kMost = (int64_t)1 << 23;
  auto go = [&](auto dt, auto e) {
    const int64_t blocks = cdiv(a.n, kThreads * kUnitsOf<dt(), e()>);
    for (a.base = 0; a.base < blocks; a.base += kMost) {
      const unsigned grid = (unsigned)(blocks - a.base < kMost ? blocks - a.base : kMost);
      if (interleaved)
        hipLaunchKernelGGL((k_rotary<dt(), e(), true>), grid, kThreads, 0, static_cast<hipStream_t>(stream), a);
      else
        hipLaunchKernelGGL((k_rotary<dt(), e(), false>), grid, kThreads, 0, static_cast<hipStream_t>(stream), a);
    }
  };
  auto with_e = [&](auto dt) {
    if (E > 1)
      go(dt, std::integral_constant<int, 16 / kEs<dt()>>{});
    else
      go(dt, std::integral_constant<int, 1>{});
  };
  if (dtype == CIN_DT_F32)
    with_e(std::integral_constant<int, CIN_DT_F32>{});
  else if (dtype == CIN_DT_F16)
    with_e(std::integral_constant<int, CIN_DT_F16>{});
  else
    with_e(std::integral_constant<int, CIN_DT_BF16>{});
  return cin_check_launch("rotary");
}

}  // extern "C"
