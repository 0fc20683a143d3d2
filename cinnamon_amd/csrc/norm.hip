// The norms around a block with its gate and residual scale on gfx950 (reference src/norm.py:15-17 and the
// residual sums of src/layers.py:202), forward and backward.
//
//   u  = y / rms(y) * pw        rms(v) = sqrt(mean(v^2) + eps) over a row's D channels (u = y without pw)
//   x  = a r + g u              the new residual stream: a a number, one learned value or one a channel,
//                               g none, one a channel, one a row or one an element
//   n  = x / rms(x) * w         what the next block reads
// backward, with gn and gx the gradients of n and x, i = 1 / rms(x) and j = 1 / rms(y):
//   t  = gn w;   dx = gx + i (t - x i^2 mean(t x));   dr = a dx;   du = g dx
//   s  = du pw;  dy = j (s - y j^2 mean(s y))         (dy = du without pw)
//   dw = sum gn x i,  dpw = sum du y j,  dg = dx u,  da = dx r over the rows, a row or an element
// A gate per channel only meets pw as the product g pw, and both have their gradient from one sum over the rows:
// S = sum dx y j;  dpw = g S,  dg = pw S.
//
// x is formed again from y and r in the backward, in fp32 as in the forward: that reads as many bytes as
// a stored x and has no rounding to x's type in it.  Arithmetic and sums are fp32, the sum over all channels and rows for a
// learned scale of one value fp64; each output is rounded once.
//
// A row is read once into registers, 8 channels a thread and chunk, by one wave (up to 1024 channels, the
// sums by DPP and swaps, no barrier) or by one workgroup.  Workgroups walk over rows, so that the channels'
// vectors are loaded once (the backward past 8192 channels reads them again, from L2) and a channel's sums over the rows stay
// in registers; each workgroup leaves one row of partial sums, which k_norm_columns adds up in a fixed order.
// Bound by HBM.  16384 rows, bf16 with post norm, a gate a channel and a learned scale, forward and backward: 7168 channels
// 178-187 us (0.94 GB, 5.0-5.3 TB/s) and 297-316 (1.41 GB, 4.5-4.7), 4096 121 (4.5) and 172 (4.7), 2048 53 (5.1) and 100 (4.0);
// bf16 with an fp32 stream, 1024 channels 34 (0.20 GB, 5.9) and 54 (0.30 GB, 5.6).  fp16 with a gate an element, 4999 rows: 1112
// channels 22 (56 MB, 2.5) and 46 (89 MB, 1.9); 1111, whose rows lie on no 16 bytes, 22-27 and 50-61.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cin_common.h"
#include "cin_runtime.h"

using namespace cin;

namespace {

constexpr int kMaxThreads = 512;
constexpr int kWideThreads = 1024;  // of the backward past 8192 channels
constexpr int64_t kMaxWidth = kWideThreads * 2 * 8;
constexpr int kWaveRows = 4;  // rows at a time of a workgroup whose waves take a row each

enum Gate { kNoGate = 0, kChannel = 1, kRow = 2, kElement = 3 };
enum Scale { kNumber = 0, kOneValue = 1, kPerChannel = 2 };
enum Sum { kSumW = 0, kSumU = 1, kSumScale = 2, kSums = 3 };

struct Vec {  // a vector over the channels
  const void* p;
  int dtype;
};

struct NormArgs {
  const void *y, *r;
  int64_t ldy, ldr;
  int64_t T;
  int D, threads;  // threads of a row
  Vec w, pw, gate, scale;
  int gate_kind, scale_kind;
  int64_t ldg;
  float scale_value, eps;
  void *n, *x;
  float* stats;  // [2, T]: 1 / rms(x), 1 / rms(y)
  // backward
  const void *gn, *gx;
  int64_t ldgn, ldgx;
  void *dy, *dr, *dgate;
  float* partial;  // [kSums, workgroups, D], then one double a workgroup for the learned scale
};

template <int DT>
constexpr int kWords = DT == CIN_DT_F32 ? 8 : 4;

// A row of a matrix, the same for all lanes: loads and stores then take a 32-bit offset a lane.
template <int DT>
__device__ __forceinline__ const uint8_t* row_at(const void* p, int64_t row, int64_t ld) {
  return static_cast<const uint8_t*>(p) + row * ld * (DT == CIN_DT_F32 ? 4 : 2);
}

// 8 adjacent elements as they lie in memory, at any element's address; cnt of them are there.
template <int DT>
struct Unit {
  uint32_t w[kWords<DT>];
  static constexpr int kEs = DT == CIN_DT_F32 ? 4 : 2;
  __device__ __forceinline__ void load(const uint8_t* row, uint32_t at) {
    const uint8_t* q = row + at * kEs;
    __builtin_memcpy(w, q, 16);
    if constexpr (DT == CIN_DT_F32) __builtin_memcpy(w + 4, q + 16, 16);
  }
  __device__ __forceinline__ void load(const uint8_t* row, uint32_t at, int cnt) {
    if (__builtin_expect(cnt == 8, 1)) return load(row, at);
    zero();
    // the rest as 4, 2 and 1 elements
    const uint8_t* q = row + at * kEs;
    if constexpr (DT == CIN_DT_F32) {
      uint4 four = {0, 0, 0, 0};
      uint2 two = {0, 0};
      uint32_t one = 0;
      if (cnt & 4) __builtin_memcpy(&four, q, 16);
      if (cnt & 2) __builtin_memcpy(&two, q + (cnt & 4) * 4, 8);
      if (cnt & 1) __builtin_memcpy(&one, q + (cnt & 6) * 4, 4);
      const uint32_t a = cnt & 2 ? two.x : one, b = cnt & 2 ? two.y : 0u, c = cnt & 2 ? one : 0u;
      const bool low = !(cnt & 4);
      w[0] = low ? a : four.x;
      w[1] = low ? b : four.y;
      w[2] = low ? c : four.z;
      w[3] = four.w;
      w[4] = low ? 0u : a;
      w[5] = low ? 0u : b;
      w[6] = low ? 0u : c;
      w[7] = 0u;
    } else {
      uint2 four = {0, 0};
      uint32_t two = 0;
      uint16_t one = 0;
      if (cnt & 4) __builtin_memcpy(&four, q, 8);
      if (cnt & 2) __builtin_memcpy(&two, q + (cnt & 4) * 2, 4);
      if (cnt & 1) __builtin_memcpy(&one, q + (cnt & 6) * 2, 2);
      const uint32_t a = cnt & 2 ? two : one, b = cnt & 2 ? one : 0u;
      const bool low = !(cnt & 4);
      w[0] = low ? a : four.x;
      w[1] = low ? b : four.y;
      w[2] = low ? 0u : a;
      w[3] = low ? 0u : b;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < kWords<DT>; ++k) w[k] = 0;
  }
  // What was widened before is widened again, instead of staying in twice the registers.
  __device__ __forceinline__ void forget() {
    if constexpr (DT != CIN_DT_F32) {
#pragma unroll
      for (int k = 0; k < kWords<DT>; ++k) asm volatile("" : "+v"(w[k]));
    }
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (DT == CIN_DT_F32) return __uint_as_float(w[e]);
    return half_bits_to_f32(DT, (uint16_t)(w[e / 2] >> (16 * (e & 1))));
  }
};

template <int DT>
__device__ __forceinline__ void store_unit(const uint8_t* row, uint32_t at, int cnt, const float (&v)[8]) {
  constexpr int es = DT == CIN_DT_F32 ? 4 : 2;
  uint8_t* q = const_cast<uint8_t*>(row) + at * es;
  uint32_t w[kWords<DT>];
#pragma unroll
  for (int k = 0; k < kWords<DT>; ++k) {
    if constexpr (DT == CIN_DT_F32)
      w[k] = __float_as_uint(v[k]);
    else
      w[k] = f32x2_to_half2_bits<DT>(v[2 * k], v[2 * k + 1]);
  }
  if (__builtin_expect(cnt == 8, 1)) {
    __builtin_memcpy(q, w, 16);
    if constexpr (DT == CIN_DT_F32) __builtin_memcpy(q + 16, w + 4, 16);
    return;
  }
  const bool low = !(cnt & 4);
  if constexpr (DT == CIN_DT_F32) {
    const uint4 four = {w[0], w[1], w[2], w[3]};
    const uint2 two = {low ? w[0] : w[4], low ? w[1] : w[5]};
    const uint32_t third = low ? w[2] : w[6], one = cnt & 2 ? third : two.x;
    if (cnt & 4) __builtin_memcpy(q, &four, 16);
    if (cnt & 2) __builtin_memcpy(q + (cnt & 4) * 4, &two, 8);
    if (cnt & 1) __builtin_memcpy(q + (cnt & 6) * 4, &one, 4);
  } else {
    const uint2 four = {w[0], w[1]};
    const uint32_t two = low ? w[0] : w[2];
    const uint16_t one = (uint16_t)(cnt & 2 ? (low ? w[1] : w[3]) : two);
    if (cnt & 4) __builtin_memcpy(q, &four, 8);
    if (cnt & 2) __builtin_memcpy(q + (cnt & 4) * 2, &two, 4);
    if (cnt & 1) __builtin_memcpy(q + (cnt & 6) * 2, &one, 2);
  }
}

__device__ inline void store_elem(void* p, int dt, int64_t i, float v) {
  if (dt == CIN_DT_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_half_bits(dt, v);
}

// 8 channels of a vector, `none` where there is no vector.
__device__ __forceinline__ void load_channels(const Vec& vec, int i, int cnt, float none, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = none;
  if (!vec.p) return;
  if (vec.dtype == CIN_DT_F32) {
    Unit<CIN_DT_F32> u;
    u.load(static_cast<const uint8_t*>(vec.p), (uint32_t)i, cnt);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = u.at(e);
  } else {
    Unit<CIN_DT_BF16> u;
    u.load(static_cast<const uint8_t*>(vec.p), (uint32_t)i, cnt);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = half_bits_to_f32(vec.dtype, (uint16_t)(u.w[e / 2] >> (16 * (e & 1))));
  }
}

__device__ __forceinline__ float row16_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, true));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  v = row16_sum(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Sums of a row's values over its threads, every thread getting them.  A workgroup's sums go through LDS: the
// buffers take turns, and two reductions lie between a buffer's readers and its next writers, of which
// each passes a barrier.
template <bool WAVE, int N>
struct RowSum {
  float (*lds)[N][kWideThreads / 64];  // [2]
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[N], int waves) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
    if constexpr (!WAVE) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) lds[turn][k][wave] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float s = 0.0f;
        for (int i = 0; i < waves; ++i) s += lds[turn][k][i];
        v[k] = s;
      }
      turn ^= 1;
    }
  }
};

// Channels of one thread: CH chunks of 8, `threads` chunks apart.
template <int CH>
struct Span {
  int at[CH], cnt[CH];
  __device__ __forceinline__ void set(int lane, int threads, int D) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      at[c] = (c * threads + lane) * 8;
      cnt[c] = min(max(D - at[c], 0), 8);
    }
  }
};

// FULL: with post norm, gate or learned scale; else x = scale_value r + y.  WAVE: a row a wave.
template <int DT, int DR, int CH, bool WAVE, bool FULL>
__global__ __launch_bounds__(WAVE ? 64 * kWaveRows : kMaxThreads) void k_norm_forward(NormArgs a) {
  __shared__ float lds[2][1][kWideThreads / 64];
  RowSum<WAVE, 1> sum{lds};
  const int lane = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int waves = blockDim.x >> 6;
  const int64_t step = WAVE ? (int64_t)gridDim.x * kWaveRows : gridDim.x;
  int64_t row = WAVE ? (int64_t)blockIdx.x * kWaveRows + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.T) return;
  Span<CH> s;
  s.set(lane, a.threads, a.D);
  float w[CH][8], pw[FULL ? CH : 1][8], g[FULL ? CH : 1][8], sc[FULL ? CH : 1][8];
  const float inv_d = 1.0f / (float)a.D;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load_channels(a.w, s.at[c], s.cnt[c], 1.0f, w[c]);
    if constexpr (FULL) {
      load_channels(a.pw, s.at[c], s.cnt[c], 1.0f, pw[c]);
      load_channels(a.gate_kind == kChannel ? a.gate : Vec{nullptr, 0}, s.at[c], s.cnt[c], 1.0f, g[c]);
      load_channels(a.scale_kind == kPerChannel ? a.scale : Vec{nullptr, 0}, s.at[c], s.cnt[c], a.scale_value, sc[c]);
    }
  }
  float scale = a.scale_value;
  if (FULL && a.scale_kind == kOneValue) {
    scale = load_elem(a.scale.p, a.scale.dtype, 0);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) sc[c][e] = scale;
  }
  for (; row < a.T; row += step) {
    Unit<DT> y[CH], ge[FULL ? CH : 1];
    Unit<DR> r[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      y[c].load(row_at<DT>(a.y, row, a.ldy), s.at[c], s.cnt[c]);
      if (a.r)
        r[c].load(row_at<DR>(a.r, row, a.ldr), s.at[c], s.cnt[c]);
      else
        r[c].zero();
      if constexpr (FULL)
        if (a.gate_kind == kElement) ge[c].load(row_at<DT>(a.gate.p, row, a.ldg), s.at[c], s.cnt[c]);
    }
    float grow = 1.0f, j = 1.0f;
    if constexpr (FULL) {
      if (a.gate_kind == kRow) grow = load_elem(a.gate.p, a.gate.dtype, row * a.ldg);
      if (a.pw.p) {
        float q[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) q[0] = __builtin_fmaf(y[c].at(e), y[c].at(e), q[0]);
        sum(q, waves);
        j = 1.0f / sqrtf(q[0] * inv_d + a.eps);
      }
    }
    float x[CH][8], q[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float u = y[c].at(e);
        if constexpr (FULL) {
          if (a.pw.p) u = u * j * pw[c][e];
          u *= a.gate_kind == kElement ? ge[c].at(e) : a.gate_kind == kRow ? grow : g[c][e];
          x[c][e] = a.r ? __builtin_fmaf(sc[c][e], r[c].at(e), u) : u;
        } else {
          x[c][e] = a.r ? __builtin_fmaf(scale, r[c].at(e), u) : u;
        }
        q[0] = __builtin_fmaf(x[c][e], x[c][e], q[0]);
      }
      if (a.x && s.cnt[c] > 0) store_unit<DR>(row_at<DR>(a.x, row, a.D), s.at[c], s.cnt[c], x[c]);
    }
    sum(q, waves);
    const float i = 1.0f / sqrtf(q[0] * inv_d + a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] = x[c][e] * i * w[c][e];
      if (s.cnt[c] > 0) store_unit<DT>(row_at<DT>(a.n, row, a.D), s.at[c], s.cnt[c], x[c]);
    }
    if (a.stats && lane == 0) {
      a.stats[row] = i;
      a.stats[a.T + row] = j;
    }
  }
}

// Behind the partial rows: a workgroup's sum for the learned scale of one value.
__host__ __device__ inline double* one_sums(const float* partial, int64_t groups, int D) {
  return reinterpret_cast<double*>(const_cast<float*>(partial) + (kSums * groups * D + 1) / 2 * 2);
}

// Partial sums of one workgroup: of its waves' rows together where each has its own.
template <int CH, bool WAVE>
__device__ __forceinline__ void leave_partial(const NormArgs& a, int which, const float (&v)[CH][8], const Span<CH>& s,
                                              float* lds) {
  float* out = a.partial + ((int64_t)which * gridDim.x + blockIdx.x) * a.D;
  if constexpr (WAVE) {
    constexpr int kW = 64 * CH * 8;
    __syncthreads();  // (the buffer's readers before)
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) lds[(threadIdx.x >> 6) * kW + s.at[c] + e] = v[c][e];
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += 64 * kWaveRows) {
      float t = lds[i];
#pragma unroll
      for (int k = 1; k < kWaveRows; ++k) t += lds[k * kW + i];
      out[i] = t;
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (s.cnt[c] > 0) store_unit<CIN_DT_F32>(reinterpret_cast<const uint8_t*>(out), s.at[c], s.cnt[c], v[c]);
  }
}

// What the backward knows of a call when it is compiled: neither post norm nor gate nor learned scale, no gate but of
// channels, anything.
enum Mode { kPlain = 0, kChannels = 1, kAny = 2 };

// What a row of the backward reads; ANY: a gate a row or an element with it.
template <int DT, int DR, int CH, bool ANY>
struct RowIn {
  Unit<DT> y[CH], gn[CH], ge[ANY ? CH : 1];
  Unit<DR> r[CH], gx[CH];
  float i, j, gate;
  __device__ __forceinline__ void load(const NormArgs& a, int64_t row, const Span<CH>& s) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (__builtin_expect(s.cnt[c] == 8, 1)) {
        y[c].load(row_at<DT>(a.y, row, a.ldy), s.at[c]);
        if (a.r) r[c].load(row_at<DR>(a.r, row, a.ldr), s.at[c]);
        if (a.gn) gn[c].load(row_at<DT>(a.gn, row, a.ldgn), s.at[c]);
        if (a.gx) gx[c].load(row_at<DR>(a.gx, row, a.ldgx), s.at[c]);
        if (ANY && a.gate_kind == kElement) ge[ANY ? c : 0].load(row_at<DT>(a.gate.p, row, a.ldg), s.at[c]);
      } else {
        y[c].load(row_at<DT>(a.y, row, a.ldy), s.at[c], s.cnt[c]);
        if (a.r) r[c].load(row_at<DR>(a.r, row, a.ldr), s.at[c], s.cnt[c]);
        if (a.gn) gn[c].load(row_at<DT>(a.gn, row, a.ldgn), s.at[c], s.cnt[c]);
        if (a.gx) gx[c].load(row_at<DR>(a.gx, row, a.ldgx), s.at[c], s.cnt[c]);
        if (ANY && a.gate_kind == kElement) ge[ANY ? c : 0].load(row_at<DT>(a.gate.p, row, a.ldg), s.at[c], s.cnt[c]);
      }
      if (!a.r) r[c].zero();
      if (!a.gn) gn[c].zero();
      if (!a.gx) gx[c].zero();
    }
    i = a.stats[row];
    j = a.stats[a.T + row];
    gate = ANY && a.gate_kind == kRow ? load_elem(a.gate.p, a.gate.dtype, row * a.ldg) : 1.0f;
  }
};

// 8 channels of a thread's chunk c in LDS, each thread's own: two 16-byte words, threads side by side.
struct Slots {
  float4* at;
  int threads, mine, chunks;
  __device__ __forceinline__ float4& half(int which, int c, int h) const {
    return at[((which * chunks + c) * 2 + h) * threads + mine];
  }
  __device__ __forceinline__ void set(int which, int c, const float (&v)[8]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) half(which, c, h) = float4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
  }
  __device__ __forceinline__ void get(int which, int c, float (&v)[8]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 t = half(which, c, h);
      v[4 * h] = t.x;
      v[4 * h + 1] = t.y;
      v[4 * h + 2] = t.z;
      v[4 * h + 3] = t.w;
    }
  }
  __device__ __forceinline__ void add(int which, int c, const float (&v)[8]) const {
    float t[8];
    get(which, c, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] += v[e];
    set(which, c, t);
  }
};

// FULL keeps the channels' vectors in LDS between the rows (w, g pw and the scale, up to 8192 channels of each) and the
// scale's sums too: in registers they would cost the next row's loads, and read again from L2 they would have to
// be waited for behind those.  WIDE, of more channels, has 1024 threads, no room for the vectors in LDS nor for the next
// row in registers: it reads the vectors again, from L2, and its sums spill (4096 x 16384 bf16, gate a channel: 566 us;
// 745 with 512 threads of four chunks).
template <int CH, bool WAVE, bool WIDE>
size_t backward_lds(bool scale_channels, int block) {
  const size_t row = (WAVE ? 64 : block) * CH * 32, own = (size_t)block * CH * 32;
  return (WIDE ? 0 : (scale_channels ? 3 : 2) * row) + (scale_channels ? own : 0);
}

// Waves a SIMD that the registers are kept to: up to 4096 channels a workgroup is small, and others cover its waits
// (4999 x 1111 fp16, gate per element: 49 us with three, 66 with two).  With a 16-bit stream three waves spill 2 registers
// and four (kChannels) 8.
template <int CH, bool WAVE, Mode MODE>
constexpr int kBackwardWaves = WAVE || CH > 1 ? 1 : MODE == kAny ? 3 : 4;

template <int DT, int DR, int CH, bool WAVE, bool WIDE, Mode MODE>
__global__ __launch_bounds__(WAVE ? 64 * kWaveRows : WIDE ? kWideThreads : kMaxThreads, (kBackwardWaves<CH, WAVE, MODE>))
void k_norm_backward(NormArgs a) {
  constexpr bool FULL = MODE != kPlain;
  __shared__ float lds1[2][1][kWideThreads / 64], lds2[2][2][kWideThreads / 64];
  __shared__ float joined[WAVE ? kWaveRows * 64 * CH * 8 : 1];
  extern __shared__ float4 slots[];
  RowSum<WAVE, 1> sum1{lds1};
  RowSum<WAVE, 2> sum2{lds2};
  const int lane = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int waves = blockDim.x >> 6;
  const int64_t step = WAVE ? (int64_t)gridDim.x * kWaveRows : gridDim.x;
  int64_t row = WAVE ? (int64_t)blockIdx.x * kWaveRows + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : blockIdx.x;
  Span<CH> s;
  s.set(lane, a.threads, a.D);
  const bool scale_channels = FULL && a.scale_kind == kPerChannel;
  constexpr bool kInLds = FULL && !WIDE, kInRegisters = !FULL && !WIDE;
  const Slots vectors{slots, WAVE ? 64 : (int)blockDim.x, lane, CH};
  const Slots scale_sums{slots + (kInLds ? 6 * CH * vectors.threads : 0), (int)blockDim.x, (int)threadIdx.x, CH};
  float w[kInRegisters ? CH : 1][8], value = a.scale_value;
  float sw[CH][8], su[FULL ? CH : 1][8];
  double sone = 0.0;  // over all channels of all rows: in fp32 it would lose half its digits
  const float inv_d = 1.0f / (float)a.D;
  if (FULL && a.scale_kind == kOneValue) value = load_elem(a.scale.p, a.scale.dtype, 0);
  auto load_products = [&](int c, float (&v)[8]) {  // g pw
    float g[8];
    load_channels(a.pw, s.at[c], s.cnt[c], 1.0f, v);
    load_channels(a.gate_kind == kChannel ? a.gate : Vec{nullptr, 0}, s.at[c], s.cnt[c], 1.0f, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= g[e];
  };
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float v[8];
    if constexpr (!WIDE) load_channels(a.w, s.at[c], s.cnt[c], 1.0f, v);
    if constexpr (kInLds) vectors.set(0, c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kInRegisters) w[c][e] = v[e];
      sw[c][e] = 0.0f;
    }
    if constexpr (FULL) {
#pragma unroll
      for (int e = 0; e < 8; ++e) su[c][e] = 0.0f;
      if constexpr (kInLds) load_products(c, v);
      if constexpr (kInLds) vectors.set(1, c, v);
      if (scale_channels) {
        load_channels(a.scale, s.at[c], s.cnt[c], 0.0f, v);
        if constexpr (kInLds) vectors.set(2, c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        scale_sums.set(0, c, v);
      }
    }
  }
  auto weights = [&](int c, float (&v)[8]) {
    if constexpr (kInLds) {
      vectors.get(0, c, v);
    } else if constexpr (WIDE) {
      load_channels(a.w, s.at[c], s.cnt[c], 1.0f, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = w[c][e];
    }
  };
  auto products = [&](int c, float (&v)[8]) {
    if constexpr (kInLds)
      vectors.get(1, c, v);
    else if constexpr (FULL)
      load_products(c, v);
  };
  auto scales = [&](int c, float (&v)[8]) {
    if (!scale_channels) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = value;
    } else if constexpr (kInLds) {
      vectors.get(2, c, v);
    } else {
      load_channels(a.scale, s.at[c], s.cnt[c], 0.0f, v);
    }
  };
  // A workgroup's waves wait for each other twice a row, so the next row's loads go out before; waves with rows
  // of their own cover each other's (and fp32 rows are as many bytes without).
  constexpr bool kAhead = !WAVE && !WIDE && DR != CIN_DT_F32;
  const bool post = FULL && a.pw.p, gated = MODE == kAny && (a.gate_kind == kRow || a.gate_kind == kElement);
  const bool inner = FULL && (a.pw.p || a.gate_kind == kChannel);  // S is summed
  using In = RowIn<DT, DR, CH, MODE == kAny>;
  auto one_row = [&](In& in, In& next) {
    if constexpr (kAhead) {
      if (row + step < a.T) next.load(a, row + step, s);
    } else {
      in.load(a, row, s);
    }
    const float i = in.i, j = in.j;
    float x[CH][8], q[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float wc[8], pc[8], sc[8];
      weights(c, wc);
      products(c, pc);
      scales(c, sc);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[c][e] = in.y[c].at(e);
        if constexpr (FULL) x[c][e] = x[c][e] * j * pc[e];
      }
      if (gated) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[c][e] *= a.gate_kind == kElement ? in.ge[MODE == kAny ? c : 0].at(e) : in.gate;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[c][e] = __builtin_fmaf(sc[e], in.r[c].at(e), x[c][e]);  // (r is 0 without a residual)
        q[0] = __builtin_fmaf(in.gn[c].at(e) * wc[e], x[c][e], q[0]);
      }
    }
    sum1(q, waves);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      in.y[c].forget();
      in.r[c].forget();
      in.gn[c].forget();
      if constexpr (MODE == kAny) in.ge[c].forget();
    }
    const float c1 = -(q[0] * inv_d * i * i * i);
    float p[2] = {0.0f, 0.0f}, one_sum = 0.0f;
    // x becomes dx, then du without a channel's gate
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float v[8], wc[8], pc[8];
      weights(c, wc);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = in.gn[c].at(e) * i;
        sw[c][e] = __builtin_fmaf(t, x[c][e], sw[c][e]);
        x[c][e] = __builtin_fmaf(t, wc[e], __builtin_fmaf(x[c][e], c1, in.gx[c].at(e)));
      }
      if (a.dr) {
        scales(c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= x[c][e];
        if (s.cnt[c] > 0) store_unit<DR>(row_at<DR>(a.dr, row, a.D), s.at[c], s.cnt[c], v);
      }
      if constexpr (FULL) {
        if (a.scale_kind == kOneValue) {
#pragma unroll
          for (int e = 0; e < 8; ++e) one_sum = __builtin_fmaf(x[c][e], in.r[c].at(e), one_sum);
        } else if (scale_channels) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = x[c][e] * in.r[c].at(e);
          scale_sums.add(0, c, v);
        }
        products(c, pc);
        if (gated) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = x[c][e] * (in.y[c].at(e) * j * pc[e]);
            p[1] += v[e];
            x[c][e] *= a.gate_kind == kElement ? in.ge[MODE == kAny ? c : 0].at(e) : in.gate;
          }
          if (a.gate_kind == kElement && a.dgate && s.cnt[c] > 0)
            store_unit<DT>(row_at<DT>(a.dgate, row, a.D), s.at[c], s.cnt[c], v);
        }
        if (inner) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float t = x[c][e] * in.y[c].at(e);
            su[c][e] = __builtin_fmaf(t, j, su[c][e]);
            p[0] = __builtin_fmaf(t, pc[e], p[0]);
          }
        }
      }
    }
    if constexpr (FULL) {
      sone += (double)one_sum;
      if (post || (MODE == kAny && a.gate_kind == kRow)) sum2(p, waves);
      if (inner) {
        const float c2 = post ? -(p[0] * inv_d * j * j * j) : 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          in.y[c].forget();
          float pc[8];
          products(c, pc);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[c][e] = x[c][e] * j * pc[e];
            if (post) x[c][e] = __builtin_fmaf(in.y[c].at(e), c2, x[c][e]);
          }
        }
      }
      if (MODE == kAny && a.gate_kind == kRow && a.dgate && lane == 0) store_elem(a.dgate, a.gate.dtype, row, p[1]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (a.dy && s.cnt[c] > 0) store_unit<DT>(row_at<DT>(a.dy, row, a.D), s.at[c], s.cnt[c], x[c]);
    row += step;
  };
  In even, odd;
  if constexpr (kAhead) {
    if (row < a.T) even.load(a, row, s);
    while (row < a.T) {
      one_row(even, odd);
      if (row >= a.T) break;
      one_row(odd, even);
    }
  } else {
    while (row < a.T) one_row(even, odd);
  }
  if (!a.partial) return;
  leave_partial<CH, WAVE>(a, kSumW, sw, s, joined);
  if constexpr (FULL) {
    if (inner) leave_partial<CH, WAVE>(a, kSumU, su, s, joined);
    if (scale_channels) {
#pragma unroll
      for (int c = 0; c < CH; ++c) scale_sums.get(0, c, sw[c]);
      leave_partial<CH, WAVE>(a, kSumScale, sw, s, joined);
    }
    if (a.scale_kind == kOneValue) {
      __shared__ double ones[kWideThreads / 64];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) sone += __shfl_xor(sone, o);
      if ((threadIdx.x & 63) == 0) ones[threadIdx.x >> 6] = sone;
      __syncthreads();
      if (threadIdx.x == 0) {
        double v = 0.0;
        for (int k = 0; k < waves; ++k) v += ones[k];
        one_sums(a.partial, gridDim.x, a.D)[blockIdx.x] = v;
      }
    }
  }
}

// One output of a sum over the rows: times a vector where there is one.
struct ColumnOut {
  void* p;
  int dtype;
  Vec times;
};
struct ColumnArgs {
  const float* partial;
  int64_t G;  // partial rows
  int D;
  ColumnOut out[kSums][2];
  void* one;
  int one_dtype;
};

// The partial rows' sums, each in the order of the rows: 32 channels a workgroup, 32 lines of rows; the
// last workgroup of blockIdx.x has the learned scale's.
__global__ __launch_bounds__(1024) void k_norm_columns(ColumnArgs a) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int groups = (a.D + 31) / 32;
  if ((int)blockIdx.x == groups) {
    if (blockIdx.y != 0 || !a.one) return;
    const double* p = one_sums(a.partial, a.G, a.D);
    __shared__ double sums[16];
    double t = 0.0;
    for (int64_t i = threadIdx.x; i < a.G; i += 1024) t += p[i];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) t += __shfl_xor(t, o);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
      double v = 0.0;
      for (int w = 0; w < 16; ++w) v += sums[w];
      store_elem(a.one, a.one_dtype, 0, (float)v);
    }
    return;
  }
  const ColumnOut& first = a.out[blockIdx.y][0];
  const ColumnOut& second = a.out[blockIdx.y][1];
  if (!first.p && !second.p) return;
  const int d = blockIdx.x * 32 + col;
  float t = 0.0f;
  if (d < a.D) {
    const float* p = a.partial + (int64_t)blockIdx.y * a.G * a.D + d;
#pragma unroll 8
    for (int64_t i = line; i < a.G; i += 32) t += p[i * a.D];
  }
  lds[line][col] = t;
  __syncthreads();
  if (line == 0 && d < a.D) {
    for (int l = 1; l < 32; ++l) t += lds[l][col];
    for (int k = 0; k < 2; ++k) {
      const ColumnOut& o = a.out[blockIdx.y][k];
      if (o.p) store_elem(o.p, o.dtype, d, o.times.p ? t * load_elem(o.times.p, o.times.dtype, d) : t);
    }
  }
}

// Chunks of a thread, threads of a row and whether a wave takes a row.
struct Shape {
  int chunks, threads;
  bool wave, wide;
};
Shape shape_of(int64_t D, bool backward) {
  const int64_t units = cdiv(D, 8);
  if (units <= 64) return {1, 64, true, false};
  if (units <= 128) return {2, 64, true, false};
  const bool wide = backward && units > 2 * kMaxThreads;
  const int chunks = units <= kMaxThreads ? 1 : units <= 2 * kMaxThreads || wide ? 2 : 4;
  return {chunks, (int)(cdiv(cdiv(units, chunks), 64) * 64), false, wide};
}

// Workgroups that walk over the rows.
int64_t groups_of(int64_t T, const Shape& s, bool backward) {
  const int64_t rows = s.wave ? cdiv(T, kWaveRows) : T;
  const int64_t waves = s.wave ? kWaveRows : s.threads / 64;
  const int64_t each = (backward ? 16 : 32) / waves;
  const int64_t most = (int64_t)cin_device_cus() * (each > 1 ? each : 1);
  return rows < most ? rows : most;
}

template <class K>
void allow_lds(K kernel, size_t bytes) {
  if (bytes > 65536) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <int DT, int DR, int CH, bool WAVE, bool WIDE, Mode MODE>
void launch_mode(const NormArgs& a, dim3 grid, dim3 block, hipStream_t stream) {
  const size_t lds = MODE == kPlain ? 0 : backward_lds<CH, WAVE, WIDE>(a.scale_kind == kPerChannel, (int)block.x);
  allow_lds(k_norm_backward<DT, DR, CH, WAVE, WIDE, MODE>, lds);
  hipLaunchKernelGGL((k_norm_backward<DT, DR, CH, WAVE, WIDE, MODE>), grid, block, lds, stream, a);
}

template <int DT, int DR, int CH, bool WAVE, bool WIDE>
void launch_backward(const NormArgs& a, const Shape& s, int64_t groups, bool full, hipStream_t stream) {
  const dim3 grid((uint32_t)groups), block(s.wave ? 64 * kWaveRows : s.threads);
  if (!full)
    launch_mode<DT, DR, CH, WAVE, WIDE, kPlain>(a, grid, block, stream);
  else if (a.gate_kind == kRow || a.gate_kind == kElement)
    launch_mode<DT, DR, CH, WAVE, WIDE, kAny>(a, grid, block, stream);
  else
    launch_mode<DT, DR, CH, WAVE, WIDE, kChannels>(a, grid, block, stream);
}

template <int DT, int DR, int CH, bool WAVE>
void launch_forward(const NormArgs& a, const Shape& s, int64_t groups, bool full, hipStream_t stream) {
  const dim3 grid((uint32_t)groups), block(s.wave ? 64 * kWaveRows : s.threads);
  if (full)
    hipLaunchKernelGGL((k_norm_forward<DT, DR, CH, WAVE, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((k_norm_forward<DT, DR, CH, WAVE, false>), grid, block, 0, stream, a);
}

template <int DT, int DR>
void launch_shape(const NormArgs& a, const Shape& s, int64_t groups, bool full, bool backward, hipStream_t stream) {
  if (!backward) {
    if (s.wave && s.chunks == 1)
      launch_forward<DT, DR, 1, true>(a, s, groups, full, stream);
    else if (s.wave)
      launch_forward<DT, DR, 2, true>(a, s, groups, full, stream);
    else if (s.chunks == 1)
      launch_forward<DT, DR, 1, false>(a, s, groups, full, stream);
    else if (s.chunks == 2)
      launch_forward<DT, DR, 2, false>(a, s, groups, full, stream);
    else
      launch_forward<DT, DR, 4, false>(a, s, groups, full, stream);
  } else if (s.wave && s.chunks == 1) {
    launch_backward<DT, DR, 1, true, false>(a, s, groups, full, stream);
  } else if (s.wave) {
    launch_backward<DT, DR, 2, true, false>(a, s, groups, full, stream);
  } else if (s.wide) {
    launch_backward<DT, DR, 2, false, true>(a, s, groups, full, stream);
  } else if (s.chunks == 1) {
    launch_backward<DT, DR, 1, false, false>(a, s, groups, full, stream);
  } else {
    launch_backward<DT, DR, 2, false, false>(a, s, groups, full, stream);
  }
}

void launch_types(const NormArgs& a, int dt, int dr, const Shape& s, int64_t groups, bool full, bool backward,
                  hipStream_t stream) {
  if (dt == CIN_DT_BF16 && dr == CIN_DT_BF16)
    launch_shape<CIN_DT_BF16, CIN_DT_BF16>(a, s, groups, full, backward, stream);
  else if (dt == CIN_DT_BF16)
    launch_shape<CIN_DT_BF16, CIN_DT_F32>(a, s, groups, full, backward, stream);
  else if (dt == CIN_DT_F16 && dr == CIN_DT_F16)
    launch_shape<CIN_DT_F16, CIN_DT_F16>(a, s, groups, full, backward, stream);
  else if (dt == CIN_DT_F16)
    launch_shape<CIN_DT_F16, CIN_DT_F32>(a, s, groups, full, backward, stream);
  else
    launch_shape<CIN_DT_F32, CIN_DT_F32>(a, s, groups, full, backward, stream);
}

bool is_type(int dt) { return dt == CIN_DT_BF16 || dt == CIN_DT_F16 || dt == CIN_DT_F32; }

// Checks of what both directions take; fills the arguments.
int common_args(NormArgs& a, const char* name, const void* y, int dtype, int64_t ldy, const void* r, int r_dtype,
                int64_t ldr, int64_t T, int64_t D, const void* w, int w_dtype, const void* pw, int pw_dtype, const void* gate,
                int gate_dtype, int gate_kind, int64_t ldg, const void* scale, int scale_dtype, int scale_kind,
                float scale_value, float eps) {
  CIN_CHECK_ARG(is_type(dtype) && is_type(r_dtype), "%s: dtype must be bf16, fp16 or fp32", name);
  CIN_CHECK_ARG(r_dtype == dtype || r_dtype == CIN_DT_F32, "%s: the residual must have y's dtype or fp32", name);
  CIN_CHECK_ARG(T >= 0 && T < (1LL << 40) && D >= 1 && D <= kMaxWidth, "%s: D must be in [1, %lld]", name, (long long)kMaxWidth);
  CIN_CHECK_ARG(ldy >= D && (!r || ldr >= D), "%s: row stride below D", name);
  CIN_CHECK_ARG((!w || is_type(w_dtype)) && (!pw || is_type(pw_dtype)), "%s: weights must be bf16, fp16 or fp32", name);
  const bool no_gates = T == 0 && (gate_kind == kRow || gate_kind == kElement);  // one for each of no rows: maybe null
  CIN_CHECK_ARG(gate_kind >= kNoGate && gate_kind <= kElement && (no_gates || (gate != nullptr) == (gate_kind != kNoGate)) &&
                    (!gate || is_type(gate_dtype)),
                "%s: bad gate", name);
  CIN_CHECK_ARG(gate_kind != kElement || (gate_dtype == dtype && ldg >= D), "%s: a gate of elements must have y's dtype and rows of D",
                name);
  CIN_CHECK_ARG(gate_kind != kRow || ldg >= 1, "%s: bad gate stride", name);
  CIN_CHECK_ARG(scale_kind >= kNumber && scale_kind <= kPerChannel && (scale != nullptr) == (scale_kind != kNumber) &&
                    (!scale || is_type(scale_dtype)),
                "%s: bad residual scale", name);
  a = {};
  a.y = y;
  a.r = r;
  a.ldy = ldy;
  a.ldr = ldr;
  a.T = T;
  a.D = (int)D;
  a.w = {w, w_dtype};
  a.pw = {pw, pw_dtype};
  a.gate = {gate, gate_dtype};
  a.scale = {scale, scale_dtype};
  a.gate_kind = gate_kind;
  a.scale_kind = scale_kind;
  a.ldg = ldg;
  a.scale_value = scale_value;
  a.eps = eps;
  return CIN_OK;
}

bool is_full(const NormArgs& a) { return a.pw.p || a.gate_kind != kNoGate || a.scale_kind != kNumber; }

}  // namespace

extern "C" {

int cin_block_norm(const void* y, int dtype, int64_t ldy, const void* r, int r_dtype, int64_t ldr, int64_t T, int64_t D,
                   const void* w, int w_dtype, const void* pw, int pw_dtype, const void* gate, int gate_dtype, int gate_kind,
                   int64_t ldg, const void* scale, int scale_dtype, int scale_kind, float scale_value, float eps, void* n,
                   void* x, float* stats, void* stream) {
  NormArgs a;
  const int rc = common_args(a, "cin_block_norm", y, dtype, ldy, r, r_dtype, ldr, T, D, w, w_dtype, pw, pw_dtype, gate,
                             gate_dtype, gate_kind, ldg, scale, scale_dtype, scale_kind, scale_value, eps);
  if (rc != CIN_OK || T == 0) return rc;
  CIN_CHECK_ARG(y && n, "cin_block_norm: null pointer");
  a.n = n;
  a.x = x;
  a.stats = stats;
  const Shape s = shape_of(D, false);
  a.threads = s.threads;
  launch_types(a, dtype, r_dtype, s, groups_of(T, s, false), is_full(a), false, (hipStream_t)stream);
  return cin_check_launch("cin_block_norm");
}

int64_t cin_block_norm_workspace(int64_t T, int64_t D) {
  if (T < 0 || D < 1 || D > kMaxWidth) {
    cin_set_error(CIN_ERR_ARG, "cin_block_norm_workspace: D must be in [1, %lld]", (long long)kMaxWidth);
    return -1;
  }
  const int64_t groups = groups_of(T, shape_of(D, true), true);
  return 4 * ((kSums * groups * D + 1) / 2 * 2) + 8 * groups;
}

int cin_block_norm_backward(const void* y, int dtype, int64_t ldy, const void* r, int r_dtype, int64_t ldr, int64_t T,
                            int64_t D, const void* w, int w_dtype, const void* pw, int pw_dtype, const void* gate,
                            int gate_dtype, int gate_kind, int64_t ldg, const void* scale, int scale_dtype, int scale_kind,
                            float scale_value, const float* stats, const void* gn, int64_t ldgn, const void* gx,
                            int64_t ldgx, void* dy, void* dr, void* dw, void* dpw, void* dgate, void* dscale,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  NormArgs a;
  const int rc = common_args(a, "cin_block_norm_backward", y, dtype, ldy, r, r_dtype, ldr, T, D, w, w_dtype, pw, pw_dtype,
                             gate, gate_dtype, gate_kind, ldg, scale, scale_dtype, scale_kind, scale_value, 0.0f);
  if (rc != CIN_OK || T == 0) return rc;
  CIN_CHECK_ARG(y && stats, "cin_block_norm_backward: null pointer");
  CIN_CHECK_ARG((!gn || ldgn >= D) && (!gx || ldgx >= D), "cin_block_norm_backward: row stride below D");
  CIN_CHECK_ARG((!dw || w) && (!dpw || pw) && (!dgate || gate) && (!dscale || scale) && (!dr || r),
                "cin_block_norm_backward: a gradient of an input that is not there");
  CIN_CHECK_ARG(!dscale || r, "cin_block_norm_backward: a scale without a residual");
  ColumnArgs c = {};
  const Vec none = {nullptr, 0};
  c.out[kSumW][0] = {dw, w_dtype, none};
  c.out[kSumU][0] = {dpw, pw_dtype, gate_kind == kChannel ? a.gate : none};
  if (gate_kind == kChannel) c.out[kSumU][1] = {dgate, gate_dtype, a.pw};
  if (scale_kind == kPerChannel) {
    c.out[kSumScale][0] = {dscale, scale_dtype, none};
  } else if (scale_kind == kOneValue) {
    c.one = dscale;
    c.one_dtype = scale_dtype;
  }
  const bool inner = c.out[kSumU][0].p || c.out[kSumU][1].p;
  const bool sums = dw || inner || dscale;
  CIN_CHECK_ARG(!sums || (workspace && workspace_bytes >= cin_block_norm_workspace(T, D)),
                "cin_block_norm_backward: workspace below cin_block_norm_workspace bytes");
  a.stats = const_cast<float*>(stats);
  a.gn = gn;
  a.gx = gx;
  a.ldgn = ldgn;
  a.ldgx = ldgx;
  a.dy = dy;
  a.dr = dr;
  a.dgate = dgate;
  a.partial = sums ? static_cast<float*>(workspace) : nullptr;
  const Shape s = shape_of(D, true);
  a.threads = s.threads;
  const int64_t groups = groups_of(T, s, true);
  launch_types(a, dtype, r_dtype, s, groups, is_full(a), true, (hipStream_t)stream);
  if (sums) {
    c.partial = a.partial;
    c.G = groups;
    c.D = (int)D;
    const int rows = c.out[kSumScale][0].p ? 3 : inner ? 2 : 1;
    hipLaunchKernelGGL(k_norm_columns, dim3((uint32_t)(cdiv(D, 32) + (c.one ? 1 : 0)), rows), dim3(1024), 0, (hipStream_t)stream, c);
  }
  return cin_check_launch("cin_block_norm_backward");
}

}  // extern "C"
