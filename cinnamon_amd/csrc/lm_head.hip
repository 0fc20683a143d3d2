// Output projection and softmax cross entropy over a large vocabulary on gfx950, without keeping
// the logits.
//
//   z[t, v]  = x[t] . w[v]                 loss_t = log(sum_v exp(z[t, v])) - z[t, y_t]
//   dz[t, v] = g_t (exp(z[t, v] - max_t) / total_t - [v = y_t])
//   dx       = dz w                        dw = dz^T x
//
// Rows whose target is ignore_index are taken out first (x is copied without them), so that no
// product runs over them.  Forward: one product whose tiles leave only each row's maximum and sum
// of exponentials and the target's logit.  Backward: by pieces of the vocabulary, a product that
// ends in dz of the piece (in x's type), then dx += dz w and dw = dz^T x of the piece.  The caller may have
// the forward keep the logits of few rows for it.
//
// One kernel runs the three products on the matrix units, with fp32 sums.  fp32 values are held as
// three bf16 ones (x = x0 + x1 + x2, each the rounding of what is left, exact to 2^-26), and their
// product is the six products of planes down to x0 y2, the small ones first: what is dropped lies
// under 2^-26 of |x y|, and the sums are those of fp32 products (2046 x 32000 x 1024: 0.64 ms, 208
// TFLOP/s; on the fp32 matrix units, in the same tiles, 1.04 ms).  An operand is read along K (its rows
// hold K) or across it (its rows are K), so no transposed copy of x, w or dz is ever made.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "cin_common.h"
#include "cin_gemm_tile.h"
#include "cin_grouped.h"
#include "cin_runtime.h"

using namespace cin;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kOut = 0x80000000u;  // an out-of-range lane offset

typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// What the products' operands hold: CIN_DT_BF16 or CIN_DT_F16; CIN_DT_F32 for three bf16 planes; kDirect
// for fp32 as it is, for few rows.
constexpr int kDirect = 3;
template <int DT>
constexpr int kEs = DT == kDirect ? 4 : 2;  // bytes of an operand's element
constexpr int kStepBytes = 128;
constexpr int kPadK = 64;  // operands that hold K in their rows have a multiple of it: whole K steps

// s_waitcnt vmcnt(N): everything but the last N vector memory operations has completed
template <int N>
__device__ __forceinline__ void wait_dma_but() {
  static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4 << 14));
}

// Workgroup tile of 16 MT WM x 16 NT WN, K steps of 128 bytes in STAGES LDS stages.
template <int WM_, int WN_, int MT_, int NT_, int STAGES>
struct Cfg {
  static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, kStages = STAGES;
  static constexpr int kThreads = 64 * WM * WN, TM = 16 * MT * WM, TN = 16 * NT * WN;
  static constexpr int kStage = (TM + TN) * 128;
  static constexpr int kCStride = TN * 2 + 16;  // a staged row of 16-bit results; rows 4 banks apart
  // staged rows: all, or one row of waves at a time where all would not fit
  static constexpr int kParts = TM * kCStride <= 160 * 1024 ? 1 : WM, kPartRows = TM / kParts;
  static constexpr int kBytes = STAGES * kStage > kPartRows * kCStride ? STAGES * kStage : kPartRows * kCStride;
  // Stages that hold all planes of fp32 operands, 0 where two do not fit.  A step then has all six products,
  // which short runs of steps need (512 x 1500 x 4096: forward 179 -> 85 us, with gradients 457 -> 265).
  static constexpr int kStages3 = 160 * 1024 / (3 * kStage) < 2 ? 0 : 160 * 1024 / (3 * kStage) < 4 ? 160 * 1024 / (3 * kStage) : 4;
};

// What a product ends in.
enum Epi {
  kStats,  // the row's maximum and sum of exponentials over the tile, and the target's logit
  kGrad,   // dz, in the operands' type (three planes of it for fp32)
  kSlab,   // fp32 partial sums (added to what is there with `add`)
  kFinal   // times a device scalar, in x's type
};

// Slabs of dx: K is split for the rows that count, which only the device knows, where their tiles are
// fewer than the CUs; in parts of 8 steps at least, and in the memory that was given.
struct Slabs {
  int tile_m, tiles_n;  // rows of a tile, tiles of a row
  int most, parts;      // workgroups, parts of K
  int64_t room;         // rows of all slabs
  __device__ int count(int64_t n) const {
    if (n == 0) return 1;
    int64_t s = most / (cdiv(n, tile_m) * tiles_n);
    if (s > room / n) s = room / n;
    if (s > parts) s = parts;
    return s < 1 ? 1 : (int)s;
  }
};

struct GemmArgs {
  const void *A, *B;
  int64_t lda, ldb;
  int64_t plane_a, plane_b;  // bytes between the planes of an fp32 operand
  int64_t M, N, K;     // N: columns to compute; K: a multiple of a K step where an operand holds K in its rows
  const int* n;        // rows there are, in place of M (or of K for kFinal)
  const int* slabs;    // how many (kSlab)
  int segs;            // planes of a 16-bit B (kFinal)
  int64_t ldc, slab;   // elements between rows of C, between planes of dz
  void* C;
  int add;
  int64_t v0, V;       // first column of the piece and columns of the vocabulary
  int64_t wa, wb;      // columns there are of an operand that is read across K
  float2* part;        // [T, tiles_n]
  float* ztarget;
  const int* target;
  const float *rowmax, *inv, *coef, *out_scale;
  float* dropped;      // [T], what rounding took off each row's dz of its target (null: not used)
};

// One operand of ROWS tile rows (of M or N) and a 128-byte K step, moved global -> LDS by DMA.
// Along K: LDS rows are tile rows of 128 bytes, 16-byte chunk c of row r at slot c ^ f(r).
// Across K: LDS rows are the step's K rows of ROWS elements, in granules of 16 elements, granule
// q of row r at q ^ f(r): the rows that one transposing read takes together lie on other banks.
template <int ROWS, int THREADS, bool ACROSS, int ES>
struct Operand {
  static constexpr int BK = kStepBytes / ES;
  static constexpr int kOps = ROWS * 8 / THREADS;
  static constexpr int kCpr = ACROSS ? ROWS * ES / 16 : 8;  // 16-byte chunks of an LDS row
  static constexpr int kGc = ES;                            // of a granule of 16 elements (across)
  static constexpr int kGran = kCpr / kGc;
  static_assert(ROWS * 8 % THREADS == 0, "whole operations");
  uint32_t voff[kOps];
  const uint8_t* p;
  int64_t ldb, kleft, bytes;
  uint32_t lds;

  __device__ static inline int f(int r) {
    if constexpr (!ACROSS) return (r >> 1) & 7;  // (the 16 rows and two chunks of a pass on 64 banks: no conflicts)
    if constexpr (ES == 4) return (r >> 2) & 3 & (kGran - 1);
    return ((r & 3) | ((r >> 3 & 1) << 2)) & (kGran - 1);
  }
  // r0: the tile's first row (along) or column (across); valid: rows (along) or columns (across)
  // from there on; k0, k1: the K range that there is
  __device__ __forceinline__ void init(const void* base, int64_t ld, int64_t r0, int64_t valid, int64_t k0, int64_t k1,
                                       int tid, uint32_t lds0) {
    ldb = ld * ES;
    lds = lds0 + (uint32_t)__builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
    kleft = k1 - k0;
    if constexpr (ACROSS) {
      p = static_cast<const uint8_t*>(base) + k0 * ldb + r0 * ES;
      bytes = valid * ES;  // of the last K row
    } else {
      const int rows = (int)(valid < ROWS ? valid : ROWS);
      p = static_cast<const uint8_t*>(base) + r0 * ldb + k0 * ES;
      bytes = (rows - 1) * ldb + kleft * ES;
    }
#pragma unroll
    for (int i = 0; i < kOps; ++i) {
      const int slot = i * THREADS + tid, r = slot / kCpr, c = slot % kCpr;
      if constexpr (ACROSS) {
        voff[i] = (uint32_t)(r * ldb) + (uint32_t)((((c / kGc) ^ f(r)) * kGc + c % kGc) * 16);
      } else {
        voff[i] = r < valid ? (uint32_t)(r * ldb) + (uint32_t)((c ^ f(r)) * 16) : kOut;
      }
    }
  }
  // K step kt of the plane that lies `plane` bytes on
  __device__ __forceinline__ void fetch(int kt, int64_t plane, uint32_t stage) {
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t so = 0;
    if constexpr (ACROSS) {
      const int64_t left = kleft - (int64_t)kt * BK;
      // K rows past the last read as zero, and nothing is read past the last row's end
      rsrc = make_rsrc(p + plane + (int64_t)kt * BK * ldb, left > 0 ? ((left < BK ? left : BK) - 1) * ldb + bytes : 0);
    } else {
      rsrc = make_rsrc(p + plane, bytes);
      so = (uint32_t)__builtin_amdgcn_readfirstlane(kt) * kStepBytes;
    }
#pragma unroll
    for (int i = 0; i < kOps; ++i) dma16(rsrc, voff[i], so, lds + stage + i * THREADS * 16);
  }
  // 16 bytes a lane: K elements 8 kq .. + 7 of half ks (of 4 bytes: 4 kq .. + 3) of tile row r16 + l16
  __device__ static __forceinline__ v4u frag(const uint8_t* st, int r16, int ks, int l16, int kq) {
    if constexpr (!ACROSS) {
      return *reinterpret_cast<const v4u*>(st + (r16 + l16) * 128 + (((4 * ks + kq) ^ f(r16 + l16)) << 4));
    } else if constexpr (ES == 4) {
      v4u v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 16 * ks + 4 * kq + e;
        v[e] = *reinterpret_cast<const uint32_t*>(st + k * (ROWS * 4) + ((((r16 >> 4)) ^ f(k)) << 6) + l16 * 4);
      }
      return v;
    } else {
      v4u v;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 32 * ks + 8 * kq + 4 * h + (l16 >> 2);
        const uint8_t* q = st + k * (ROWS * 2) + ((((r16 >> 4)) ^ f(k)) << 5) + (l16 & 3) * 8;
        const s4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)q);
        const uint2 u = __builtin_bit_cast(uint2, t);
        v[2 * h] = u.x;
        v[2 * h + 1] = u.y;
      }
      return v;
    }
  }
};

// c += a b over a half step: lane (l16, kq) holds column l16 of b and rows 4 kq .. + 3 of a
template <int DT>
__device__ __forceinline__ v4f mma(v4u a, v4u b, v4f c) {
  if constexpr (DT == kDirect) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  } else
  if constexpr (DT == CIN_DT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// The planes of the products of an fp32 operand pair, small terms first.
constexpr int kPairs32 = 6;
__device__ inline void planes_of(int seg, int& a, int& b) {
  a = seg == 0 ? 2 : (seg == 1 || seg == 3 ? 1 : 0);
  b = seg == 2 ? 2 : (seg == 1 || seg == 4 ? 1 : 0);
}

__device__ inline float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// A row of dx or dw is mostly its targets' entries of dz times rows of w or x, and the rounding of those
// few numbers to 16 bits does not average out.  So kGrad leaves what it took off each row's target entry;
// k_ce_dx adds it times the target's row of w, and here the rows of x whose targets are rows m0 .. of a dw
// tile come once more with it, as further K steps: the targets are looked through, 64 rows found at a time, in
// their order.  Errors against 64 bits without it, with it, and of the results' own rounding: bf16 16368 x 32000 x
// 1024 1.82e-3, 1.66e-3, 1.66e-3; fp16 1800 x 50257 x 1001 2.36e-4, 2.08e-4, 2.08e-4.  A step is not fetched ahead
// and takes about 3 us: forward and gradients of 16384 x V x 1024, bf16, V 32000: 3797 -> 3807 us, 4000: 673 -> 682,
// 500: 249 -> 271; 8192 x 131072 x 4096: 1%.
template <class C, int DT>
__device__ __forceinline__ void add_dropped(const GemmArgs& g, uint8_t* smem, int64_t rows, int64_t m0, int64_t n0, int wave,
                                            int lane, v4f (&acc)[C::MT][C::NT]) {
  using A = Operand<C::TM, C::kThreads, true, 2>;
  using B = Operand<C::TN, C::kThreads, true, 2>;
  constexpr int kPer = 16, kWaves = C::kThreads / 64;  // targets a thread looks at together
  static_assert(C::kStage + C::kThreads * kPer * 4 + kWaves * 4 <= C::kBytes, "a K step, the rows found, counts");
  int* found = reinterpret_cast<int*>(smem + C::kStage);
  int* counts = found + C::kThreads * kPer;
  const int tid = wave * 64 + lane;
  const uint32_t first = (uint32_t)(g.v0 + m0);
  const uint16_t* x = static_cast<const uint16_t*>(g.B);
  for (int64_t t0 = 0; t0 < rows; t0 += C::kThreads * kPer) {
    const int64_t t = t0 + tid * kPer;
    uint32_t hits = 0;
    int y[kPer];
    if (t + kPer <= rows) {
      __builtin_memcpy(y, g.target + t, sizeof(y));
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) y[e] = t + e < rows ? g.target[t + e] : -1;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) hits |= (uint32_t)(y[e] >= 0 && (uint32_t)y[e] - first < (uint32_t)C::TM) << e;
    int at = __popc(hits);
    const int mine = at;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(at, o);
      at += lane >= o ? v : 0;
    }
    if (lane == 63) counts[wave] = at;
    __syncthreads();
    int all = 0;
    at -= mine;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int v = counts[w];
      at += w < wave ? v : 0;
      all += v;
    }
    for (; hits; hits &= hits - 1) found[at++] = (int)(t + __builtin_ctz(hits));
    for (int s = 0; s < all; s += 64) {
      const int left = all - s < 64 ? all - s : 64;
      for (int q = tid; q < C::TM * 8; q += C::kThreads) reinterpret_cast<v4u*>(smem)[q] = v4u{0, 0, 0, 0};
      __syncthreads();  // (and the rows found are there)
      v4u v[B::kOps];
#pragma unroll
      for (int i = 0; i < B::kOps; ++i) {
        const int slot = i * C::kThreads + tid, r = slot / B::kCpr, c = slot % B::kCpr;
        const int64_t col = n0 + (((c / B::kGc) ^ B::f(r)) * B::kGc + c % B::kGc) * 8;
        // (any row and column that there are, where it is none)
        v[i] = *reinterpret_cast<const v4u*>(x + found[r < left ? s + r : s] * g.ldb + (col < g.wb ? col : 0));
        if (r >= left || col >= g.wb) v[i] = v4u{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < B::kOps; ++i)
        *reinterpret_cast<v4u*>(smem + C::TM * 128 + (i * C::kThreads + tid) * 16) = v[i];
      if (tid < left) {
        const int row = found[s + tid], m = g.target[row] - (int)first;
        *reinterpret_cast<uint16_t*>(smem + tid * (C::TM * 2) + (((m >> 4) ^ A::f(tid)) << 5) + (m & 15) * 2) =
            (uint16_t)f32_to_half_bits(DT, g.dropped[row]);
      }
      __syncthreads();
#pragma unroll 1
      for (int ks = 0; ks < 2; ++ks) {
        v4u b[C::NT];
#pragma unroll
        for (int j = 0; j < C::NT; ++j) b[j] = B::frag(smem + C::TM * 128, (wave % C::WN * C::NT + j) * 16, ks, lane & 15, lane >> 4);
#pragma unroll
        for (int i = 0; i < C::MT; ++i) {
          const v4u a = A::frag(smem, (wave / C::WN * C::MT + i) * 16, ks, lane & 15, lane >> 4);
#pragma unroll
          for (int j = 0; j < C::NT; ++j) acc[i][j] = mma<DT>(b[j], a, acc[i][j]);
        }
      }
      lds_barrier();
    }
    __syncthreads();
  }
}

template <class C, int DT, int EPI>
__global__ __launch_bounds__(C::kThreads, 2) void k_ce_gemm(GemmArgs g) {
  constexpr bool kAcrossA = EPI == kFinal, kAcrossB = EPI == kSlab || EPI == kFinal;
  constexpr int MT = C::MT, NT = C::NT, kSegs = DT == CIN_DT_F32 ? kPairs32 : 1, BK = kStepBytes / kEs<DT>;
  constexpr bool kTogether = DT == CIN_DT_F32 && C::kStages3 > 0, k16 = DT == CIN_DT_BF16 || DT == CIN_DT_F16;
  constexpr int kStages = kTogether ? C::kStages3 : C::kStages, kPlanes = kTogether ? 3 : 1, kStage = C::kStage * kPlanes;
  __shared__ __attribute__((aligned(128))) uint8_t smem[kStages * kStage > C::kBytes ? kStages * kStage : C::kBytes];
  const int64_t rows = __builtin_amdgcn_readfirstlane(*g.n);
  const int64_t M = EPI == kFinal ? g.M : rows, Kall = EPI == kFinal ? rows : g.K;
  const uint32_t tiles_m = (uint32_t)cdiv(M, C::TM), tiles_n = (uint32_t)cdiv(g.N, C::TN);
  const uint32_t tiles = tiles_m * tiles_n, total = EPI == kSlab ? tiles * *g.slabs : tiles;
  if (blockIdx.x >= total) return;
  uint32_t tm, tn, tile = xcd_remap(blockIdx.x, total), part = 0;
  if constexpr (EPI == kSlab) {  // the tiles of a part of K side by side, which share its rows of w
    part = tile / tiles;
    tile -= part * tiles;
  }
  raster<4>(tile, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * C::TM, n0 = (int64_t)tn * C::TN;
  int64_t k0 = 0, k1 = Kall;
  if constexpr (EPI == kSlab) {
    const int64_t per = cdiv(cdiv(Kall, BK), *g.slabs) * BK;
    k0 = part * per;
    k1 = k0 + per < Kall ? k0 + per : Kall;
  }
  int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  int l16 = tid & 15, kq = tid >> 4 & 3;
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
  Operand<C::TM, C::kThreads, kAcrossA, kEs<DT>> oa;
  Operand<C::TN, C::kThreads, kAcrossB, kEs<DT>> ob;
  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  v4f low[kTogether ? MT : 1][kTogether ? NT : 1] = {};  // the small products
  const int nk = k1 > k0 ? (int)((k1 - k0 + BK - 1) / BK) : 0;
  if (nk > 0) {
    // w has rows up to the vocabulary's end, as tile rows or as K
    oa.init(g.A, g.lda, m0, (kAcrossA ? g.wa : M) - m0, k0, k1, tid, lds0);
    ob.init(g.B, g.ldb, n0, (kAcrossB ? g.wb : g.V - g.v0) - n0, k0,
            EPI == kSlab && k1 > g.V - g.v0 ? g.V - g.v0 : k1, tid, lds0 + C::TM * 128 * kPlanes);
  }
  int fk = 0, seg = 0;  // the K step and pair of planes that are fetched next
  const auto fetch = [&](uint32_t stage) {
    if constexpr (kTogether) {
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        oa.fetch(fk, p * g.plane_a, stage + p * C::TM * 128);
        ob.fetch(fk, p * g.plane_b, stage + p * C::TN * 128);
      }
      ++fk;
      return;
    }
    int64_t pa = 0, pb = 0;
    if constexpr (kSegs > 1) {
      int ia, ib;
      planes_of(seg, ia, ib);
      pa = ia * g.plane_a;
      pb = ib * g.plane_b;
    } else if constexpr (EPI == kFinal) {
      pb = (g.segs - 1 - seg) * g.plane_b;  // the low parts first
    }
    oa.fetch(fk, pa, stage);
    ob.fetch(fk, pb, stage);
    if (++fk == nk) {
      fk = 0;
      ++seg;
    }
  };
  const int steps = nk * (EPI == kFinal && kSegs == 1 ? g.segs : kTogether ? 1 : kSegs);
  constexpr int kOps = (decltype(oa)::kOps + decltype(ob)::kOps) * kPlanes;
#pragma unroll
  for (int q = 0; q < kStages - 1; ++q)
    if (q < steps) fetch(q * kStage);
  for (int kt = 0; kt < steps; ++kt) {
    // step kt has landed once no more than the kStages - 2 behind it are on their way
    if (kStages > 2 && kt + kStages - 2 < steps)
      wait_dma_but<(kStages - 2) * kOps>();
    else
      wait_dma();
    lds_barrier();
    const uint32_t st = (kt % kStages) * kStage;
    // where step kt - 1 was, read by all
    if (kt + kStages - 1 < steps) fetch((kt + kStages - 1) % kStages * kStage);
    const uint8_t* sa = smem + st;
    const uint8_t* sb = sa + C::TM * 128 * kPlanes;
    if constexpr (kTogether) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        v4u bf[3][NT];
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
          for (int j = 0; j < NT; ++j) bf[p][j] = ob.frag(sb + p * C::TN * 128, (wn * NT + j) * 16, ks, l16, kq);
        v4u af[3][MT];
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
          for (int i = 0; i < MT; ++i) af[p][i] = oa.frag(sa + p * C::TM * 128, (wm * MT + i) * 16, ks, l16, kq);
#pragma unroll
        for (int q = 0; q < kPairs32; ++q) {
          int ia, ib;
          planes_of(q, ia, ib);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              v4f& c = q + 1 < kPairs32 ? low[i][j] : acc[i][j];
              c = mma<DT>(bf[ib][j], af[ia][i], c);
            }
        }
      }
    } else {
      // The fp32 matrix units add one product after the other, each sum rounded: a sum of its own for each step
      // of 32 leaves a fifth of the error where K is long (logits of 4096 products of variance 1: 4.2e-5 to 7.9e-5
      // -> 0.8e-5 to 1.4e-5; K of dw is the rows).  Forward of 16 x 100000 x 2048 181 -> 186 us, of 128 489 -> 534.
      constexpr bool kOwn = DT == kDirect && EPI != kFinal;
      v4f own[kOwn ? MT : 1][kOwn ? NT : 1] = {};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        v4u bf[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) bf[j] = ob.frag(sb, (wn * NT + j) * 16, ks, l16, kq);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const v4u af = oa.frag(sa, (wm * MT + i) * 16, ks, l16, kq);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            v4f& c = kOwn ? own[kOwn ? i : 0][kOwn ? j : 0] : acc[i][j];
            c = mma<DT>(bf[j], af, c);
          }
        }
      }
      if constexpr (kOwn) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] += own[i][j];
      }
    }
  }
  if constexpr (kTogether) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] += low[i][j];
  }
  lds_barrier();
  if constexpr (EPI == kFinal && k16) {
    // the lane's number anew: kept through the loop it would take a register of the operands
    const int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    tid = wave * 64 + lane;
    l16 = lane & 15;
    kq = lane >> 4;
    if (g.dropped) add_dropped<C, DT>(g, smem, Kall, m0, n0, wave, lane, acc);
  }
  // the lane holds rows m0 + (wm MT + i) 16 + l16, columns n0 + (wn NT + j) 16 + 4 kq + r
  const int64_t nl = n0 + wn * NT * 16 + 4 * kq;
  if constexpr (EPI == kStats) {
    float2* st = reinterpret_cast<float2*>(smem);
    if (g.C) {  // the logits, for few rows
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + (wm * MT + i) * 16 + l16;
#pragma unroll
        for (int j = 0; j < NT; ++j)
          if (m < M && nl + j * 16 < g.ldc)
            *reinterpret_cast<float4*>(static_cast<float*>(g.C) + m * g.ldc + nl + j * 16) =
                make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      }
    }
    if (n0 + C::TN > g.N) {  // columns past the vocabulary add nothing
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (nl + j * 16 + r >= g.N) {
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j][r] = -__builtin_inff();
          }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int ml = (wm * MT + i) * 16 + l16;
      const bool in = m0 + ml < M;
      // (few waves hold a row's target)
      const int64_t at = (in ? g.target[m0 + ml] : -1) - nl;
      if (at >= 0 && at < NT * 16 && (at & 15) < 4) {
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) z = (int)at == j * 16 + r ? acc[i][j][r] : z;
        g.ztarget[m0 + ml] = z;
      }
      float mx = acc[i][0][0];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      float s = 0.0f;
      // (a wave with no column of the vocabulary, or nothing but -inf, adds nothing)
      const float ref = mx == -__builtin_inff() ? 0.0f : mx;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s += exp_of(acc[i][j][r] - ref);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (kq == 0) st[wn * C::TM + ml] = make_float2(mx, s);
    }
    __syncthreads();
    for (int m = tid; m < C::TM; m += C::kThreads) {
      if (m0 + m >= M) continue;
      float2 a = st[m];
      float s = 0.0f;
#pragma unroll
      for (int w = 1; w < C::WN; ++w) a.x = fmaxf(a.x, st[w * C::TM + m].x);
      const float ref = a.x == -__builtin_inff() ? 0.0f : a.x;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) s += st[w * C::TM + m].y * exp_of(st[w * C::TM + m].x - ref);
      g.part[(m0 + m) * tiles_n + tn] = make_float2(a.x, s);
    }
    return;
  }
  if constexpr (EPI == kSlab) {
    float* out = static_cast<float*>(g.C) + part * rows * g.ldc;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + (wm * MT + i) * 16 + l16;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int64_t n = nl + j * 16;
        if (m >= M || n >= g.N) continue;  // (N is a multiple of 4)
        float4* q = reinterpret_cast<float4*>(out + m * g.ldc + n);
        float4 v = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        if (g.add) {
          const float4 o = *q;
          v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
        }
        *q = v;
      }
    }
    return;
  }
  const float scale = EPI == kFinal ? *g.out_scale : 1.0f;
  if constexpr (EPI == kGrad) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + (wm * MT + i) * 16 + l16;
      const bool in = m < M;
      const float mx = in ? g.rowmax[m] : 0.0f, inv = in ? g.inv[m] : 0.0f, cf = in ? g.coef[m] : 0.0f;
      const float pc = inv * cf;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = exp_of(acc[i][j][r] - mx) * pc;
      const int64_t at = (in ? g.target[m] : -1) - g.v0 - nl;
      if (at >= 0 && at < NT * 16 && (at & 15) < 4) {
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool here = (int)at == j * 16 + r;
            acc[i][j][r] -= here ? cf : 0.0f;
            v = here ? acc[i][j][r] : v;
          }
        if constexpr (k16)
          if (g.dropped) g.dropped[m] = v - half_bits_to_f32(DT, (uint16_t)f32_to_half_bits(DT, v));
      }
    }
    if (g.v0 + n0 + C::TN > g.V) {  // columns past the vocabulary are part of the next products' K
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (g.v0 + nl + j * 16 + r >= g.V) {
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j][r] = 0.0f;
          }
    }
  } else {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] *= scale;
  }
  const int64_t N = g.N;
  if constexpr ((DT == CIN_DT_F32 && EPI == kFinal) || DT == kDirect) {
    float* out = static_cast<float*>(g.C);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + (wm * MT + i) * 16 + l16;
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int64_t n = nl + j * 16;
        if (n + 4 <= N) {
          __builtin_memcpy(out + m * g.ldc + n, &acc[i][j], 16);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < N) out[m * g.ldc + n + r] = acc[i][j][r];
        }
      }
    }
    return;
  }
  // 16-bit rows through LDS, so that the stores run along them; for fp32 one plane after the other
  constexpr int kHalf = DT == CIN_DT_F16 ? CIN_DT_F16 : CIN_DT_BF16;
  constexpr int kChunks = C::TN / 8;
#pragma unroll 1
  for (int plane = 0; plane < (DT == CIN_DT_F32 ? 3 : 1); ++plane) {
    uint16_t* out = static_cast<uint16_t*>(g.C) + plane * g.slab;
#pragma unroll
    for (int part = 0; part < C::kParts; ++part) {
      if (C::kParts == 1 || wm == part) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint2 h = make_uint2(f32x2_to_half2_bits<kHalf>(acc[i][j][0], acc[i][j][1]),
                                       f32x2_to_half2_bits<kHalf>(acc[i][j][2], acc[i][j][3]));
            const int row = ((C::kParts == 1 ? wm : 0) * MT + i) * 16 + l16;
            *reinterpret_cast<uint2*>(smem + row * C::kCStride + ((wn * NT + j) * 16 + kq * 4) * 2) = h;
            if constexpr (DT == CIN_DT_F32) {
              acc[i][j][0] -= bf16_lo(h.x);
              acc[i][j][1] -= bf16_hi(h.x);
              acc[i][j][2] -= bf16_lo(h.y);
              acc[i][j][3] -= bf16_hi(h.y);
            }
          }
      }
      __syncthreads();
      const int64_t mp = m0 + part * C::kPartRows;
      for (int q = tid; q < C::kPartRows * kChunks; q += C::kThreads) {
        const int m = q / kChunks, n = (q % kChunks) * 8;
        if (mp + m >= M || n0 + n >= N) continue;
        const v4u v = *reinterpret_cast<const v4u*>(smem + m * C::kCStride + n * 2);
        uint16_t* d = out + (mp + m) * g.ldc + n0 + n;
        if (n0 + n + 8 <= N) {
          __builtin_memcpy(d, &v, 16);  // (from any element's address)
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n0 + n + e < N) d[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
        }
      }
      if (DT == CIN_DT_F32 || part + 1 < C::kParts) __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
constexpr int kRowPer = 8;  // targets a thread looks at together

// The int32 state: the rows that count, workgroups that are done, whether logits were mended, and T entries
// each of map, pos, target.
struct IntState {
  int *n, *done, *mended, *map, *pos, *target;
  IntState(int32_t* p, int64_t T) : n(p), done(p + 1), mended(p + 2), map(p + 4), pos(map + T), target(pos + T) {}
};

// The rows that count, in order: map[i] the row, target[i] its target (-1 outside the vocabulary),
// pos[t] = i or -1 for an ignored row (whose loss is 0), n their number.  One workgroup of THREADS.
template <int THREADS>
__device__ __forceinline__ int find_rows(const int64_t* __restrict__ y, int64_t T, int64_t V, int64_t ignore,
                                         const IntState& st, float* __restrict__ rowloss, bool write, int* lds_map) {
  __shared__ int wsum[THREADS / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int64_t t0 = 0; t0 < T; t0 += THREADS * kRowPer) {
    // A wave has 64 kRowPer rows in a run, a lane one of each 64, so that loads and stores are whole lines.
    const int64_t first = t0 + (int64_t)wave * 64 * kRowPer + lane;
    int64_t v[kRowPer];
    int before_me[kRowPer], mine = 0;
#pragma unroll
    for (int j = 0; j < kRowPer; ++j) v[j] = first + j * 64 < T ? y[first + j * 64] : ignore;
#pragma unroll
    for (int j = 0; j < kRowPer; ++j) {
      const uint64_t kept = __ballot(v[j] != ignore);
      before_me[j] = mine + __popcll(kept & ((1ull << lane) - 1));
      mine += __popcll(kept);
    }
    if (lane == 0) wsum[wave] = mine;
    __syncthreads();
    int before = base, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) before += wsum[w];
      all += wsum[w];
    }
#pragma unroll
    for (int j = 0; j < kRowPer; ++j) {
      const int64_t t = first + j * 64;
      if (t >= T) break;
      const bool kept = v[j] != ignore;
      const int i = before + before_me[j];
      if (lds_map && kept) lds_map[i] = (int)t;
      if (write) {
        if (kept) {
          st.map[i] = (int)t;
          st.target[i] = v[j] >= 0 && v[j] < V ? (int)v[j] : -1;
        } else {
          rowloss[t] = 0.0f;
        }
        st.pos[t] = kept ? i : -1;
      }
    }
    base += all;
    __syncthreads();
  }
  if (write && tid == 0) {
    *st.n = base;
    *st.done = 0;
    *st.mended = 0;
  }
  return base;
}

__global__ __launch_bounds__(1024) void k_ce_rows(const int64_t* __restrict__ y, int64_t T, int64_t V, int64_t ignore,
                                                  IntState st, float* __restrict__ rowloss) {
  find_rows<1024>(y, T, V, ignore, st, rowloss, true, nullptr);
}

// The next bf16 part of a value, which is taken off it.  A finite value has finite parts (one within half a
// step of 2^128 would round to infinity); an infinity is its own first part and leaves 0.
__device__ __forceinline__ uint32_t take_part(float& v) {
  uint32_t b = f32_to_bf16_bits(v);
  const bool inf = (b & 0x7fff) == 0x7f80;
  if (inf && fabsf(v) < __builtin_inff()) --b;
  v = inf && !(fabsf(v) < __builtin_inff()) ? 0.0f : v - __uint_as_float(b << 16);
  return b;
}

// Rows of x (all, or map's first *n) with zeros up to Dp columns, as operands of DT.
template <int DT>
__device__ __forceinline__ void copy_piece(const void* __restrict__ x, int64_t ldx, int64_t D, int64_t row, int64_t i,
                                           int64_t c, uint16_t* __restrict__ out, int64_t Dp, int64_t plane) {
  using E = std::conditional_t<DT == CIN_DT_F32 || DT == kDirect, float, uint16_t>;
  const E* s = static_cast<const E*>(x) + row * ldx + c;
  uint16_t* d = out + i * Dp + c;
  E v[8];
  if (c + 8 <= D) {
    __builtin_memcpy(v, s, sizeof(v));  // (16 bytes at a time from any element's address)
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < D ? s[e] : (E)0;
  }
  if constexpr (DT == kDirect) {
    __builtin_memcpy(__builtin_assume_aligned(reinterpret_cast<float*>(out) + i * Dp + c, 16), v, 32);
  } else if constexpr (DT == CIN_DT_F32) {
    bool far = false;  // a value that rounds to infinity, or is one
#pragma unroll
    for (int e = 0; e < 8; ++e) far |= fabsf(v[e]) >= 0x1.ffp127f;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      v4u h;
      if (far) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = take_part(v[2 * e]);
          h[e] = lo | take_part(v[2 * e + 1]) << 16;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[e] = f32x2_to_bf16x2_bits(v[2 * e], v[2 * e + 1]);
          v[2 * e] -= bf16_lo(h[e]);
          v[2 * e + 1] -= bf16_hi(h[e]);
        }
      }
      *reinterpret_cast<v4u*>(d + p * plane) = h;
    }
  } else {
    __builtin_memcpy(__builtin_assume_aligned(d, 16), v, 16);
  }
}
template <int DT>
__global__ __launch_bounds__(256) void k_ce_copy(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t D,
                                                 const int* __restrict__ map, const int* __restrict__ n,
                                                 uint16_t* __restrict__ out, int64_t Dp, int64_t plane) {
  const int64_t pieces = Dp / 8, have = n ? *n : rows;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < have * pieces; q += (int64_t)gridDim.x * 256) {
    const int64_t i = q / pieces;
    copy_piece<DT>(x, ldx, D, map ? (int64_t)map[i] : i, i, (q - i * pieces) * 8, out, Dp, plane);
  }
}

// k_ce_rows and k_ce_copy in one launch for few rows: every workgroup finds the rows, the first one
// writes the state.
constexpr int kFewRows = 256 * kRowPer;
template <int DT>
__global__ __launch_bounds__(256) void k_ce_rows_copy(const int64_t* __restrict__ y, int64_t T, int64_t V, int64_t ignore,
                                                      IntState st, float* __restrict__ rowloss, const void* __restrict__ x,
                                                      int64_t ldx, int64_t D, uint16_t* __restrict__ out, int64_t Dp) {
  __shared__ int map[kFewRows];
  const int n = find_rows<256>(y, T, V, ignore, st, rowloss, blockIdx.x == 0, map);
  const uint32_t pieces = (uint32_t)(Dp / 8), total = n * pieces;  // (at most 2^11 x 2^15)
  for (uint32_t q = blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256) {
    const uint32_t i = q / pieces;
    copy_piece<DT>(x, ldx, D, map[i], i, (q - i * pieces) * 8, out, Dp, T * Dp);
  }
}

// Sum of a value a thread over the workgroup, in 64 bits.
__device__ inline double block_sum(double v) {
  __shared__ double w[16];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) s += w[i];
  __syncthreads();
  return s;
}

// The rows' losses added in their order, over their number with `mean` (0 / 0 is NaN).
__device__ __forceinline__ void add_losses(const float* rowloss, int64_t T, int n, int mean, float* loss) {
  double sum = 0;
  for (int64_t t = threadIdx.x; t < T; t += blockDim.x)
    sum += __hip_atomic_load(&rowloss[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  sum = block_sum(sum);
  if (threadIdx.x == 0) *loss = (float)(mean ? sum / n : sum);
}

// The product of rows m of x and n of w that are held in parts, by a wave.
__device__ inline float product_of_parts(const GemmArgs& g, int64_t m, int64_t n, int lane) {
  const uint8_t* x = static_cast<const uint8_t*>(g.A) + m * g.lda * 2;
  const uint8_t* w = static_cast<const uint8_t*>(g.B) + n * g.ldb * 2;
  double s = 0;
  for (int64_t c = lane * 2; c < g.K; c += 128) {
    float a[2] = {0.f, 0.f}, b[2] = {0.f, 0.f};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(x + p * g.plane_a + c * 2);
      const uint32_t v = *reinterpret_cast<const uint32_t*>(w + p * g.plane_b + c * 2);
      a[0] += bf16_lo(u);
      a[1] += bf16_hi(u);
      b[0] += bf16_lo(v);
      b[1] += bf16_hi(v);
    }
    s += (double)a[0] * b[0] + (double)a[1] * b[1];
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
  return (float)s;
}

// Six products of parts make NaN of an infinity: it meets parts of 0 and of either sign.  (So does a sum
// that leaves the range on its way.)  Where a tile's sum is NaN its logits are formed again from whole
// values, here for the statistics and in k_ce_mend for dz: -inf masks an entry of the vocabulary for fp32
// as it does for 16 bits.  (2046 x 32000 x 1024, forward: 0.83 ms, with one such entry 1.73; with 3200 scattered ones,
// in every tile, 111.)  Maximum and sum of row i's such tiles, NaN where the row has a logit that is
// NaN or +inf, at the first of them; its target's logit if it is theirs.
__device__ inline float2 mended_tiles(const GemmArgs& g, const float2* __restrict__ part, int tiles, int tile_n, int64_t i,
                                      int target, int lane, float& ztarget) {
  float m = -__builtin_inff(), s = 0.0f;
  for (int t = 0; t < tiles; ++t) {
    const float y = part[i * tiles + t].y;
    if (y == y) continue;
    const int64_t end = (int64_t)(t + 1) * tile_n < g.V ? (int64_t)(t + 1) * tile_n : g.V;
    for (int64_t v = (int64_t)t * tile_n; v < end; ++v) {
      const float z = product_of_parts(g, i, v, lane);
      if (!(z < __builtin_inff())) return make_float2(__builtin_nanf(""), __builtin_nanf(""));
      if (v == target) ztarget = z;
      if (z == -__builtin_inff()) continue;
      if (z > m) {
        s = s * exp_of(m - z) + 1.0f;
        m = z;
      } else {
        s += exp_of(z - m);
      }
    }
  }
  return make_float2(m, s);
}

// A wave per row: the tiles' maxima and sums joined, the row's loss (NaN for a target outside the
// vocabulary).  With `loss`, for few rows, the workgroup that ends last adds them up; for more a
// launch of its own does, as each workgroup's fence costs more than it (4096 rows: 34 us of forward
// with the launch, 107 without).
// PARTS: operands are held in parts, tile_n columns a tile.
struct NoArgs {};
template <bool PARTS>
__global__ __launch_bounds__(256) void k_ce_join(std::conditional_t<PARTS, GemmArgs, NoArgs> g, int tile_n,
                                                 const float2* __restrict__ part, int tiles, int64_t T, IntState st,
                                                 const float* __restrict__ ztarget, float* __restrict__ rowmax,
                                                 float* __restrict__ inv, float* __restrict__ rest,
                                                 float* __restrict__ rowloss, int mean,
                                                 float* __restrict__ loss) {
  const int lane = threadIdx.x & 63, n = *st.n;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i < n) {
    float m = -__builtin_inff(), s = 0.0f, zt = 0.0f;
    bool mend = false;
    float2 more;
    if constexpr (PARTS) {
      zt = ztarget[i];
      for (int t = lane; t < tiles; t += 64) {
        const float2 p = part[i * tiles + t];
        if (p.y == p.y)
          m = fmaxf(m, p.x);
        else
          mend = true;
      }
      mend = __ballot(mend) != 0;
      if (mend) {
        more = mended_tiles(g, part, tiles, tile_n, i, st.target[i], lane, zt);
        m = fmaxf(m, more.x);
      }
    } else {
      for (int t = lane; t < tiles; t += 64) m = fmaxf(m, part[i * tiles + t].x);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    for (int t = lane; t < tiles; t += 64) {
      const float2 p = part[i * tiles + t];
      if (!mend || p.y == p.y) s += p.y * exp_of(p.x - m);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
    if (mend) {
      s += more.y * exp_of(more.x - m);
      if (lane == 0 && s == s) *st.mended = 1;
    }
    if (lane == 0) {
      const float loss_i = st.target[i] < 0 ? __builtin_nanf("") : (m - (PARTS ? zt : ztarget[i])) + logf(s);
      rowmax[i] = m;
      inv[i] = 1.0f / s;
      rest[i] = -expm1f(-loss_i);
      rowloss[st.map[i]] = loss_i;
    }
  }
  if (!loss) return;
  __shared__ int before;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) before = __hip_atomic_fetch_add(st.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (before != (int)gridDim.x - 1) return;
  __threadfence();
  add_losses(rowloss, T, n, mean, loss);
}
constexpr int kJoinAlone = 64;  // rows up to which it does

__global__ __launch_bounds__(1024) void k_ce_loss(const float* __restrict__ rowloss, int64_t T, const int* __restrict__ n,
                                                  int mean, float* __restrict__ loss) {
  add_losses(rowloss, T, *n, mean, loss);
}

// What dz is scaled by: coef[i] = g_i 2^a with all products in range (fp16 holds 2^-24 .. 65504,
// and p - 1 lies in [-1, 1]: top 2^15), and out_scale = 2^-a times what all rows share.  A gradient
// shared by all rows (stride 0) stays out of coef.
struct Coef {
  float s, out;
};
// By the whole workgroup.
template <int THREADS>
__device__ inline Coef coef_of(const float* __restrict__ grad, int64_t stride, int mean, float top, int rows,
                               const int* __restrict__ map) {
  __shared__ float wmax[THREADS / 64];
  Coef c{top, 1.0f / top};
  if (stride == 0) {
    c.out *= mean ? grad[0] / (float)rows : grad[0];
    return c;
  }
  float m = 0.0f;
  for (int i = threadIdx.x; i < rows; i += THREADS) m = fmaxf(m, fabsf(grad[(int64_t)map[i] * stride]));
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = m;
  __syncthreads();
  for (int w = 0; w < THREADS / 64; ++w) m = fmaxf(m, wmax[w]);
  if (m > 0.0f && m < __builtin_inff()) {
    int e;
    frexpf(m, &e);  // m <= 2^e
    e = e < -100 ? -100 : (e > 100 ? 100 : e);
    c.s = ldexpf(top, -e);
    c.out = ldexpf(1.0f / top, e);
  }
  return c;
}

// Where the backward leaves what its products are scaled by.
struct Scales {
  float *out, *coef, *row;  // row: for few rows, null for many
  float* dropped;           // for many of 16 bits, else null
  int* slabs;
};

// And dx's slabs.  One workgroup.
__global__ __launch_bounds__(1024) void k_ce_coef(const float* __restrict__ grad, int64_t stride, int mean, int half,
                                                  const int* __restrict__ n, const int* __restrict__ map,
                                                  const int* __restrict__ target, Scales to, Slabs slabs) {
  const int rows = *n;
  const Coef c = coef_of<1024>(grad, stride, mean, half ? 32768.0f : 1.0f, rows, map);
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = stride == 0 ? c.s : grad[(int64_t)map[i] * stride] * c.s;
    to.coef[i] = target[i] < 0 ? __builtin_nanf("") : g;
  }
  if (threadIdx.x == 0) {
    *to.out = rows ? c.out : 0.0f;
    *to.slabs = slabs.count(rows);
  }
}

// The same for few rows.  A row's largest entry of dz is its target's, g (p - 1), and with few rows the
// rounding of those few numbers does not average out of dx and dw.  So dz is divided by 1 - p, which
// makes that entry a power of two, and c = g (1 - p) = 2^e m, m in [1/2, 1), is brought in by other ways:
// 2^e with dz, m in fp32 with dx's sums and, for dw, with x, held as two 16-bit parts.  The gradients are
// then as near as their own rounding allows (relative error of 16 x 32000 x 1024, bf16, a gradient for
// each row: 1.65e-3, without it 2.5e-3).  dw takes twice the products: of x 32000 x 1024 backward 59 -> 63
// us with 64 rows, 72 -> 82 with 128, 104 -> 121 with 256, and 140 -> 174 with 512, too many for it (see
// add_dropped for those).
constexpr int kFewExact = 256;
template <int DT>
__global__ __launch_bounds__(256) void k_ce_coef_few(const float* __restrict__ grad, int64_t stride, int mean,
                                                     const int* __restrict__ n, const int* __restrict__ map,
                                                     const int* __restrict__ target, const float* __restrict__ rest,
                                                     Scales to, Slabs slabs, const uint16_t* __restrict__ x, int64_t Dp,
                                                     uint16_t* __restrict__ scaled, int64_t plane) {
  constexpr float top = DT == CIN_DT_F16 ? 32768.0f : 1.0f;
  constexpr int kLeast = DT == CIN_DT_F16 ? -24 : -60;  // of e: dz's powers of two stay in its type
  const int rows = *n;
  const Coef c = coef_of<256>(grad, stride, mean, top, rows, map);
  // m and e of row i; r: its 1 - p, kept from 0 (the row's other entries are then at most 1 too)
  const auto row = [&](int i, int& e, float& r) {
    r = fmaxf(rest[i], 5.9604644775390625e-8f);
    const float v = (stride == 0 ? 1.0f : grad[(int64_t)map[i] * stride] * (c.s / top)) * r;
    e = 0;
    if (!(fabsf(v) < 1.0f)) return v;  // (1, NaN or infinite)
    frexpf(v, &e);
    e = v == 0.0f ? 0 : (e < kLeast ? kLeast : (e > 0 ? 0 : e));
    return ldexpf(v, -e);
  };
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < rows; i += 256) {
      int e;
      float r;
      to.row[i] = row(i, e, r);
      to.coef[i] = target[i] < 0 ? __builtin_nanf("") : ldexpf(top, e) / r;
    }
    if (threadIdx.x == 0) {
      *to.out = rows ? c.out : 0.0f;
      *to.slabs = slabs.count(rows);
    }
  }
  const uint32_t pieces = (uint32_t)(Dp / 8), total = rows * pieces;  // (at most 2^8 x 2^15)
  for (uint32_t q = blockIdx.x * 256 + threadIdx.x; q < total; q += gridDim.x * 256) {
    const uint32_t i = q / pieces;
    int e;
    float r;
    const float m = row((int)i, e, r);
    const int64_t at = i * Dp + (q - i * pieces) * 8;
    const v4u v = *reinterpret_cast<const v4u*>(x + at);
    v4u hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = half_bits_to_f32(DT, (uint16_t)v[k]) * m, b = half_bits_to_f32(DT, (uint16_t)(v[k] >> 16)) * m;
      hi[k] = f32x2_to_half2_bits<DT>(a, b);
      lo[k] = f32x2_to_half2_bits<DT>(a - half_bits_to_f32(DT, (uint16_t)hi[k]), b - half_bits_to_f32(DT, (uint16_t)(hi[k] >> 16)));
    }
    *reinterpret_cast<v4u*>(scaled + at) = hi;
    *reinterpret_cast<v4u*>(scaled + plane + at) = lo;
  }
}

// dz of the logits that are formed again (see mended_tiles), as kGrad's: a wave looks at 64 columns of a row.
__global__ __launch_bounds__(256) void k_ce_mend(GemmArgs g, const int* __restrict__ mended) {
  if (!*mended) return;
  const int lane = threadIdx.x & 63;
  const int64_t cols = g.N < g.V - g.v0 ? g.N : g.V - g.v0, chunks = cdiv(cols, 64), total = *g.n * chunks;
  for (int64_t q = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); q < total; q += (int64_t)gridDim.x * 4) {
    const int64_t i = q / chunks, c0 = (q - i * chunks) * 64;
    const float mx = g.rowmax[i], inv = g.inv[i], cf = g.coef[i], pc = inv * cf;
    if (!(pc == pc)) continue;  // the row's own loss or gradient is NaN
    uint16_t* d = static_cast<uint16_t*>(g.C) + i * g.ldc + c0 + lane;
    uint64_t nans = __ballot(c0 + lane < cols && (*d & 0x7fff) > 0x7f80);
    for (; nans; nans &= nans - 1) {
      const int at = __builtin_ctzll(nans);
      const float z = product_of_parts(g, i, c0 + at, lane);
      float v = exp_of(z - mx) * pc - (g.target[i] == g.v0 + c0 + at ? cf : 0.0f);
      if (lane == at) {
#pragma unroll
        for (int p = 0; p < 3; ++p) d[p * g.slab] = (uint16_t)take_part(v);
      }
    }
  }
}

// dz of a piece of the vocabulary from kept logits, as kGrad's: for few rows they are fewer bytes than the
// weight (20 x 100000 x 2048, forward and gradients: bf16 441 -> 371 us, fp32 819 -> 681).
template <int DT>
__global__ __launch_bounds__(256) void k_ce_grad(const float* __restrict__ z, int64_t ldl, GemmArgs g) {
  using E = std::conditional_t<DT == kDirect, float, uint16_t>;
  const uint32_t pieces = (uint32_t)(g.N / 8);
  const int64_t total = (int64_t)*g.n * pieces;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t i = q / pieces, c = (q - i * pieces) * 8;
    const float mx = g.rowmax[i], cf = g.coef[i], pc = g.inv[i] * cf;
    const int64_t at = (int64_t)g.target[i] - g.v0 - c;
    float v[8];
    __builtin_memcpy(v, __builtin_assume_aligned(z + i * ldl + g.v0 + c, 16), 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = exp_of(v[e] - mx) * pc - (at == e ? cf : 0.0f);
      if (g.v0 + c + e >= g.V) v[e] = 0.0f;
    }
    E* d = static_cast<E*>(g.C) + i * g.ldc + c;
    if constexpr (DT == kDirect) {
      __builtin_memcpy(__builtin_assume_aligned(d, 16), v, 32);
    } else {
      v4u h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = f32x2_to_half2_bits<DT>(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<v4u*>(d) = h;
    }
  }
}

// dx[t] = out_scale (row[pos[t]]) times the sum of the slabs' row pos[t] (and what dz's rounding dropped
// times the target's row of w), zero for an ignored row.
template <int DT>
__global__ __launch_bounds__(256) void k_ce_dx(const float* __restrict__ slabs, Scales by, const int* __restrict__ n, int64_t Dp,
                                               const int* __restrict__ pos, const int* __restrict__ target,
                                               const void* __restrict__ w, int64_t ldw,
                                               int64_t T, int64_t D, void* __restrict__ dx) {
  const float shared = *by.out;
  const int splits = *by.slabs;
  const int64_t slab = *n * Dp, pieces = Dp / 4;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < T * pieces; q += (int64_t)gridDim.x * 256) {
    const int64_t t = q / pieces, c = (q - t * pieces) * 4;
    if (c >= D) continue;
    const int i = pos[t];
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i >= 0) {
      for (int s = 0; s < splits; ++s) {
        const float4 b = *reinterpret_cast<const float4*>(slabs + s * slab + i * Dp + c);
        a = make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
      }
      if constexpr (DT != CIN_DT_F32) {
        const int y = target[i];
        if (by.dropped && y >= 0) {
          const float r = by.dropped[i];
          const uint2 h = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w) + y * ldw + c);
          a.x += r * half_bits_to_f32(DT, (uint16_t)h.x);
          a.y += r * half_bits_to_f32(DT, (uint16_t)(h.x >> 16));
          a.z += r * half_bits_to_f32(DT, (uint16_t)h.y);
          a.w += r * half_bits_to_f32(DT, (uint16_t)(h.y >> 16));
        }
      }
    }
    const float scale = by.row && i >= 0 ? shared * by.row[i] : shared;
    const float v[4] = {a.x * scale, a.y * scale, a.z * scale, a.w * scale};
    const int64_t at = t * D + c;
    if constexpr (DT == CIN_DT_F32) {
      float* d = static_cast<float*>(dx) + at;
      if (c + 4 <= D)
        __builtin_memcpy(d, v, 16);
      else
        for (int e = 0; e < 4; ++e)
          if (c + e < D) d[e] = v[e];
    } else {
      uint16_t* d = static_cast<uint16_t*>(dx) + at;
      const uint2 h = make_uint2(f32x2_to_half2_bits<DT>(v[0], v[1]), f32x2_to_half2_bits<DT>(v[2], v[3]));
      if (c + 4 <= D)
        __builtin_memcpy(d, &h, 8);
      else
        for (int e = 0; e < 4; ++e)
          if (c + e < D) d[e] = (uint16_t)((e < 2 ? h.x : h.y) >> (16 * (e & 1)));
    }
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Tiles.  Wide ones read their operands less often and keep the matrix units busier (without loads
// the 256 x 256 tile's loop runs at 1.62 PFLOP/s, with operands that hit the L2 at 1.32, at full length
// at 1.23); narrow ones leave fewer compute units idle in a small product, and the narrowest, with more
// steps on their way, stream w for a few rows (16 x 100000 x 2048 of fp32, forward: 188 us with the 32 x 64
// tile, 266 with 64 x 64).  8192 x 131072 x 4096, bf16: x w^T 1.32 and 1.24 PFLOP/s
// with the two widest; 16368 x 32000 x 1024: 1.07 and 0.97, 0.89 with 128 x 128.
using Widest = Cfg<2, 4, 8, 6, 2>;  // 256 x 384, 8 waves of 128 x 96: 250 registers, all of the LDS
using Wide = Cfg<2, 4, 8, 4, 2>;    // 256 x 256, 8 waves of 128 x 64
using Medium = Cfg<2, 2, 4, 4, 2>;  // 128 x 128, 4 waves of 64 x 64, two workgroups a CU
// (two workgroups a CU of these where operands are one plane; with all parts of fp32 in a step, one)
using Narrow = Cfg<1, 4, 4, 1, 4>;  // 64 x 64, 4 waves of 64 x 16
using Thin = Cfg<1, 4, 2, 1, 6>;    // 32 x 64, 4 waves of 32 x 16: up to 32 rows, few tiles
constexpr int kTiles = 5;
constexpr int kTileM[kTiles] = {Widest::TM, Wide::TM, Medium::TM, Narrow::TM, Thin::TM};
constexpr int kTileN[kTiles] = {Widest::TN, Wide::TN, Medium::TN, Narrow::TN, Thin::TN};
constexpr int kTileThreads[kTiles] = {Widest::kThreads, Wide::kThreads, Medium::kThreads, Narrow::kThreads, Thin::kThreads};
// A tile's rate against that of the 256 x 256 ones.  With full grids, forward of 8192 x 24576 x 4096 in bf16: 1387,
// 1262, 1095, 631 and 458 TFLOP/s, that is 1.10, 1, 0.87, 0.50 and 0.36 (fp16 the same within 1%; 8192 x 24576 x 1024:
// 1.11, 1, 0.92, 0.45, 0.32; fp32 in parts, 4096 x 24576 x 1024: 1.08, 1, 0.89, 0.61, 0.48).  The narrower ones have
// that from several workgroups on a CU; one on each (4096 x 4096, 2048 x 2048, 1024 x 1024 and 512 x 1024 rows and
// columns, K 8192) gives 0.6, 0.3 and 0.2, as their rounds are counted here, and they are taken in between.
constexpr double kTileRate[kTiles] = {1.08, 1.0, 0.75, 0.4, 0.25};

// The time of m x n outputs in parts of K, in units of one output's share at the 256 x 256 tile's rate.
double tile_time(int tile, int64_t m, int64_t n, double parts, double part) {
  const double count = (double)cdiv(m, kTileM[tile]) * (double)cdiv(n, kTileN[tile]) * parts;
  const double rounds = ceil(count / cin_device_cus());
  return rounds * kTileM[tile] * kTileN[tile] / kTileRate[tile] * part;
}
// fp32 operands of 4 bytes come for few rows only, and in the three smaller tiles.
int first_tile(int op) { return op == kDirect ? 2 : 0; }
int pick_tile(int op, int64_t m, int64_t n, int first = 0) {
  int best = first_tile(op) > first ? first_tile(op) : first;
  for (int t = best + 1; t < kTiles; ++t)
    if (tile_time(t, m, n, 1, 1) < tile_time(best, m, n, 1, 1)) best = t;
  return best;
}
// dw's: no wider ones, where its product runs as fast (8192 x 65536 x 4096: 3.43 ms with the widest, 3.45 with
// 256 x 256) and add_dropped would take registers from its loop (3.68 ms).
int pick_dw_tile(int op, int64_t m, int64_t n) { return pick_tile(op, m, n, 1); }
template <int DT, int EPI, class F>
void with_tile(int tile, F f) {
  if constexpr (DT != kDirect) {
    if constexpr (EPI != kFinal)
      if (tile == 0) return f(Widest{});
    if (tile <= 1) return f(Wide{});
  }
  if (tile <= 2)
    f(Medium{});
  else if (tile == 3)
    f(Narrow{});
  else
    f(Thin{});
}

// A launch has fewer than 2^32 threads: k_ce_join takes 64 a row.
constexpr int64_t kMaxT = ((int64_t)1 << 26) - 4, kMaxV = (int64_t)1 << 29, kMaxD = (int64_t)1 << 18;
constexpr int64_t kPieceBytes = (int64_t)1 << 30;  // dz of one piece
constexpr int64_t kMaxPiece = (int64_t)1 << 20;    // its columns: 256 rows lie within 2^31 bytes

int64_t align_up(int64_t v, int64_t a) { return cdiv(v, a) * a; }
constexpr int64_t kAlign = 256;  // columns of a piece: whole tiles

// fp32 with so few rows is multiplied as it is: its products are bound by reading w, which three planes
// more than double, and w needs no copy of three (forward of 16 x 100000 x 2048: 187 us, in parts 675; with
// gradients 678 and 1435; of 128: 533 and 998, 1504 and 2668; of 256: 938 and 1113, but 3614 and 3178).
constexpr int64_t kDirectRows = 128;

struct Plan {
  int op;               // what the operands hold
  int planes, es;       // of an operand: 3 for fp32 in parts; bytes of an element
  int64_t Dp;           // columns of x and w as the products read them
  int tile;             // of the forward product
  int64_t tiles_n;      // its column tiles
  int64_t piece, ldz;   // columns of a piece, elements between rows of dz
  int splits, slab_tile;  // slabs of dx if all rows count, the tile of its product
  Slabs split;
  // bytes
  int64_t part, ztarget, dz, slabs, scaled, coef;
  bool few;  // rows: k_ce_coef_few
};

Plan make_plan(int dtype, int64_t T, int64_t D, int64_t V) {
  Plan p;
  const int64_t Tp = T > 0 ? T : 1;
  p.op = dtype == CIN_DT_F32 && Tp <= kDirectRows ? kDirect : dtype;
  p.planes = p.op == CIN_DT_F32 ? 3 : 1;
  p.es = p.op == kDirect ? 4 : 2;
  p.Dp = align_up(D, kPadK);
  p.tile = pick_tile(p.op, Tp, V);
  p.tiles_n = cdiv(V, kTileN[p.tile]);
  int64_t most = align_up(kPieceBytes / (Tp * p.es * p.planes) + 1, kAlign);
  if (most > kMaxPiece) most = kMaxPiece;
  const int64_t pieces = cdiv(V, most);
  p.piece = align_up(cdiv(V, pieces), kAlign);
  p.ldz = p.piece + 64;  // rows not a multiple of 16 KiB apart
  // dx: K, the piece, is split where the tiles are fewer than the CUs, in parts of 8 steps at least
  const int64_t steps = p.piece / kPadK;
  double best = 0;
  for (int t = first_tile(p.op); t < kTiles; ++t) {
    const int64_t count = cdiv(Tp, kTileM[t]) * cdiv(p.Dp, kTileN[t]);
    int64_t s = cin_device_cus() / count;
    if (s > steps / 8) s = steps / 8;
    if (s < 1) s = 1;
    const double time = tile_time(t, Tp, p.Dp, (double)s, 1.0 / s);
    if (t == first_tile(p.op) || time < best) {
      best = time;
      p.splits = (int)s;
      p.slab_tile = t;
    }
  }
  const int64_t slab_n = cdiv(p.Dp, kTileN[p.slab_tile]), workgroups = cdiv(Tp, kTileM[p.slab_tile]) * slab_n * p.splits;
  p.split = Slabs{kTileM[p.slab_tile], (int)slab_n, (int)(workgroups < cin_device_cus() ? workgroups : cin_device_cus()),
                  (int)(steps / 8), Tp * p.splits};
  p.part = align_up(Tp * p.tiles_n * 8, 256);
  p.ztarget = align_up(Tp * 4, 256);
  p.dz = align_up(p.planes * Tp * p.ldz * p.es, 256);
  p.slabs = align_up(p.splits * Tp * p.Dp * 4, 256);
  p.few = dtype != CIN_DT_F32 && Tp <= kFewExact;
  p.scaled = p.few ? align_up(2 * Tp * p.Dp * p.es, 256) : 0;
  p.coef = align_up((2 * Tp + 2) * 4, 256);
  return p;
}

// Whether a product's launch has fewer than 2^32 threads.
bool grid_fits(int tile, int64_t m, int64_t n) {
  return (double)cdiv(m, kTileM[tile]) * (double)cdiv(n, kTileN[tile]) * kTileThreads[tile] < 4294967296.0;
}

int check(const char* name, int dtype, int64_t T, int64_t D, int64_t V, Plan& p) {
  CIN_CHECK_ARG(dtype == CIN_DT_BF16 || dtype == CIN_DT_F32 || dtype == CIN_DT_F16, "%s: bad dtype %d", name, dtype);
  CIN_CHECK_ARG(T >= 0 && T <= kMaxT, "%s: T must be in [0, 2^26 - 4]", name);
  CIN_CHECK_ARG(V >= 1 && V <= kMaxV, "%s: V must be in [1, 2^29]", name);
  CIN_CHECK_ARG(D >= 1 && D <= kMaxD, "%s: D must be in [1, 2^18]", name);
  // (the products over a piece of the vocabulary are smaller: T x piece < 2^30 + 256 T)
  p = make_plan(dtype, T, D, V);
  CIN_CHECK_ARG(grid_fits(p.tile, T, V) && grid_fits(p.slab_tile, T, p.Dp) && grid_fits(pick_dw_tile(p.op, p.piece, D), p.piece, D),
                "%s: T x V, T x D or V x D is too large", name);
  return CIN_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool w_fits(const void* w, int64_t ldw, int es) {
  return aligned16(w) && ldw * es % 16 == 0 && ldw <= 4 * kMaxD;
}

template <class F>
void with_dtype(int dtype, F f) {
  if (dtype == CIN_DT_F32)
    f(std::integral_constant<int, CIN_DT_F32>{});
  else if (dtype == CIN_DT_F16)
    f(std::integral_constant<int, CIN_DT_F16>{});
  else
    f(std::integral_constant<int, CIN_DT_BF16>{});
}

// The same for what the operands hold.
template <class F>
void with_op(int op, F f) {
  if (op == kDirect)
    f(std::integral_constant<int, kDirect>{});
  else
    with_dtype(op, f);
}

template <int EPI>
void gemm(int op, int tile, const GemmArgs& g, int64_t max_m, int splits, hipStream_t s) {
  with_op(op, [&](auto dt) {
    with_tile<dt(), EPI>(tile, [&](auto c) {
      using C = decltype(c);
      const int64_t tiles = cdiv(max_m, C::TM) * cdiv(g.N, C::TN) * splits;
      hipLaunchKernelGGL((k_ce_gemm<C, dt(), EPI>), (unsigned)tiles, C::kThreads, 0, s, g);
    });
  });
}

void copy_rows(int op, const void* x, int64_t ldx, int64_t rows, int64_t D, const int* map, const int* n, void* out,
               int64_t Dp, hipStream_t s) {
  const int64_t blocks = cdiv(rows * (Dp / 8), 256);
  const unsigned grid = (unsigned)(blocks < 8192 ? blocks : 8192);
  // (16-bit elements are copied, whichever they are)
  with_op(op == CIN_DT_F16 ? CIN_DT_BF16 : op, [&](auto dt) {
    hipLaunchKernelGGL(k_ce_copy<dt()>, grid, 256, 0, s, x, ldx, rows, D, map, n, static_cast<uint16_t*>(out), Dp, rows * Dp);
  });
}

}  // namespace

extern "C" {

int64_t cin_linear_ce_workspace(int dtype, int64_t T, int64_t D, int64_t V, int backward) {
  Plan p;
  if (check("linear_ce_workspace", dtype, T, D, V, p)) return -1;
  return backward ? p.dz + p.slabs + p.scaled + p.coef : p.part + p.ztarget;
}

int cin_linear_ce_forward(const void* x, int dtype, int64_t T, int64_t D, int64_t ldx, const void* w, int64_t V,
                          int64_t ldw, const int64_t* target, int64_t ignore_index, int mean, void* xc, void* wp,
                          int32_t* state_i, float* state_f, float* rowloss, float* loss, void* workspace,
                          int64_t workspace_bytes, float* logits, void* stream) {
  const char* name = "linear_ce_forward";
  Plan p;
  if (int rc = check(name, dtype, T, D, V, p)) return rc;
  CIN_CHECK_ARG(ldx >= D && ldw >= D, "%s: rows overlap", name);
  CIN_CHECK_ARG(state_i && w && (T == 0 || (x && target && xc && state_f && rowloss)), "%s: null pointer", name);
  CIN_CHECK_ARG(wp || (p.planes == 1 && w_fits(w, ldw, p.es) && p.Dp == D), "%s: w needs a padded copy", name);
  CIN_CHECK_ARG(aligned16(xc) && aligned16(wp) && aligned16(workspace) && aligned16(logits),
                "%s: xc, wp, workspace and logits must lie on 16 bytes", name);
  CIN_CHECK_ARG(workspace_bytes >= p.part + p.ztarget && workspace, "%s: workspace needs %lld bytes", name,
                (long long)(p.part + p.ztarget));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const IntState st(state_i, T);
  float2* part = static_cast<float2*>(workspace);
  float* zt = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.part);
  if (T == 0 || T > kFewRows)
    hipLaunchKernelGGL(k_ce_rows, 1, 1024, 0, s, target, T, V, ignore_index, st, rowloss);
  GemmArgs g{};
  if (T > 0) {
    if (T > kFewRows) {
      copy_rows(p.op, x, ldx, T, D, st.map, st.n, xc, p.Dp, s);
    } else {
      const unsigned grid = (unsigned)cdiv(T * (p.Dp / 8), 256);
      with_op(p.op == CIN_DT_F16 ? CIN_DT_BF16 : p.op, [&](auto dt) {
        hipLaunchKernelGGL(k_ce_rows_copy<dt()>, grid < 256 ? grid : 256, 256, 0, s, target, T, V, ignore_index, st, rowloss,
                           x, ldx, D, static_cast<uint16_t*>(xc), p.Dp);
      });
    }
    if (wp) copy_rows(p.op, w, ldw, V, D, nullptr, nullptr, wp, p.Dp, s);
    g.A = xc;
    g.lda = p.Dp;
    g.B = wp ? wp : w;
    g.ldb = wp ? p.Dp : ldw;
    g.plane_a = T * p.Dp * p.es;
    g.plane_b = V * p.Dp * p.es;
    g.N = g.V = V;
    g.K = p.Dp;
    g.n = st.n;
    g.part = part;
    g.ztarget = zt;
    g.target = st.target;
    g.C = logits;
    g.ldc = align_up(V, kPadK);
    gemm<kStats>(p.op, p.tile, g, T, 1, s);
  }
  // (without rows one workgroup: the sum of none)
  const unsigned rows4 = (unsigned)(T > 0 ? cdiv(T, 4) : 1);
  float* here = T <= kJoinAlone ? loss : nullptr;
  if (p.planes > 1)
    hipLaunchKernelGGL(k_ce_join<true>, rows4, 256, 0, s, g, kTileN[p.tile], part, (int)p.tiles_n, T, st, zt, state_f, state_f + T,
                       state_f + 2 * T, rowloss, mean, here);
  else
    hipLaunchKernelGGL(k_ce_join<false>, rows4, 256, 0, s, NoArgs{}, 0, part, (int)p.tiles_n, T, st, zt, state_f, state_f + T,
                       state_f + 2 * T, rowloss, mean, here);
  if (loss && T > kJoinAlone) hipLaunchKernelGGL(k_ce_loss, 1, 1024, 0, s, rowloss, T, st.n, mean, loss);
  return cin_check_launch(name);
}

int cin_linear_ce_backward(const void* xc, int dtype, int64_t T, int64_t D, const void* w, int64_t V, int64_t ldw,
                           const int32_t* state_i, const float* state_f, const float* grad, int64_t grad_stride,
                           int mean, void* dx, void* dw, void* workspace, int64_t workspace_bytes,
                           const float* logits, void* stream) {
  const char* name = "linear_ce_backward";
  Plan p;
  if (int rc = check(name, dtype, T, D, V, p)) return rc;
  CIN_CHECK_ARG(w_fits(w, ldw, p.es) && (p.planes > 1 ? ldw == p.Dp : ldw >= p.Dp),
                "%s: w's rows must be padded as the forward's", name);
  CIN_CHECK_ARG(grad_stride >= 0, "%s: negative gradient stride", name);
  CIN_CHECK_ARG(T > 0 && state_i && state_f && xc && w && grad, "%s: null pointer", name);
  CIN_CHECK_ARG(aligned16(xc) && aligned16(dx) && aligned16(workspace) && aligned16(logits),
                "%s: xc, dx, workspace and logits must lie on 16 bytes", name);
  CIN_CHECK_ARG(!logits || p.planes == 1, "%s: fp32 with this many rows takes no logits", name);
  CIN_CHECK_ARG(workspace && workspace_bytes >= p.dz + p.slabs + p.scaled + p.coef, "%s: workspace needs %lld bytes", name,
                (long long)(p.dz + p.slabs + p.scaled + p.coef));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const IntState st(const_cast<int32_t*>(state_i), T);
  char* ws = static_cast<char*>(workspace);
  void* dz = ws;
  float* slabs = reinterpret_cast<float*>(ws + p.dz);
  uint16_t* scaled = reinterpret_cast<uint16_t*>(ws + p.dz + p.slabs);
  float* f = reinterpret_cast<float*>(ws + p.dz + p.slabs + p.scaled);
  float* rows = f + 2 + T;
  const Scales by{f, f + 2, p.few ? rows : nullptr, !p.few && dtype != CIN_DT_F32 ? rows : nullptr, reinterpret_cast<int*>(f + 1)};
  if (p.few) {
    const unsigned grid = (unsigned)cdiv(T * (p.Dp / 8), 256);
    with_dtype(dtype, [&](auto dt) {
      if constexpr (dt() != CIN_DT_F32)
        hipLaunchKernelGGL(k_ce_coef_few<dt()>, grid < 256 ? grid : 256, 256, 0, s, grad, grad_stride, mean, st.n, st.map,
                           st.target, state_f + 2 * T, by, p.split, static_cast<const uint16_t*>(xc), p.Dp, scaled, T * p.Dp);
    });
  } else {
    hipLaunchKernelGGL(k_ce_coef, 1, 1024, 0, s, grad, grad_stride, mean, dtype == CIN_DT_F16, st.n, st.map, st.target, by,
                       p.split);
  }
  const char* wb = static_cast<const char*>(w);
  for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
    const int64_t cols = v0 + p.piece < V ? p.piece : V - v0;
    GemmArgs g{};
    g.A = xc;
    g.lda = p.Dp;
    g.B = wb + v0 * ldw * p.es;
    g.ldb = ldw;
    g.plane_a = T * p.Dp * p.es;
    g.plane_b = V * p.Dp * p.es;
    g.N = align_up(cols, kPadK);  // with the zeros that fill the next product's last K step
    g.K = p.Dp;
    g.n = st.n;
    g.C = dz;
    g.ldc = p.ldz;
    g.slab = T * p.ldz;
    g.v0 = v0;
    g.V = V;
    g.target = st.target;
    g.rowmax = state_f;
    g.inv = state_f + T;
    g.coef = by.coef;
    g.dropped = by.dropped;
    if (logits) {
      const int64_t blocks = cdiv(T * (g.N / 8), 256);
      with_op(p.op, [&](auto dt) {
        if constexpr (dt() != CIN_DT_F32)
          hipLaunchKernelGGL(k_ce_grad<dt()>, (unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, s, logits,
                             align_up(V, kPadK), g);
      });
    } else {
      gemm<kGrad>(p.op, pick_tile(p.op, T, g.N), g, T, 1, s);
      if (p.planes > 1) hipLaunchKernelGGL(k_ce_mend, 256, 256, 0, s, g, st.mended);
    }
    GemmArgs h{};
    h.n = st.n;
    h.A = dz;
    h.lda = p.ldz;
    h.wa = p.ldz;
    h.wb = p.Dp;
    h.plane_a = T * p.ldz * p.es;
    h.v0 = v0;
    h.V = V;
    if (dx) {
      h.B = g.B;
      h.ldb = ldw;
      h.plane_b = g.plane_b;
      h.N = p.Dp;
      h.K = g.N;
      h.slabs = by.slabs;
      h.C = slabs;
      h.ldc = p.Dp;
      h.add = v0 > 0;
      gemm<kSlab>(p.op, p.slab_tile, h, T, p.splits, s);
    }
    if (dw) {
      h.B = p.few ? scaled : xc;
      h.segs = p.few ? 2 : 1;
      h.ldb = p.Dp;
      h.plane_b = g.plane_a;
      h.M = cols;
      h.N = D;
      h.C = static_cast<char*>(dw) + v0 * D * (dtype == CIN_DT_F32 ? 4 : 2);
      h.ldc = D;
      h.out_scale = by.out;
      h.target = st.target;
      h.dropped = by.dropped;
      gemm<kFinal>(p.op, pick_dw_tile(p.op, cols, D), h, cols, 1, s);
    }
  }
  if (dx) {
    const int64_t blocks = cdiv(T * (p.Dp / 4), 256);
    with_dtype(dtype, [&](auto dt) {
      hipLaunchKernelGGL(k_ce_dx<dt()>, (unsigned)(blocks < 16384 ? blocks : 16384), 256, 0, s, slabs, by, st.n,
                         p.Dp, st.pos, st.target, w, ldw, T, D, dx);
    });
  }
  return cin_check_launch(name);
}

}  // extern "C"
