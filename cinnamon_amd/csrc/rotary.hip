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

// One of the two tensors, [B, L, heads, D] with unit channel stride.
struct Side {
  const void* x;
  void* y;
  int64_t xb, xl, xh, yb, yl, yh;
  int64_t heads;
};

struct RotaryArgs {
  Side q, k;
  int64_t B, L, D;
  const float *cos, *sin;
  int64_t P, ldt;
  int rot, start;
  const int64_t* positions;
  int64_t pb, pl;
  int interleaved, inverse;
};

template <int DT>
__device__ inline void store_elem(void* p, int64_t i, float v) {
  if constexpr (DT == CIN_DT_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_half_bits(DT, v);
}

// One thread per rotated pair or copied channel.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryArgs a) {
  const int half = a.rot / 2;
  const int64_t units = a.D - half;  // pairs first, then the copied channels
  const int64_t heads = a.q.heads + a.k.heads;
  const int64_t n = a.B * a.L * heads * units;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int64_t u = i % units, h = i / units % heads, tok = i / units / heads;
    const int64_t b = tok / a.L, l = tok % a.L;
    const bool of_k = h >= a.q.heads;
    const Side& s = of_k ? a.k : a.q;
    const int64_t hh = of_k ? h - a.q.heads : h;
    const int64_t xi = b * s.xb + l * s.xl + hh * s.xh, yi = b * s.yb + l * s.yl + hh * s.yh;
    if (u >= half) {
      int64_t c = u - half;
      if (c >= a.start) c += a.rot;
      store_elem<DT>(s.y, yi + c, load_elem(s.x, DT, xi + c));
      continue;
    }
    const int64_t p = a.positions ? a.positions[b * a.pb + l * a.pl] : l;
    float c = 1.0f, d = 0.0f;
    if (p >= a.P) {
      c = d = __builtin_nanf("");
    } else if (p >= 0) {
      c = a.cos[p * a.ldt + u];
      d = a.sin[p * a.ldt + u];
    }
    if (a.inverse) d = -d;
    const int64_t c0 = a.start + (a.interleaved ? 2 * u : u), c1 = c0 + (a.interleaved ? 1 : half);
    const float x0 = load_elem(s.x, DT, xi + c0), x1 = load_elem(s.x, DT, xi + c1);
    store_elem<DT>(s.y, yi + c0, x0 * c - x1 * d);
    store_elem<DT>(s.y, yi + c1, x0 * d + x1 * c);
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
  const double total = (double)B * L * heads * D;
  CIN_CHECK_ARG(total < 9e15, "rotary: too many elements");
  const RotaryArgs a{{q, q_out, sqb, sql, sqh, soqb, soql, soqh, H}, {k, k_out, skb, skl, skh, sokb, sokl, sokh, Hk},
                     B, L, D, cos, sin, P, ldt, (int)rot, (int)start, positions, spb, spl, interleaved, inverse};
  const int64_t blocks = cdiv(B * L * heads * (D - rot / 2), kThreads);
  const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
  auto go = [&](auto dt) {
    hipLaunchKernelGGL(k_rotary<dt()>, grid, kThreads, 0, static_cast<hipStream_t>(stream), a);
  };
  if (dtype == CIN_DT_F32)
    go(std::integral_constant<int, CIN_DT_F32>{});
  else if (dtype == CIN_DT_F16)
    go(std::integral_constant<int, CIN_DT_F16>{});
  else
    go(std::integral_constant<int, CIN_DT_BF16>{});
  return cin_check_launch("rotary");
}

}  // extern "C"
