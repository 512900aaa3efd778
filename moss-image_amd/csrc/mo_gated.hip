// The gated activation between the two products of a feed-forward, and activations in 8 bits, for gfx950.
//
//   out = act(g) cap(u):  SiTU  act = 4 tanh(g / 4) s, cap = 25 tanh(u / 25), s = 1 / (1 + exp(-g))
//                         SiLU  act = g s, cap = u
//   backward, d the output's gradient:  d u = d act cap', d g = d cap act'
//                         SiTU  act' = (1 - t^2) s + 4 t s (1 - s), t = tanh(g / 4); cap' = 1 - tanh(u / 25)^2
//                         SiLU  act' = s (1 + g (1 - s)), cap' = 1
// (the reference's SiTU-GLU: model.py:27-38.)
//
// fp32 inside, each result rounded once. A gate takes one exponential, e = exp(-|g| / 2): s is 1 / (1 + e^2) or
// e^2 / (1 + e^2), 1 - s the other, tanh |g / 4| is (1 - e) / (1 + e) and 1 - t^2 is 4 e / (1 + e)^2: as differences from 1
// the last two would be nothing but rounding for a gate that is far from zero. Near zero that difference cancels, and the odd series takes over:
// x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835, below 1/4, where the rest is under 2^-26 of x. tanh(u / 25) is
// nearly always there, so its exponential is behind a branch. With the library's tanhf and expf the forward pass was
// bound by arithmetic.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mo_block.h"
#include "mo_keep.h"

namespace {

using mo_block::GatedArgs;
using mo_block::KeepArgs;
using namespace mo_keep;

__device__ __forceinline__ uint32_t divide(uint32_t n, const mo_block::Divisor& by) {
  return (__umulhi(by.m, n) + n) >> by.s;
}

// exp(-x c) for 0 <= x: 2^(-x c log2 e), the product's rounding put right, which would be x c units of the result.
// `high` and `low` are c log2 e in two parts. Past 4096 x is as good as infinite.
__device__ __forceinline__ float decay(float x, float high, float low) {
  x = x > 4096.0f ? 4096.0f : x;  // keeps a NaN
  const float power = -x * high;
  const float rest = fmaf(-x, high, -power) - x * low;
  const float e = __builtin_amdgcn_exp2f(power);
  return fmaf(e, rest * 0.69314718f, e);
}
constexpr float kSeries = 0.25f;
__device__ __forceinline__ float tanh_series(float x) {
  const float y = x * x;
  return fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), x);
}
// s = sigmoid g, t = tanh(g / 4), rest = 1 - s and bend = 1 - t^2. log2 e / 2 = 0.72134752 + 1.4e-8 - ...
struct Gate {
  float s, t, rest, bend;
};
__device__ __forceinline__ Gate gate_of(float g) {
  const float e = decay(fabsf(g), 0x1.715476p-1f, 0x1.4ae0cp-27f), e2 = e * e;
  const float one = 1.0f + e, two = 1.0f + e2, r = __builtin_amdgcn_rcpf(one * two);
  const float near = one * r, far = e2 * near, q = two * r;
  Gate to;
  to.s = g >= 0.0f ? near : far;
  to.s = g != g ? g : to.s;
  to.rest = g >= 0.0f ? far : near;
  to.bend = 4.0f * e * (q * q);
  const float x = 0.25f * g;
  to.t = fabsf(x) < kSeries ? tanh_series(x) : copysignf((1.0f - e) * q, g);
  return to;
}
__device__ __forceinline__ float sigmoid_of(float g) {
  const float e = decay(fabsf(g), 0x1.715476p+0f, 0x1.4ae0cp-26f);
  const float s = (g >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e);
  return g != g ? g : s;
}
struct Cap {
  float c, bend;  // tanh(u / 25), 1 - its square
};
__device__ __forceinline__ Cap cap_of(float u) {
  const float x = u * 0.04f;
  Cap to;
  to.c = tanh_series(x);
  to.bend = 1.0f - to.c * to.c;
  if (!(fabsf(x) < kSeries)) {
    const float e = decay(fabsf(u), 0x1.d8be08p-4f, 0x1.7f5ffep-32f);  // exp(-2 |u| / 25)
    const float q = __builtin_amdgcn_rcpf(1.0f + e);
    to.c = copysignf((1.0f - e) * q, u);
    to.bend = 4.0f * e * (q * q);
  }
  return to;
}

// A lane's place: row, first column, how many of its 8 are in the row, its group and whether it has a row at all.
struct Spot {
  uint32_t row, at, n;
  bool live;
  __device__ __forceinline__ Spot(uint32_t rows, uint32_t cols, uint32_t lanes, const mo_block::Divisor& by) {
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    row = divide(item, by);
    at = (item - row * lanes) * 8;
    live = row < rows;
    n = live && at < cols ? min(8u, cols - at) : 0;
  }
};

template <bool kOdd, class T>
__device__ __forceinline__ void load_row(float (&to)[8], const void* base, uint64_t stride, const Spot& s) {
  widen(to, load8<kOdd>((const T*)base + (s.n ? s.row * stride + s.at : 0), s.n));
}
template <class T>
__device__ __forceinline__ void write_kept(const float (&v)[8], int8_t* values, uint8_t* exponents, uint64_t stride,
                                           uint64_t exponents_stride, const Spot& s) {
  uint32_t exponent;
  const uint2 q = encode<T>(v, exponent);
  if (!s.live) return;
  *(uint2*)(values + s.row * stride + s.at) = q;
  if (s.at % kGroup == 0) exponents[s.row * exponents_stride + s.at / kGroup] = (uint8_t)exponent;
}
__device__ __forceinline__ void read_kept(float (&to)[8], const void* values, const uint8_t* exponents, uint64_t stride,
                                          uint64_t exponents_stride, const Spot& s) {
  uint2 q = {0, 0};
  uint32_t exponent = 0;
  if (s.live) {
    q = *(const uint2*)((const int8_t*)values + s.row * stride + s.at);
    exponent = exponents[s.row * exponents_stride + s.at / kGroup];
  }
  decode(to, q, exponent);
}

// A lane has eight neighbouring columns, so that a wave reads 1 KB of a row side by side; one pass, nothing held. SiLU is bound by
// memory, SiTU by its arithmetic too: bfloat16, 4608 x 8192 (226 MB) 41 us, 5.5 TB/s, and 46 to 49. SiTU of 17792 x 12288 (1.31 GB), in
// which a SIMD issues 189 000 vector instructions, takes 245 us at the full clock, 5.4 TB/s, and 285 where power holds it at 2 GHz;
// 4608 x 8192, both inputs written in 8 bits (304 MB) 65, 4.7 TB/s.
template <class T, bool kKeep, bool kOdd>
__device__ __forceinline__ void forward(const GatedArgs& a) {
  const Spot s(a.rows, a.cols, a.lanes, a.by_lanes);
  float u[8], g[8];
  load_row<kOdd, T>(u, a.up, a.up_stride, s);
  load_row<kOdd, T>(g, a.gate, a.gate_stride, s);
  if (kKeep) {
    write_kept<T>(u, a.kept_up, a.kept_up_exponents, a.values_stride, a.exponents_stride, s);
    write_kept<T>(g, a.kept_gate, a.kept_gate_exponents, a.values_stride, a.exponents_stride, s);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (a.silu) {
      u[i] = u[i] * (g[i] * sigmoid_of(g[i]));
    } else {
      const Gate gate = gate_of(g[i]);
      u[i] = 100.0f * (gate.t * gate.s) * cap_of(u[i]).c;
    }
  }
  store8<kOdd>((T*)a.out + s.row * a.out_stride + s.at, u, s.n);
}

// Bound by memory: 17792 x 12288 (2.19 GB) in 370 us at either clock, 5.9 TB/s; 4608 x 8192 (377 MB) 63 us, SiLU 61, 6 TB/s; from 8 bits
// (304 MB) 63, 4.8 TB/s.
template <class T, bool kKept, bool kOdd>
__device__ __forceinline__ void backward(const GatedArgs& a) {
  const Spot s(a.rows, a.cols, a.lanes, a.by_lanes);
  float u[8], g[8], d[8];
  if (kKept) {
    read_kept(u, a.up, a.up_exponents, a.values_stride, a.exponents_stride, s);
    read_kept(g, a.gate, a.gate_exponents, a.values_stride, a.exponents_stride, s);
  } else {
    load_row<kOdd, T>(u, a.up, a.up_stride, s);
    load_row<kOdd, T>(g, a.gate, a.gate_stride, s);
  }
  load_row<kOdd, T>(d, a.grad, a.grad_stride, s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float act, slope, cap, cap_slope;
    if (a.silu) {
      const float gate = sigmoid_of(g[i]);
      act = g[i] * gate, slope = gate * (1.0f + g[i] * (1.0f - gate)), cap = u[i], cap_slope = 1.0f;
    } else {
      const Gate gate = gate_of(g[i]);
      const Cap to = cap_of(u[i]);
      act = 4.0f * gate.t * gate.s, slope = gate.bend * gate.s + act * gate.rest, cap = 25.0f * to.c, cap_slope = to.bend;
    }
    u[i] = d[i] * act * cap_slope;
    g[i] = d[i] * cap * slope;
  }
  store8<kOdd>((T*)a.out + s.row * a.out_stride + s.at, u, s.n);
  store8<kOdd>((T*)a.out_gate + s.row * a.out_stride + s.at, g, s.n);
}

// To 8 bits and back, bound by memory: 17792 x 3072 bfloat16 (166 MB each way) in 29.1 and 24.8 us, 5.7 and 6.7 TB/s.
template <class T, bool kOdd>
__device__ __forceinline__ void pack(const KeepArgs& a) {
  const Spot s(a.rows, a.cols, a.lanes, a.by_lanes);
  float v[8];
  load_row<kOdd, T>(v, a.x, a.stride, s);
  write_kept<T>(v, a.values, a.exponents, (uint64_t)a.groups * kGroup, a.groups, s);
}
template <class T, bool kOdd>
__device__ __forceinline__ void restore(const KeepArgs& a) {
  const Spot s(a.rows, a.cols, a.lanes, a.by_lanes);
  float v[8];
  read_kept(v, a.values, a.exponents, (uint64_t)a.groups * kGroup, a.groups, s);
  store8<kOdd>((T*)a.out + s.row * a.stride + s.at, v, s.n);
}

// "odd": columns that are no multiple of eight (4608 x 8191 55 and 90 us both ways, 8192 47 and 63).
#define MO_GATED(T, t, odd)                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void mo_gated_forward_##t(GatedArgs a) { forward<T, false, odd>(a); }      \
  extern "C" __global__ __launch_bounds__(256) void mo_gated_forward_keep_##t(GatedArgs a) { forward<T, true, odd>(a); }  \
  extern "C" __global__ __launch_bounds__(256) void mo_gated_backward_##t(GatedArgs a) { backward<T, false, odd>(a); }    \
  extern "C" __global__ __launch_bounds__(256) void mo_gated_backward_kept_##t(GatedArgs a) { backward<T, true, odd>(a); } \
  extern "C" __global__ __launch_bounds__(256) void mo_keep_pack_##t(KeepArgs a) { pack<T, odd>(a); }                     \
  extern "C" __global__ __launch_bounds__(256) void mo_keep_restore_##t(KeepArgs a) { restore<T, odd>(a); }
MO_GATED(_Float16, f16, false)
MO_GATED(__bf16, bf16, false)
MO_GATED(float, f32, false)
MO_GATED(_Float16, f16_odd, true)
MO_GATED(__bf16, bf16_odd, true)
MO_GATED(float, f32_odd, true)

}  // namespace
