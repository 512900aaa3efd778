// Rotary positions of attention heads, with the heads' RMS norm where a block has one, for gfx950.
//
//   n = x rsqrt(mean x^2 + eps), y = n w          (no norm: y = x)
//   out(f, s) = (y_f cos - y_s sin, y_s cos + y_f sin) for each pair (f, s) of the first rotary_dim
//               values of a head: (i, i + rotary_dim / 2), or neighbours (2i, 2i + 1) where interleaved;
//               the values after them are passed on
//   backward     g = the same turn by the opposite angle of the output's gradient; d weight = sum g n;
//               d x = r (g w - n mean(g w n)), r the factor of the norm
// (the reference's block: RMSNorm model.py:154-172, rotate_rope :41-56, applied :59-91; its angles :136-151)
//
// All arithmetic is fp32 and each result is rounded once, where the composed form rounds to the tokens'
// type after every step. Bound by memory: one read and one write of the heads a direction (two reads and
// one write backward with a norm), and the table from cache for all but one head of a token. So each lane
// moves 16 bytes at a time: a head's row is shared out over the lanes of a part of a wave, kVec pairs a
// lane, and the row's sums are taken by lane exchanges. 4608 tokens, 24 heads of 128, bf16, both sides with norms: forward
// 30 to 31 us (3.7 TB/s), backward 51 to 53 (3.2) and 4 for the weights' sums. Four heads a lane, which reads the angles once:
// 44 and 77.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mo_rotary.h"

namespace {

using mo_rotary::Args;
using mo_rotary::Side;

constexpr uint32_t kBF16 = 1, kF32 = 2;  // MO_DTYPE_*

// n consecutive values to or from memory; the host has checked the alignment of n elements.
template <class T, int n>
struct alignas(sizeof(T) * n > 16 ? 16 : sizeof(T) * n) Pack {
  T v[n];
};
template <class T, int n>
__device__ __forceinline__ void load(float (&to)[n], const T* p) {
  const Pack<T, n> a = *(const Pack<T, n>*)p;
#pragma unroll
  for (int i = 0; i < n; ++i) to[i] = (float)a.v[i];
}
template <class T, int n>
__device__ __forceinline__ void store(T* p, const float (&from)[n]) {
  Pack<T, n> a;
#pragma unroll
  for (int i = 0; i < n; ++i) a.v[i] = (T)from[i];
  *(Pack<T, n>*)p = a;
}
template <int n>
__device__ __forceinline__ void load_kind(float (&to)[n], const void* base, uint64_t at, uint32_t kind) {
  if (kind == kF32)
    load<float, n>(to, (const float*)base + at);
  else if (kind == kBF16)
    load<__bf16, n>(to, (const __bf16*)base + at);
  else
    load<_Float16, n>(to, (const _Float16*)base + at);
}

// A lane's kVec pairs of a head: where the first and the second of each lie.
template <int kVec>
struct Pairs {
  uint32_t pair;     // first pair
  bool on, turned;   // in the head; within the rotary part
  bool apart;        // first at `pair`, second at pair + rotary_dim / 2; else neighbours from 2 * pair
  uint32_t half;
  __device__ __forceinline__ Pairs(const Args& a, uint32_t p) : pair(p) {
    half = a.rotary_dim / 2;
    on = 2 * pair < a.head_dim;
    turned = pair < half;
    apart = turned && !a.interleaved;
  }
  template <class Load>
  __device__ __forceinline__ void get(float (&f)[kVec], float (&s)[kVec], Load&& at) const {
    if (apart) {
      at(f, pair);
      at(s, pair + half);
    } else {
      float lo[kVec], hi[kVec];
      at(lo, 2 * pair);
      at(hi, 2 * pair + kVec);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        f[i] = 2 * i < kVec ? lo[2 * i % kVec] : hi[2 * i % kVec];
        s[i] = 2 * i + 1 < kVec ? lo[(2 * i + 1) % kVec] : hi[(2 * i + 1) % kVec];
      }
    }
  }
  template <class Store>
  __device__ __forceinline__ void put(const float (&f)[kVec], const float (&s)[kVec], Store&& at) const {
    if (apart) {
      at(f, pair);
      at(s, pair + half);
    } else {
      float lo[kVec], hi[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (2 * i < kVec) lo[2 * i % kVec] = f[i]; else hi[2 * i % kVec] = f[i];
        if (2 * i + 1 < kVec) lo[(2 * i + 1) % kVec] = s[i]; else hi[(2 * i + 1) % kVec] = s[i];
      }
      at(lo, 2 * pair);
      at(hi, 2 * pair + kVec);
    }
  }
};

// Sum over `lanes` neighbouring lanes (a power of two, 1 to 64), the same bits in each: within a row of 16 by
// DPP (swapped neighbours, swapped pairs, mirrored halves, mirrored row), past it through the exchange unit.
template <int kControl>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kControl, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum_lanes(float v, uint32_t lanes) {
  if (lanes > 1) v += dpp<0xB1>(v);
  if (lanes > 2) v += dpp<0x4E>(v);
  if (lanes > 4) v += dpp<0x141>(v);
  if (lanes > 8) v += dpp<0x140>(v);
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}

__device__ __forceinline__ uint32_t divide(uint32_t n, const mo_rotary::Divisor& by) {
  return (__umulhi(by.m, n) + n) >> by.s;
}

// Lanes of a head (a power of two) and the pairs a lane holds: kVec at a time, kIter times.
template <int kVec>
struct Shape {
  static constexpr int kIter = kVec >= 4 ? 1 : kVec == 2 ? 2 : 4;
};

template <class T, int kVec, bool kBackward>
__device__ __forceinline__ void rotary(const Args& a, uint32_t lanes) {
  constexpr int kIter = Shape<kVec>::kIter;
  const Side& side = a.side[blockIdx.y];
  if (blockIdx.x >= side.blocks) return;
  const uint32_t rows = a.batch * a.tokens * side.heads;  // below 2^31
  const uint32_t per = 256 / lanes, in_row = threadIdx.x % lanes;
  const bool norm = side.weight != nullptr;
  const float inv_dim = 1.0f / (float)a.head_dim;

  float wf[kIter][kVec], ws[kIter][kVec], sum_f[kIter][kVec], sum_s[kIter][kVec];
#pragma unroll
  for (int k = 0; k < kIter; ++k) {
    const Pairs<kVec> at(a, (in_row + k * lanes) * kVec);
#pragma unroll
    for (int i = 0; i < kVec; ++i) wf[k][i] = ws[k][i] = 1.0f, sum_f[k][i] = sum_s[k][i] = 0.0f;
    if (norm && at.on)
      at.get(wf[k], ws[k], [&](float (&to)[kVec], uint32_t e) { load_kind<kVec>(to, side.weight, e, a.weight_kind); });
  }

  // every lane of a wave takes the same number of turns, so that the exchanges find all of them
  const uint32_t step = side.blocks * per;
  for (uint32_t first = blockIdx.x * per; first < rows; first += step) {
    const uint32_t row = first + threadIdx.x / lanes;
    const bool live = row < rows;
    const uint32_t token = live ? divide(row, side.by_heads) : 0, head = live ? row - token * side.heads : 0;
    const uint32_t b = divide(token, a.by_tokens), t = token - b * a.tokens;
    const T* x = (const T*)side.x + (int64_t)b * side.x_batch + (int64_t)t * side.x_token + (int64_t)head * side.x_head;
    const T* g = (const T*)side.grad + (int64_t)b * side.g_batch + (int64_t)t * side.g_token +
                 (int64_t)head * side.g_head;
    T* out = (T*)side.out + (uint64_t)row * a.head_dim;
    const uint64_t angle = b * a.table_batch + (uint64_t)t * a.rotary_dim;

    float xf[kIter][kVec], xs[kIter][kVec], gf[kIter][kVec], gs[kIter][kVec];
    float squares = 0.0f, along = 0.0f;
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Pairs<kVec> at(a, (in_row + k * lanes) * kVec);
      const bool on = live && at.on;
#pragma unroll
      for (int i = 0; i < kVec; ++i) xf[k][i] = xs[k][i] = gf[k][i] = gs[k][i] = 0.0f;
      if (on && (!kBackward || norm)) at.get(xf[k], xs[k], [&](float (&to)[kVec], uint32_t e) { load<T, kVec>(to, x + e); });
      if (on && kBackward) at.get(gf[k], gs[k], [&](float (&to)[kVec], uint32_t e) { load<T, kVec>(to, g + e); });
#pragma unroll
      for (int i = 0; i < kVec; ++i) squares += xf[k][i] * xf[k][i] + xs[k][i] * xs[k][i];
    }
    float r = 1.0f;
    if (norm) r = rsqrtf(sum_lanes(squares, lanes) * inv_dim + a.eps);
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Pairs<kVec> at(a, (in_row + k * lanes) * kVec);
      float sin[kVec], cos[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) sin[i] = 0.0f, cos[i] = 1.0f;
      if (live && at.turned) {
        load_kind<kVec>(sin, a.table, angle + at.pair, a.table_kind);
        load_kind<kVec>(cos, a.table, angle + at.half + at.pair, a.table_kind);
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (!kBackward) {
          const float f = norm ? xf[k][i] * r * wf[k][i] : xf[k][i], s = norm ? xs[k][i] * r * ws[k][i] : xs[k][i];
          xf[k][i] = at.turned ? f * cos[i] - s * sin[i] : f;
          xs[k][i] = at.turned ? s * cos[i] + f * sin[i] : s;
        } else {
          const float f = at.turned ? gf[k][i] * cos[i] + gs[k][i] * sin[i] : gf[k][i];
          const float s = at.turned ? gs[k][i] * cos[i] - gf[k][i] * sin[i] : gs[k][i];
          xf[k][i] *= r;
          xs[k][i] *= r;
          if (norm) {
            sum_f[k][i] += f * xf[k][i];
            sum_s[k][i] += s * xs[k][i];
          }
          gf[k][i] = f * wf[k][i];
          gs[k][i] = s * ws[k][i];
          along += gf[k][i] * xf[k][i] + gs[k][i] * xs[k][i];
        }
      }
    }
    if (kBackward && norm) {
      const float mean = sum_lanes(along, lanes) * inv_dim;
#pragma unroll
      for (int k = 0; k < kIter; ++k)
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          gf[k][i] = r * (gf[k][i] - xf[k][i] * mean);
          gs[k][i] = r * (gs[k][i] - xs[k][i] * mean);
        }
    }
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Pairs<kVec> at(a, (in_row + k * lanes) * kVec);
      if (!live || !at.on) continue;
      auto to = [&](const float (&v)[kVec], uint32_t e) { store<T, kVec>(out + e, v); };
      if (kBackward)
        at.put(gf[k], gs[k], to);
      else
        at.put(xf[k], xs[k], to);
    }
  }

  if (kBackward && norm) {
    // the workgroup's sum for each value of the head, rows in a fixed order
    __shared__ float sums[256 * 2 * kVec];
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        sums[threadIdx.x * 2 * kVec + 2 * i] = sum_f[k][i];
        sums[threadIdx.x * 2 * kVec + 2 * i + 1] = sum_s[k][i];
      }
      __syncthreads();
      for (uint32_t v = threadIdx.x; v < lanes * 2 * kVec; v += 256) {
        float total = 0.0f;
        for (uint32_t i = 0; i < per; ++i) total += sums[i * lanes * 2 * kVec + v];
        const uint32_t pair = (v / (2 * kVec) + k * lanes) * kVec + v % (2 * kVec) / 2;
        const Pairs<kVec> at(a, pair);
        const uint32_t e = at.apart ? pair + (v & 1) * at.half : 2 * pair + (v & 1);
        if (at.on) side.partial[(uint64_t)blockIdx.x * a.head_dim + e] = total;
      }
    }
  }
}

#define MO_ROTARY(T, t, n)                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void mo_rotary_forward_##t##_##n(Args a, uint32_t lanes) {    \
    rotary<T, n, false>(a, lanes);                                                                           \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void mo_rotary_backward_##t##_##n(Args a, uint32_t lanes) {   \
    rotary<T, n, true>(a, lanes);                                                                            \
  }
MO_ROTARY(_Float16, f16, 1)
MO_ROTARY(_Float16, f16, 2)
MO_ROTARY(_Float16, f16, 4)
MO_ROTARY(_Float16, f16, 8)
MO_ROTARY(__bf16, bf16, 1)
MO_ROTARY(__bf16, bf16, 2)
MO_ROTARY(__bf16, bf16, 4)
MO_ROTARY(__bf16, bf16, 8)
MO_ROTARY(float, f32, 1)
MO_ROTARY(float, f32, 2)
MO_ROTARY(float, f32, 4)

// The norm weights' gradients: the workgroups' sums of 16 values a workgroup, in a fixed order, 64 runs of
// them side by side and then the runs.
extern "C" __global__ __launch_bounds__(1024) void mo_rotary_weight_sum(Args a) {
  __shared__ float sums[64][17];
  const Side& side = a.side[blockIdx.y];
  if (!side.weight_grad) return;
  const uint32_t e = blockIdx.x * 16 + threadIdx.x % 16, part = threadIdx.x / 16;
  float total = 0.0f;
  if (e < a.head_dim) {
#pragma unroll 8
    for (uint32_t i = part; i < side.blocks; i += 64) total += side.partial[(uint64_t)i * a.head_dim + e];
  }
  sums[part][threadIdx.x % 16] = total;
  __syncthreads();
  if (part || e >= a.head_dim) return;
  for (int i = 1; i < 64; ++i) total += sums[i][threadIdx.x];
  if (a.weight_kind == kF32)
    ((float*)side.weight_grad)[e] = total;
  else if (a.weight_kind == kBF16)
    ((__bf16*)side.weight_grad)[e] = (__bf16)total;
  else
    ((_Float16*)side.weight_grad)[e] = (_Float16)total;
}

// Sines and cosines of coordinate x band, the product rounded to fp32 as the composed form rounds it, times
// the amplitude: out[t] = axes * bands sines, then as many cosines. One lane an angle;
// 4.0 us for 4608 rows of 64 angles, 2.0 for a few: a launch.
extern "C" __global__ __launch_bounds__(256) void mo_rotary_table_kernel(const float* __restrict__ coordinates,
                                                                         const float* __restrict__ bands,
                                                                         void* __restrict__ out, uint64_t rows,
                                                                         uint32_t axes, uint32_t n_bands,
                                                                         float amplitude, uint32_t kind) {
  const uint32_t angles = axes * n_bands;
  const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t row = at / angles;
  if (row >= rows) return;
  const uint32_t i = (uint32_t)(at % angles);
  const float phase = __fmul_rn(coordinates[row * axes + i / n_bands], bands[i % n_bands]);
  float s, c;
  sincosf(phase, &s, &c);
  s *= amplitude, c *= amplitude;
  const uint64_t to = row * 2 * angles + i;
  if (kind == kF32)
    ((float*)out)[to] = s, ((float*)out)[to + angles] = c;
  else if (kind == kBF16)
    ((__bf16*)out)[to] = (__bf16)s, ((__bf16*)out)[to + angles] = (__bf16)c;
  else
    ((_Float16*)out)[to] = (_Float16)s, ((_Float16*)out)[to + angles] = (_Float16)c;
}

}  // namespace
