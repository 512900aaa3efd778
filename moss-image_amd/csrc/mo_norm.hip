// Layer and RMS norms with a weight, a bias and a modulation for each sample, for gfx950.
//
//   n = (x - m) r, r = 1 / sqrt(mean (x - m)^2 + eps), m the row's mean (RMS: 0)
//   y = n w + b,  out = y (1 + scale_s) + shift_s, s the sample that the row belongs to
//   backward, g the output's gradient: h = g (1 + scale_s) w, dx = r (h - mean h - n mean(h n)) (RMS: no mean h);
//   with P_s = sum g n and Q_s = sum g over the rows of s:  d scale_s = w P_s + b Q_s, d shift_s = Q_s,
//   d w = sum_s (1 + scale_s) P_s, d b = sum_s (1 + scale_s) Q_s
// (the reference's block: RMSNorm model.py:154-172, modulated :291-314.)
//
// All arithmetic is fp32 and each result is rounded once. The mean is taken first and the squares around it, so that
// a row far from zero loses nothing. Bound by memory: a row is read once, held in registers by up to 1024 lanes of 8
// or 16 values, and the forward pass can write it in 8 bits on the way, which the backward pass reads in place
// of it. P and Q stay in registers over a workgroup's rows; what a workgroup has of a sample is stored when its rows of
// the sample end, at slot (workgroup + sample), which no other pair has, and added up in that order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mo_block.h"
#include "mo_keep.h"

namespace {

using mo_block::NormArgs;
using namespace mo_keep;

constexpr uint32_t kNone = 0xffffffffu;  // the sample of a row that is in none

__device__ __forceinline__ uint32_t divide(uint32_t n, const mo_block::Divisor& by) {
  return (__umulhi(by.m, n) + n) >> by.s;
}

// The sample that `row` is in, and the first row from which that may not hold.
__device__ __forceinline__ uint32_t sample_of(const NormArgs& a, uint32_t row, int64_t& until) {
  until = (int64_t)1 << 62;
  if (!a.scale && !a.shift) return 0;
  if (!a.cu) {
    const uint32_t s = divide(row, a.by_share);
    until = (int64_t)(s + 1) * a.by_share.d;
    return s;
  }
  uint32_t low = 0, high = a.samples;  // the number of samples that end at or before the row
  while (low < high) {
    const uint32_t mid = (low + high) / 2;
    if (a.cu[mid + 1] <= (int64_t)row)
      low = mid + 1;
    else
      high = mid;
  }
  if (low == a.samples) return kNone;
  const int64_t first = a.cu[low];
  if (first > (int64_t)row) {
    until = first;
    return kNone;
  }
  until = a.cu[low + 1];
  return low;
}

template <int kControl>
__device__ __forceinline__ float dpp_float(float v) {
  return __builtin_bit_cast(float, dpp<kControl>(__builtin_bit_cast(uint32_t, v)));
}
__device__ __forceinline__ float sum_wave(float v) {
  v += dpp_float<0xB1>(v);   // swapped neighbours
  v += dpp_float<0x4E>(v);   // swapped pairs
  v += dpp_float<0x141>(v);  // mirrored halves of a row of 16
  v += dpp_float<0x140>(v);  // mirrored rows
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Sums over a row's lanes, the same bits in each: by wave, then across the waves through LDS. Two buffers in turn,
// so that one barrier a call is enough: who writes a buffer again has passed the barrier after its last reading.
template <int N>
__device__ __forceinline__ void sum_row(float (&v)[N], uint32_t waves, float* room, uint32_t& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sum_wave(v[i]);
  if (waves == 1) return;
  float* to = room + (turn & 1) * 32;
  ++turn;
  const uint32_t wave = threadIdx.x / 64;
  if (threadIdx.x % 64 == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i * 16 + wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float total = 0.0f;
    for (uint32_t w = 0; w < waves; ++w) total += to[i * 16 + w];
    v[i] = total;
  }
}

// Where a lane's 8 values, kIter times, lie in a row.
struct Place {
  uint32_t at, n;  // first column, how many of them are in the row
  __device__ __forceinline__ Place(const NormArgs& a, uint32_t lane, int k) {
    at = (lane + k * a.lanes) * 8;
    n = at < a.dim ? min(8u, a.dim - at) : 0;
  }
};

template <bool kOdd, int kIter>
__device__ __forceinline__ void vectors(float (&to)[kIter][8], const NormArgs& a, uint32_t lane, const void* from,
                                        uint64_t offset, uint32_t kind, float otherwise) {
#pragma unroll
  for (int k = 0; k < kIter; ++k) {
    const Place p(a, lane, k);
#pragma unroll
    for (int i = 0; i < 8; ++i) to[k][i] = otherwise;
    if (from) load8_kind<kOdd>(to[k], from, offset + (p.n ? p.at : 0), kind, p.n);
  }
}

template <class T, int kIter, bool kKeep, bool kOdd>
__device__ __forceinline__ void forward(const NormArgs& a) {
  __shared__ float room[64];
  uint32_t turn = 0;
  const uint32_t side = threadIdx.x / a.lanes, lane = threadIdx.x - side * a.lanes, waves = a.lanes / 64;
  const uint32_t first = (blockIdx.x * a.per + side) * a.chunk;
  const uint32_t end = min(a.rows, first + a.chunk);
  const float inv_dim = 1.0f / (float)a.dim;
  float weight[kIter][8], bias[kIter][8], factor[kIter][8], shift[kIter][8];
  vectors<kOdd, kIter>(weight, a, lane, a.weight, 0, a.weight_kind, 1.0f);
  vectors<kOdd, kIter>(bias, a, lane, a.bias, 0, a.weight_kind, 0.0f);
  int64_t until = 0;
  uint32_t sample = kNone;
  for (uint32_t row = first; row < end; ++row) {
    if ((int64_t)row >= until) {
      sample = sample_of(a, row, until);
      if (sample != kNone) {
        vectors<kOdd, kIter>(factor, a, lane, a.scale, sample * a.scale_stride, a.scale_kind, 0.0f);
        vectors<kOdd, kIter>(shift, a, lane, a.shift, sample * a.shift_stride, a.scale_kind, 0.0f);
      }
    }
    float x[kIter][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Place p(a, lane, k);
      widen(x[k], load8<kOdd>((const T*)a.x + row * a.x_stride + (p.n ? p.at : 0), p.n));
      if (kKeep) {
        uint32_t exponent;
        const uint2 q = encode<T>(x[k], exponent);
        if (p.at < a.groups * kGroup) {
          *(uint2*)(a.kept + (uint64_t)row * a.groups * kGroup + p.at) = q;
          if (lane % 4 == 0) a.kept_exponents[(uint64_t)row * a.groups + p.at / kGroup] = (uint8_t)exponent;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[0] += x[k][i];
    }
    float mean = 0.0f;
    if (a.layer) {
      sum_row(sum, waves, room, turn);
      mean = sum[0] * inv_dim;
    }
    sum[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Place p(a, lane, k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] = (uint32_t)i < p.n ? x[k][i] - mean : 0.0f;
        sum[0] += x[k][i] * x[k][i];
      }
    }
    sum_row(sum, waves, room, turn);
    const float r = rsqrtf(sum[0] * inv_dim + a.eps);
    if (a.stats && lane == 0) {
      a.stats[2 * (uint64_t)row] = mean;
      a.stats[2 * (uint64_t)row + 1] = r;
    }
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Place p(a, lane, k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] = x[k][i] * r * weight[k][i] + bias[k][i];
        x[k][i] = sample == kNone ? 0.0f : x[k][i] + x[k][i] * factor[k][i] + shift[k][i];
      }
      store8<kOdd>((T*)a.out + (uint64_t)row * a.dim + p.at, x[k], p.n);
    }
  }
}

template <class T, int kIter, bool kKept, bool kOdd>
__device__ __forceinline__ void backward(const NormArgs& a) {
  __shared__ float room[64];
  uint32_t turn = 0;
  const uint32_t side = threadIdx.x / a.lanes, lane = threadIdx.x - side * a.lanes, waves = a.lanes / 64;
  const uint32_t group = blockIdx.x * a.per + side, first = group * a.chunk;
  const uint32_t end = min(a.rows, first + a.chunk);
  const float inv_dim = 1.0f / (float)a.dim;
  float gain[kIter][8];  // (1 + scale) w
  float along[kIter][8], plain[kIter][8];  // P and Q
  int64_t until = 0;
  uint32_t sample = kNone;

  auto flush = [&]() {
    if (sample == kNone || !a.partial) return;
    float* to = a.partial + (uint64_t)(group + sample) * 2 * a.pitch;
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const uint32_t at = (lane + k * a.lanes) * 8;
      if (at < a.pitch) {
        store8(to + at, along[k]);
        store8(to + a.pitch + at, plain[k]);
      }
    }
  };

  for (uint32_t row = first; row < end; ++row) {
    if ((int64_t)row >= until) {
      flush();
      sample = sample_of(a, row, until);
      float weight[kIter][8];
      vectors<kOdd, kIter>(weight, a, lane, a.weight, 0, a.weight_kind, 1.0f);
      vectors<kOdd, kIter>(gain, a, lane, sample == kNone ? nullptr : a.scale, sample * a.scale_stride, a.scale_kind, 0.0f);
#pragma unroll
      for (int k = 0; k < kIter; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          gain[k][i] = sample == kNone ? 0.0f : weight[k][i] + weight[k][i] * gain[k][i];
          along[k][i] = plain[k][i] = 0.0f;
        }
    }
    const float mean = a.stats[2 * (uint64_t)row], r = a.stats[2 * (uint64_t)row + 1];
    float n[kIter][8], h[kIter][8];
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Place p(a, lane, k);
      float g[8];
      if (kKept) {
        uint2 q = {0, 0};
        uint32_t exponent = 0;
        if (p.n) {
          q = *(const uint2*)((const int8_t*)a.x + (uint64_t)row * a.groups * kGroup + p.at);
          exponent = a.x_exponents[(uint64_t)row * a.groups + p.at / kGroup];
        }
        decode(n[k], q, exponent);
      } else {
        widen(n[k], load8<kOdd>((const T*)a.x + row * a.x_stride + (p.n ? p.at : 0), p.n));
      }
      widen(g, load8<kOdd>((const T*)a.grad + row * a.grad_stride + (p.n ? p.at : 0), p.n));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[k][i] = (uint32_t)i < p.n ? (n[k][i] - mean) * r : 0.0f;
        h[k][i] = g[i] * gain[k][i];
        along[k][i] += g[i] * n[k][i];
        plain[k][i] += g[i];
        sums[0] += h[k][i] * n[k][i];
        sums[1] += h[k][i];
      }
    }
    sum_row(sums, waves, room, turn);
    const float mean_along = sums[0] * inv_dim, mean_plain = a.layer ? sums[1] * inv_dim : 0.0f;
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
      const Place p(a, lane, k);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[k][i] = sample == kNone ? 0.0f : r * (h[k][i] - mean_plain - n[k][i] * mean_along);
      store8<kOdd>((T*)a.out + (uint64_t)row * a.dim + p.at, h[k], p.n);
    }
  }
  flush();
}

// Names: type, times a lane holds 8 values; "odd": a dim that is no multiple of eight.
#define MO_NORM(T, t, k, odd, name)                                                                          \
  extern "C" __global__ __launch_bounds__(1024) void mo_norm_forward_##t##_##name(NormArgs a) {              \
    forward<T, k, false, odd>(a);                                                                            \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(1024) void mo_norm_forward_keep_##t##_##name(NormArgs a) {         \
    forward<T, k, true, odd>(a);                                                                             \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(1024) void mo_norm_backward_##t##_##name(NormArgs a) {             \
    backward<T, k, false, odd>(a);                                                                           \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(1024) void mo_norm_backward_kept_##t##_##name(NormArgs a) {        \
    backward<T, k, true, odd>(a);                                                                            \
  }
#define MO_NORMS(T, t)           \
  MO_NORM(T, t, 1, false, 1)     \
  MO_NORM(T, t, 2, false, 2)     \
  MO_NORM(T, t, 1, true, 1_odd)  \
  MO_NORM(T, t, 2, true, 2_odd)
MO_NORMS(_Float16, f16)
MO_NORMS(__bf16, bf16)
MO_NORMS(float, f32)

__device__ __forceinline__ float value_kind(const void* base, uint64_t at, uint32_t kind) {
  return kind == 2 ? ((const float*)base)[at] : kind == 1 ? (float)((const __bf16*)base)[at]
                                                          : (float)((const _Float16*)base)[at];
}

// A sample's sums over its workgroups for 32 columns: 32 runs of them side by side, then the runs, both in order.
extern "C" __global__ __launch_bounds__(1024) void mo_norm_sums(NormArgs a) {
  __shared__ float room[2][32][33];
  const uint32_t column = threadIdx.x % 32, run = threadIdx.x / 32, sample = blockIdx.y;
  const uint32_t at = blockIdx.x * 32 + column;
  int64_t low = 0, high = a.rows;
  if (a.scale || a.shift) {
    low = a.cu ? a.cu[sample] : (int64_t)sample * a.by_share.d;
    high = a.cu ? a.cu[sample + 1] : low + a.by_share.d;
    low = low < 0 ? 0 : low;
    high = high > (int64_t)a.rows ? (int64_t)a.rows : high;
  }
  float along = 0.0f, plain = 0.0f;
  if (at < a.dim && low < high) {
    const uint32_t from = (uint32_t)low / a.chunk, to = (uint32_t)(high - 1) / a.chunk;
    for (uint32_t i = from + run; i <= to; i += 32) {
      const float* p = a.partial + (uint64_t)(i + sample) * 2 * a.pitch + at;
      along += p[0];
      plain += p[a.pitch];
    }
  }
  room[0][run][column] = along;
  room[1][run][column] = plain;
  __syncthreads();
  if (run || at >= a.dim) return;
  for (int i = 1; i < 32; ++i) {
    along += room[0][i][column];
    plain += room[1][i][column];
  }
  const uint64_t here = (uint64_t)sample * a.dim + at;
  if (a.scale_grad) {
    const float w = a.weight ? value_kind(a.weight, at, a.weight_kind) : 1.0f;
    const float b = a.bias ? value_kind(a.bias, at, a.weight_kind) : 0.0f;
    store_kind(a.scale_grad, here, a.scale_kind, w * along + b * plain);
  }
  if (a.shift_grad) store_kind(a.shift_grad, here, a.scale_kind, plain);
  const float factor = a.scale ? 1.0f + value_kind(a.scale, sample * a.scale_stride + at, a.scale_kind) : 1.0f;
  along *= factor;
  plain *= factor;
  if (a.sample_sums) {
    a.sample_sums[(uint64_t)sample * 2 * a.pitch + at] = along;
    a.sample_sums[(uint64_t)sample * 2 * a.pitch + a.pitch + at] = plain;
  } else {
    if (a.weight_grad) store_kind(a.weight_grad, at, a.weight_kind, along);
    if (a.bias_grad) store_kind(a.bias_grad, at, a.weight_kind, plain);
  }
}

// The weight's and the bias's gradients from the samples' sums, in order.
extern "C" __global__ __launch_bounds__(256) void mo_norm_sample_sums(NormArgs a) {
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  if (at >= a.dim) return;
  float along = 0.0f, plain = 0.0f;
  for (uint32_t s = 0; s < a.samples; ++s) {
    along += a.sample_sums[(uint64_t)s * 2 * a.pitch + at];
    plain += a.sample_sums[(uint64_t)s * 2 * a.pitch + a.pitch + at];
  }
  if (a.weight_grad) store_kind(a.weight_grad, at, a.weight_kind, along);
  if (a.bias_grad) store_kind(a.bias_grad, at, a.weight_kind, plain);
}

}  // namespace
