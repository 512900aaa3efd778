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
// a row far from zero loses no more than the mean's own rounding. Bound by memory: a row is read once, held in registers by up to 512 lanes of 8
// to 32 values, and the forward pass can write it in 8 bits on the way, which the backward pass reads in place
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
  float* to = room + (turn & 1) * N * 16;
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

// Rows one after the other that a batch takes: their sums cross the waves together, and a batch's rows are read while
// the one before is worked on. (Two batches ahead take registers for which a workgroup less fits on a CU: a backward pass
// through 8 bits took 107 us where this takes 71.)
template <int kIter>
constexpr int kBatch = kIter == 1 ? 2 : 1;

// A workgroup's (or, side by side, a wave's) rows, batch by batch; a batch ends where a sample does.
struct Walk {
  uint32_t row, end, sample, count;  // the batch: first row, the sample, rows
  int64_t until;
  __device__ __forceinline__ Walk(const NormArgs& a, uint32_t first, uint32_t most) : row(first), end(min(a.rows, first + a.chunk)) {
    find(a, most);
  }
  __device__ __forceinline__ void find(const NormArgs& a, uint32_t most) {
    if (row >= end) {
      sample = kNone, count = 0;
      return;
    }
    sample = __builtin_amdgcn_readfirstlane(sample_of(a, row, until));
    take(most);
  }
  __device__ __forceinline__ void take(uint32_t most) {
    count = min(most, end - row);
    if (until < (int64_t)row + count) count = (uint32_t)(until - row);
  }
  __device__ __forceinline__ void next(const NormArgs& a, uint32_t most) {
    row += count;
    if ((int64_t)row >= until || row >= end)
      find(a, most);
    else
      take(most);
  }
};

// Bound by memory: bfloat16, 4608 rows of 3072 (57 MB) in 13.4 us, 4.2 TB/s; 17792 rows that are written in 8 bits too (275 MB)
// in 56, 4.9 TB/s (a large copy: 5.1).
template <class T, int kIter, bool kKeep, bool kOdd>
__device__ __forceinline__ void forward(const NormArgs& a) {
  constexpr int kRows = kBatch<kIter>;
  __shared__ float room[2 * kRows * 16];
  uint32_t turn = 0;
  const uint32_t side = a.per > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
  const uint32_t lane = threadIdx.x - side * a.lanes, waves = a.lanes / 64;
  const float inv_dim = 1.0f / (float)a.dim;
  Walk now(a, (blockIdx.x * a.per + side) * a.chunk, kRows);
  if (now.row >= now.end) return;
  struct Raw {
    Eight<T> x[kRows][kIter];
  };
  // rows that are none are read from and written to windows of no length: branches around memory instructions would
  // have every wait be for all of them
  auto read = [&](Raw& raw, const Walk& w) {
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
      const bool live = i < w.count;
      const uint32_t row = live ? w.row + i : 0;
      const Window<T, kOdd> x((const T*)a.x + row * a.x_stride, live ? a.dim : 0);
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        const Place p(a, lane, k);
        raw.x[i][k] = x.read(0, p.at, live ? p.n : 0);
      }
    }
  };
  Raw raw;
  read(raw, now);
  float gain[kIter][8], level[kIter][8];  // w (1 + scale), b (1 + scale) + shift
  bool fresh = true;
  while (true) {
    if (fresh) {
      const bool none = now.sample == kNone;
      float factor[kIter][8], shift[kIter][8];
      vectors<kOdd, kIter>(gain, a, lane, a.weight, 0, a.weight_kind, 1.0f);
      vectors<kOdd, kIter>(level, a, lane, a.bias, 0, a.weight_kind, 0.0f);
      vectors<kOdd, kIter>(factor, a, lane, none ? nullptr : a.scale, now.sample * a.scale_stride, a.scale_kind, 0.0f);
      vectors<kOdd, kIter>(shift, a, lane, none ? nullptr : a.shift, now.sample * a.shift_stride, a.scale_kind, 0.0f);
#pragma unroll
      for (int k = 0; k < kIter; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gain[k][e] += gain[k][e] * factor[k][e];
          level[k][e] += level[k][e] * factor[k][e] + shift[k][e];
        }
    }
    float x[kRows][kIter][8], sum[kRows], mean[kRows];
    uint2 kept[kRows][kIter];
    uint32_t exponent[kRows][kIter];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      sum[i] = mean[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        widen(x[i][k], raw.x[i][k]);
        if (kKeep) kept[i][k] = encode<T>(x[i][k], exponent[i][k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[i] += x[i][k][e];
      }
    }
    // before this batch's writes: a wait for later loads would wait for those too
    Walk then = now;
    then.next(a, kRows);
    read(raw, then);
    if (a.layer) {
      sum_row(sum, waves, room, turn);
#pragma unroll
      for (int i = 0; i < kRows; ++i) mean[i] = sum[i] * inv_dim;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      sum[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        const Place p(a, lane, k);
        const float here = p.n ? mean[i] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // what is not in the row is zero already, and stays it
          x[i][k][e] -= kOdd ? ((uint32_t)e < p.n ? mean[i] : 0.0f) : here;
          sum[i] += x[i][k][e] * x[i][k][e];
        }
      }
    }
    sum_row(sum, waves, room, turn);
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
      const bool live = i < now.count;
      const uint32_t row = live ? now.row + i : 0, pitch = a.groups * kGroup;
      const float r = rsqrtf(sum[i] * inv_dim + a.eps);
      const Window<float, false> stats(a.stats + 2 * (uint64_t)row, live && a.stats ? 2 : 0);
      typedef uint32_t Pair __attribute__((ext_vector_type(2)));
      __builtin_amdgcn_raw_buffer_store_b64(Pair{__builtin_bit_cast(uint32_t, mean[i]), __builtin_bit_cast(uint32_t, r)}, stats.buffer,
                                            lane == 0 ? 0 : kNowhere, 0, 0);
      const Window<T, kOdd> out((const T*)a.out + (uint64_t)row * a.dim, live ? a.dim : 0);
      const Window<int8_t, false> values(a.kept + (uint64_t)row * pitch, kKeep && live ? pitch : 0);
      const Window<uint8_t, false> exponents(a.kept_exponents + (uint64_t)row * a.groups, kKeep && live ? a.groups : 0);
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        const Place p(a, lane, k);
        Eight<T> result;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = x[i][k][e] * r * gain[k][e] + level[k][e];
          result.v[e] = (T)(now.sample == kNone ? 0.0f : v);
        }
        out.write(result, 0, p.at, live ? p.n : 0);
        if (kKeep) {
          __builtin_amdgcn_raw_buffer_store_b64(Pair{kept[i][k].x, kept[i][k].y}, values.buffer, p.at, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b8((uint8_t)exponent[i][k], exponents.buffer, lane % 4 == 0 ? p.at / kGroup : kNowhere, 0, 0);
        }
      }
    }
    fresh = then.sample != now.sample;
    now = then;
    if (now.row >= now.end) return;
  }
}

// Bound by memory, and by how few workgroups there may be, which leave their sums: bfloat16, 4608 rows of 3072 (85 MB) in 21 us,
// 4.1 TB/s; 17792 rows from 8 bits (275 MB) in 65, 4.2 TB/s. With 32 values a lane (8193 to 16384 a row) 24 to 67 of a lane's
// registers go to scratch: 4608 rows of 12288 (340 MB) in 79, 4.3 TB/s.
template <class T, int kIter, bool kKept, bool kOdd>
__device__ __forceinline__ void backward(const NormArgs& a) {
  constexpr int kRows = kBatch<kIter>;
  __shared__ float room[2 * 2 * kRows * 16];
  uint32_t turn = 0;
  const uint32_t side = a.per > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
  const uint32_t lane = threadIdx.x - side * a.lanes, waves = a.lanes / 64, group = blockIdx.x * a.per + side;
  const float inv_dim = 1.0f / (float)a.dim;
  Walk now(a, group * a.chunk, kRows);
  if (now.row >= now.end) return;
  struct Raw {
    Eight<T> x[kKept ? 1 : kRows][kIter], g[kRows][kIter];
    uint2 values[kKept ? kRows : 1][kIter];
    uint32_t exponents[kKept ? kRows : 1][kIter];
    float2 stats[kRows];
  };
  auto read = [&](Raw& raw, const Walk& w) {  // without branches, as in the forward pass
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
      const bool live = i < w.count;
      const uint32_t row = live ? w.row + i : 0, pitch = a.groups * kGroup;
      const Window<T, kOdd> x((const T*)a.x + row * a.x_stride, live ? a.dim : 0);
      const Window<T, kOdd> g((const T*)a.grad + row * a.grad_stride, live ? a.dim : 0);
      const Window<int8_t, false> q((const int8_t*)a.x + (uint64_t)row * pitch, live ? pitch : 0);
      const Window<uint8_t, false> exponent(a.x_exponents + (uint64_t)row * a.groups, live ? a.groups : 0);
      raw.stats[i] = ((const float2*)a.stats)[row];
      if (!live) raw.stats[i] = float2{0.0f, 0.0f};  // and zeros for what is read: nothing for any sum
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        const Place p(a, lane, k);
        if (kKept) {
          typedef uint32_t Pair __attribute__((ext_vector_type(2)));
          const Pair pair = __builtin_amdgcn_raw_buffer_load_b64(q.buffer, p.n ? p.at : kNowhere, 0, 0);
          raw.values[i][k] = uint2{pair.x, pair.y};
          raw.exponents[i][k] = __builtin_amdgcn_raw_buffer_load_b8(exponent.buffer, p.n ? p.at / kGroup : kNowhere, 0, 0);
        } else {
          raw.x[i][k] = x.read(0, p.at, live ? p.n : 0);
        }
        raw.g[i][k] = g.read(0, p.at, live ? p.n : 0);
      }
    }
  };
  Raw raw;
  read(raw, now);
  float gain[kIter][8];  // (1 + scale) w
  float along[kIter][8], plain[kIter][8];  // P and Q
  auto flush = [&](uint32_t sample) {
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
  bool fresh = true;
  while (true) {
    if (fresh) {
      float weight[kIter][8];
      vectors<kOdd, kIter>(weight, a, lane, a.weight, 0, a.weight_kind, 1.0f);
      vectors<kOdd, kIter>(gain, a, lane, now.sample == kNone ? nullptr : a.scale, now.sample * a.scale_stride, a.scale_kind, 0.0f);
#pragma unroll
      for (int k = 0; k < kIter; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gain[k][e] = now.sample == kNone ? 0.0f : weight[k][e] + weight[k][e] * gain[k][e];
          along[k][e] = plain[k][e] = 0.0f;
        }
    }
    float n[kRows][kIter][8], h[kRows][kIter][8], r[kRows], sums[2 * kRows];
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
      const float mean = raw.stats[i].x;
      r[i] = raw.stats[i].y;
      sums[2 * i] = sums[2 * i + 1] = 0.0f;
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        const Place p(a, lane, k);
        float g[8];
        if (kKept)
          decode(n[i][k], raw.values[i][k], raw.exponents[i][k]);
        else
          widen(n[i][k], raw.x[i][k]);
        widen(g, raw.g[i][k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          n[i][k][e] = (n[i][k][e] - mean) * r[i];  // past the row's end g is zero
          h[i][k][e] = g[e] * gain[k][e];
          along[k][e] += g[e] * n[i][k][e];
          plain[k][e] += g[e];
          sums[2 * i] += h[i][k][e] * n[i][k][e];
          sums[2 * i + 1] += h[i][k][e];
        }
      }
    }
    // before this batch's writes: a wait for later loads would wait for those too
    Walk then = now;
    then.next(a, kRows);
    read(raw, then);
    sum_row(sums, waves, room, turn);
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
      const bool live = i < now.count;
      const float mean_along = sums[2 * i] * inv_dim, mean_plain = a.layer ? sums[2 * i + 1] * inv_dim : 0.0f;
      const Window<T, kOdd> out((const T*)a.out + (uint64_t)(live ? now.row + i : 0) * a.dim, live ? a.dim : 0);
#pragma unroll
      for (int k = 0; k < kIter; ++k) {
        const Place p(a, lane, k);
        Eight<T> result;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          result.v[e] = (T)(now.sample == kNone ? 0.0f : r[i] * (h[i][k][e] - mean_plain - n[i][k][e] * mean_along));
        out.write(result, 0, p.at, live ? p.n : 0);
      }
    }
    const bool done = then.row >= then.end;
    fresh = !done && then.sample != now.sample;
    if (done || fresh) flush(now.sample);
    now = then;
    if (now.row >= now.end) return;
  }
}

// Names: type, times a lane holds 8 values; "odd": a dim that is no multiple of eight, or rows off the 4-byte grid.
#define MO_NORM(T, t, k, odd, name)                                                                          \
  extern "C" __global__ __launch_bounds__(512) void mo_norm_forward_##t##_##name(NormArgs a) {              \
    forward<T, k, false, odd>(a);                                                                            \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(512) void mo_norm_forward_keep_##t##_##name(NormArgs a) {         \
    forward<T, k, true, odd>(a);                                                                             \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(512) void mo_norm_backward_##t##_##name(NormArgs a) {             \
    backward<T, k, false, odd>(a);                                                                           \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(512) void mo_norm_backward_kept_##t##_##name(NormArgs a) {        \
    backward<T, k, true, odd>(a);                                                                            \
  }
#define MO_NORMS(T, t)           \
  MO_NORM(T, t, 1, false, 1)     \
  MO_NORM(T, t, 2, false, 2)     \
  MO_NORM(T, t, 4, false, 4)     \
  MO_NORM(T, t, 1, true, 1_odd)  \
  MO_NORM(T, t, 2, true, 2_odd)  \
  MO_NORM(T, t, 4, true, 4_odd)
MO_NORMS(_Float16, f16)
MO_NORMS(__bf16, bf16)
MO_NORMS(float, f32)

__device__ __forceinline__ float value_kind(const void* base, uint64_t at, uint32_t kind) {
  return kind == 2 ? ((const float*)base)[at] : kind == 1 ? (float)((const __bf16*)base)[at]
                                                          : (float)((const _Float16*)base)[at];
}

// A sample's sums over its workgroups for 16 columns: 64 runs of them side by side, then eight runs at a time, then the
// eight, all in order. Bound by the time to memory and back: 512 workgroups' sums of 3072 columns (13 MB) in 5.5 us, 7.5 with 64
// columns and 16 runs.
extern "C" __global__ __launch_bounds__(1024) void mo_norm_sums(NormArgs a) {
  __shared__ float room[2][64][17];
  const uint32_t column = threadIdx.x % 16, run = threadIdx.x / 16, sample = blockIdx.y;
  const uint32_t at = blockIdx.x * 16 + column;
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
#pragma unroll 8
    for (uint32_t i = from + run; i <= to; i += 64) {
      const float* p = a.partial + (uint64_t)(i + sample) * 2 * a.pitch + at;
      along += p[0];
      plain += p[a.pitch];
    }
  }
  room[0][run][column] = along;
  room[1][run][column] = plain;
  __syncthreads();
  if (run < 16) {  // the first eight add up the one, the others the other
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += room[run / 8][run % 8 * 8 + i][column];
    __builtin_amdgcn_wave_barrier();
    room[run / 8][run % 8 * 8][column] = sum;
  }
  __syncthreads();
  if (run || at >= a.dim) return;
  along = plain = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    along += room[0][i * 8][column];
    plain += room[1][i * 8][column];
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

// The weight's and the bias's gradients from the samples' sums, in order: a launch's latency, 4.2 us for four samples.
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
