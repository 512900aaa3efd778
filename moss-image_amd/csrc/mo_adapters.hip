// Low-rank adapters of many requests at once beside a shared projection, for gfx950.
//
//   h = x a_i^T,  y = result + c_i h b_i^T, i the adapter of the request that the row belongs to
//   backward, g the output's gradient:  d h = c_i g b_i,  d x = add + d h a_i,
//   d a_i = sum d h^T x,  d b_i = c_i sum g^T h over the rows of i's requests
// (one request with one adapter: the reference's LoRA linear, lora.py:60-86.)
//
// Three kernels: shrink (h and d h: rows against a weight's ranks, reduced over the features), expand (y and d x:
// reduced over the rank), outer (both weights' gradients: reduced over the rows). All are bound by the tokens that they
// read and write, so the matrix instructions have room: bfloat16 operands go into 16 x 16 x 32 ones, and the fp32
// numbers between the products in two bfloat16 parts, which leaves out 2^-16 of them at most; float16 and float32 go
// into the fp32 ones, 16 x 16 x 4, where float16 parts would under- and overflow.
//
// Rows are taken in tiles that lie in one request. Tile and request are found from the workgroup's number alone: what
// lies between a tile's border and a request's is at slot (tile + request), which no other pair has.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mo_adapters.h"
#include "mo_keep.h"

namespace {

using namespace mo_adapters;
using namespace mo_keep;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kNone = 0xffffffffu;

// ---- operands of the matrix instructions: eight values a lane, 32 of the reduced dimension a fragment ----

struct Eight32 {
  float v[8];
};

template <class T>
struct Path {  // fp32 instructions: lane (i, k) has values k * 8 to k * 8 + 7, one instruction for each of the eight
  typedef Eight32 Fragment;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ Fragment load(const T* p, uint32_t n) {
    Fragment f;
    widen(f.v, load8(p, n));
    return f;
  }
  static __device__ __forceinline__ Fragment part(const float (&v)[8], int) {
    Fragment f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = v[i];
    return f;
  }
  static __device__ __forceinline__ void multiply(f32x4& to, const Fragment& a, const Fragment& b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) to = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], to, 0, 0, 0);
  }
  // value q of each of eight rows
  static __device__ __forceinline__ Fragment column(const Eight<T> (&rows)[8], int q) {
    Fragment f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = (float)rows[i].v[q];
    return f;
  }
  static __device__ __forceinline__ Eight<T> decoded(uint2 values, uint32_t exponent) {
    float v[8];
    decode(v, values, exponent);
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = (T)v[i];
    return r;
  }
};

template <>
struct Path<__bf16> {
  typedef bf16x8 Fragment;
  static constexpr int kParts = 2;
  static __device__ __forceinline__ Fragment load(const __bf16* p, uint32_t n) {
    return __builtin_bit_cast(Fragment, load8(p, n));
  }
  // The upper half of an fp32 number (cut, so that nothing overflows), and the rest of it rounded to the nearest. What
  // is not finite has no rest.
  static __device__ __forceinline__ Fragment part(const float (&v)[8], int which) {
    Fragment f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, v[i]);
      const float high = __builtin_bit_cast(float, bits & 0xffff0000u);
      f[i] = which == 0 ? (__bf16)high : (bits & 0x7f800000u) == 0x7f800000u ? (__bf16)0.0f : (__bf16)(v[i] - high);
    }
    return f;
  }
  static __device__ __forceinline__ void multiply(f32x4& to, const Fragment& a, const Fragment& b) {
    to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, to, 0, 0, 0);
  }
  static __device__ __forceinline__ Fragment column(const Eight<__bf16> (&rows)[8], int q) {
    Fragment f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = rows[i].v[q];
    return f;
  }
  static __device__ __forceinline__ Eight<__bf16> decoded(uint2 values, uint32_t exponent) {
    float v[8];
    decode(v, values, exponent);
    Eight<__bf16> r;
#pragma unroll
    for (int i = 0; i < 8; ++i)  // seven bits under a power of two: exact
      r.v[i] = __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, v[i]) >> 16));
    return r;
  }
};

// ---- which rows have which adapter --------------------------------------------------------------------

__device__ __forceinline__ float scale_of(const Requests& by, uint32_t adapter) {
  return by.scale ? by.scale[adapter] * by.factor : by.factor;
}

// Where request s begins, within [0, rows] whatever the numbers given.
__device__ __forceinline__ uint32_t begins(const Requests& by, uint32_t s) {
  if (!by.cu) return s * by.share;
  const int64_t at = by.cu[s];
  return at < 0 ? 0 : at > (int64_t)by.rows ? by.rows : (uint32_t)at;
}
__device__ __forceinline__ uint32_t adapter_of(const Requests& by, uint32_t s) {
  if (!by.index) return by.adapters == 1 ? 0 : s;
  const int64_t i = by.index[s];
  return i < 0 || i >= (int64_t)by.adapters ? kNone : (uint32_t)i;
}

// Rows `low` to `high` - 1 of one request with its adapter; none where the slot is between two pairs.
struct Tile {
  uint32_t low, high, adapter;
};

// The requests, and before and behind them the rows that are in none: requests + 2 pieces, the rows of slot's.
template <uint32_t kRows>
__device__ __forceinline__ Tile tile_of(const Requests& by, uint32_t slot) {
  const uint32_t pieces = by.requests + 2;
  auto border = [&](uint32_t s) { return s == 0 ? 0u : s == pieces ? by.rows : begins(by, s - 1); };
  uint32_t low = 0, high = pieces - 1;  // the last piece whose first slot is not past this one
  while (high - low >= 64) {
    const uint32_t middle = (low + high + 1) / 2;
    if (border(middle) / kRows + middle <= slot)
      low = middle;
    else
      high = middle - 1;
  }
  const uint32_t mine = low + threadIdx.x % 64;
  const bool reached = mine <= high && border(mine) / kRows + mine <= slot;
  low += __popcll(__ballot(reached)) - 1;
  low = __builtin_amdgcn_readfirstlane(low);
  const uint32_t first = (slot - low) * kRows;
  Tile t;
  t.low = max(border(low), first);
  t.high = min(border(low + 1), first + kRows);
  t.adapter = low == 0 || low == pieces - 1 ? kNone : adapter_of(by, low - 1);
  return t;
}

// ---- shrink ------------------------------------------------------------------------------------------

// A workgroup has kTiles * 16 rows, all ranks and one split of the features; its waves take 64 features in turn and add
// up through LDS. The rows are the instruction's columns, so a lane ends with four neighbouring ranks of a row.
template <class T, int kRanks, int kTiles>
__device__ __forceinline__ void shrink(const Shrink& a) {
  typedef Path<T> P;
  constexpr uint32_t kRows = kTiles * 16, kPitch = kRanks * 16 + 4;
  __shared__ float room[4][kRows][kPitch];
  const Tile tile = tile_of<kRows>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = threadIdx.x / 64, i = lane % 16, k = lane / 16;
  f32x4 sum[kRanks][kTiles];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sum[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (tile.adapter != kNone) {
    const T* x[kTiles];
    const T* w[kRanks];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) x[t] = (const T*)a.x + min(tile.low + t * 16 + i, tile.high - 1) * a.x_stride + k * 8;
#pragma unroll
    for (int r = 0; r < kRanks; ++r)
      w[r] = (const T*)a.w + ((uint64_t)tile.adapter * rank + min(r * 16 + i, rank - 1)) * a.features + k * 8;
    const uint32_t first = blockIdx.y * a.span, last = min(a.features, first + a.span);
    auto step = [&](uint32_t at, auto whole) {
      typename P::Fragment xs[2][kTiles], ws[2][kRanks];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t from = at + u * 32, mine = from + k * 8;
        const uint32_t n = whole ? 8 : mine >= last ? 0 : min(8u, last - mine);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) xs[u][t] = P::load(x[t] + (n ? from : 0), n);
#pragma unroll
        for (int r = 0; r < kRanks; ++r) ws[u][r] = P::load(w[r] + (n ? from : 0), n);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < kRanks; ++r)
#pragma unroll
          for (int t = 0; t < kTiles; ++t) P::multiply(sum[r][t], ws[u][r], xs[u][t]);
    };
    uint32_t at = first + wave * 64;
    for (; at + 64 <= last; at += 256) step(at, std::true_type{});
    if (at < last) step(at, std::false_type{});
  }
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) *(f32x4*)&room[wave][t * 16 + i][r * 16 + k * 4] = sum[r][t];
  __syncthreads();
  const float scale = a.scaled && tile.adapter != kNone ? scale_of(a.by, tile.adapter) : 1.0f;
  float* to = a.to + ((uint64_t)blockIdx.y * a.by.rows + tile.low) * rank;
  const uint32_t rows = tile.high - tile.low;
  for (uint32_t e = threadIdx.x; e < rows * (kRanks * 16); e += 256) {
    const uint32_t row = e / (kRanks * 16), j = e % (kRanks * 16);
    if (j < rank) to[(uint64_t)row * rank + j] = (room[0][row][j] + room[1][row][j] + room[2][row][j] + room[3][row][j]) * scale;
  }
}

// ---- expand ------------------------------------------------------------------------------------------

// A workgroup has kTiles * 16 rows, whose h stays in registers, and `cols` columns a wave, 32 at a time. The columns are
// the instructions' rows, spread so that a lane ends with eight neighbouring columns of a row: 16 bytes to read
// and to write. With ranks up to 16 the two parts of h lie beside each other in one fragment.
template <class T, int kRank, int kTiles>
__device__ __forceinline__ void expand(const Expand& a) {
  typedef Path<T> P;
  constexpr uint32_t kRows = kTiles * 16;
  constexpr bool kBeside = kRank == 16 && P::kParts == 2;
  constexpr int kSteps = kRank < 32 ? 1 : kRank / 32, kParts = kBeside ? 1 : P::kParts;
  const Tile tile = tile_of<kRows>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = threadIdx.x / 64, i = lane % 16, k = lane / 16;
  const bool has = tile.adapter != kNone;
  typename P::Fragment h[kParts][kSteps][kTiles];
  float scale = 0.0f;
  if (has) {
    scale = a.scaled ? scale_of(a.by, tile.adapter) : 1.0f;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const uint32_t row = min(tile.low + t * 16 + i, tile.high - 1);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t j = kBeside ? k % 2 * 8 : s * 32 + k * 8, n = j >= rank ? 0 : min(8u, rank - j);
        float v[8];
        widen(v, load8(a.h + (uint64_t)row * rank + (n ? j : 0), n));
        for (uint32_t p = 1; p < a.splits; ++p) {
          float more[8];
          widen(more, load8(a.h + ((uint64_t)p * a.by.rows + row) * rank + (n ? j : 0), n));
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += more[e];
        }
        if (a.h_sum && blockIdx.y == 0 && wave == 0 && n && (!kBeside || k < 2) && tile.low + t * 16 + i < tile.high)
          store8(a.h_sum + (uint64_t)row * rank + j, v, n);
        if (kBeside) {
          const typename P::Fragment low = P::part(v, 1);
          h[0][s][t] = P::part(v, 0);
          if (k >= 2) h[0][s][t] = low;
        } else {
#pragma unroll
          for (int p = 0; p < kParts; ++p) h[p][s][t] = P::part(v, p);
        }
      }
    }
  } else if (a.h_sum && blockIdx.y == 0) {
    for (uint32_t e = threadIdx.x; e < (tile.high - tile.low) * rank; e += 256) a.h_sum[(uint64_t)tile.low * rank + e] = 0.0f;
  }
  const uint32_t first = (blockIdx.y * 4 + wave) * a.cols, last = min(a.features, first + a.cols);
  for (uint32_t at = first; at < last; at += 32) {
    const uint32_t col = at + k * 8, count = col >= a.features ? 0 : min(8u, a.features - col);
    Eight<T> base[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const uint32_t row = min(tile.low + t * 16 + i, tile.high - 1);
      const uint32_t n = a.base ? count : 0;
      base[t] = load8((const T*)a.base + (n ? row * a.base_stride + col : 0), n);
    }
    f32x4 sum[2][kTiles];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int t = 0; t < kTiles; ++t) sum[half][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (has) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t n = min(at + i / 4 * 8 + half * 4 + i % 4, a.features - 1);
        const T* v = (const T*)a.v + ((uint64_t)tile.adapter * a.features + n) * rank;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const uint32_t j = kBeside ? k % 2 * 8 : s * 32 + k * 8, m = j >= rank ? 0 : min(8u, rank - j);
          const typename P::Fragment f = P::load(v + (m ? j : 0), m);
#pragma unroll
          for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int t = 0; t < kTiles; ++t) P::multiply(sum[half][t], f, h[p][s][t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const uint32_t row = tile.low + t * 16 + i;
      float v[8];
      widen(v, base[t]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = has ? v[e] + scale * sum[e / 4][t][e % 4] : v[e];
      if (row < tile.high && count) store8((T*)a.to + (uint64_t)row * a.features + col, v, count);
    }
  }
}

// ---- outer -------------------------------------------------------------------------------------------

// A workgroup has 128 columns, 64 ranks at most and an adapter's rows in one split; its waves take 32 rows in turn and
// add up through LDS. A lane reads eight neighbouring columns of eight rows, and column q of all lanes makes the operand of
// instruction q: the rows, which are reduced, lie beside each other in a lane without a way through LDS. Rows
// past a request's end count as zeros on both sides (what lies there may be infinite).
template <class T, int kRanks, bool kKept>
__device__ __forceinline__ void outer(const Requests& by, const Side& a, uint32_t tile, float* room) {
  typedef Path<T> P;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, i = lane % 16, k = lane / 16;
  const uint32_t split = blockIdx.y, adapter = blockIdx.z % by.adapters, rank0 = blockIdx.z / by.adapters * (kRanks * 16);
  const uint32_t col = tile * kOuterCols + i * 8, count = col >= a.cols ? 0 : min(8u, a.cols - col);
  const uint32_t from = split * a.span, to = min(by.rows, from + a.span);
  f32x4 sum[kRanks][8];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int q = 0; q < 8; ++q) sum[r][q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  bool any = false;
  uint32_t turn = 0;

  auto step = [&](uint32_t row0, uint32_t high, auto whole) {
    Eight<T> wide[8];
    float narrow[kRanks][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t row = row0 + k * 8 + e;
      const bool in = whole || row < high;
      const uint32_t n = in ? count : 0;
      if (kKept) {
        uint2 q = {0, 0};
        uint32_t exponent = 0;
        if (n) {
          q = *(const uint2*)((const int8_t*)a.wide + (uint64_t)row * a.groups * kGroup + col);
          exponent = a.exponents[(uint64_t)row * a.groups + col / kGroup];
        }
        wide[e] = P::decoded(q, exponent);
      } else {
        wide[e] = load8((const T*)a.wide + (n ? row * a.stride + col : 0), n);
      }
#pragma unroll
      for (int r = 0; r < kRanks; ++r) {
        const uint32_t j = min(rank0 + r * 16 + i, by.rank - 1);
        narrow[r][e] = in ? a.narrow[(uint64_t)row * by.rank + j] : 0.0f;
      }
    }
#pragma unroll
    for (int r = 0; r < kRanks; ++r)
#pragma unroll
      for (int p = 0; p < P::kParts; ++p) {
        const typename P::Fragment f = P::part(narrow[r], p);
#pragma unroll
        for (int q = 0; q < 8; ++q) P::multiply(sum[r][q], f, P::column(wide, q));
      }
  };

  // the adapter's requests, 64 looked at at once
  for (uint32_t s0 = 0; s0 < by.requests; s0 += 64) {
    const uint32_t s = s0 + lane;
    uint32_t low = 0, high = 0;
    if (s < by.requests && adapter_of(by, s) == adapter) {
      low = max(begins(by, s), from);
      high = min(begins(by, s + 1), to);
    }
    uint64_t found = __ballot(low < high);
    any = any || found;
    while (found) {
      const int at = __builtin_ctzll(found);
      found &= found - 1;
      const uint32_t first = __builtin_amdgcn_readlane(low, at), last = __builtin_amdgcn_readlane(high, at);
      for (uint32_t row0 = first; row0 < last; row0 += 32, ++turn) {
        if (turn % 4 != wave) continue;
        if (row0 + 32 <= last)
          step(row0, last, std::true_type{});
        else
          step(row0, last, std::false_type{});
      }
    }
  }
  if (!any && a.splits > 1) return;  // nothing reads this plane

  // waves 2 and 3 to 0 and 1, then 1 to 0
  constexpr uint32_t kHeld = kRanks * 32;
#pragma unroll
  for (uint32_t apart = 2; apart; apart /= 2) {
    float* spot = room + (wave % apart) * kHeld * 64 + lane;
    __syncthreads();
    if (wave >= apart && wave < 2 * apart) {
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int e = 0; e < 32; ++e) spot[(r * 32 + e) * 64] = sum[r][e / 4][e % 4];
    }
    __syncthreads();
    if (wave < apart) {
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int e = 0; e < 32; ++e) sum[r][e / 4][e % 4] += spot[(r * 32 + e) * 64];
    }
  }
  if (wave || !count) return;
  const bool last = a.splits == 1;
  const float scale = last && a.scaled ? scale_of(by, adapter) : 1.0f;
  const uint64_t size = (uint64_t)a.cols * by.rank;
  float* plane = a.planes + ((uint64_t)split * by.adapters + adapter) * size;
  T* out = (T*)a.to + adapter * size;
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t j = rank0 + r * 16 + k * 4 + e;
      if (j >= by.rank) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = sum[r][q][e] * scale;
      if (a.turned) {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) {
          if (q >= count) continue;
          const uint64_t at = (uint64_t)(col + q) * by.rank + j;
          if (last)
            out[at] = (T)v[q];
          else
            plane[at] = v[q];
        }
      } else {
        const uint64_t at = (uint64_t)j * a.cols + col;
        if (last)
          store8(out + at, v, count);
        else
          store8(plane + at, v, count);
      }
    }
}

template <class T, int kRanks>
__device__ __forceinline__ void outer_sides(const Outer& a) {
  __shared__ float room[2 * kRanks * 32 * 64];
  const bool second = blockIdx.x >= a.side[0].tiles;
  const Side& side = a.side[second];
  if (blockIdx.y >= side.splits) return;
  const uint32_t tile = blockIdx.x - (second ? a.side[0].tiles : 0);
  if (side.exponents)
    outer<T, kRanks, true>(a.by, side, tile, room);
  else
    outer<T, kRanks, false>(a.by, side, tile, room);
}

// The planes of a gradient's splits that have rows of the adapter, added up in order.
template <class T>
__device__ __forceinline__ void join(const Outer& a) {
  __shared__ unsigned long long active;
  const Side& side = a.side[blockIdx.z];
  const uint64_t size = (uint64_t)side.cols * a.by.rank;
  if (!side.to || side.splits == 1 || (uint64_t)blockIdx.x * 1024 >= size) return;
  const uint32_t adapter = blockIdx.y;
  if (threadIdx.x == 0) active = 0;
  __syncthreads();
  for (uint32_t s = threadIdx.x; s < a.by.requests; s += 256) {
    if (adapter_of(a.by, s) != adapter) continue;
    const uint32_t low = begins(a.by, s), high = begins(a.by, s + 1);
    if (low >= high) continue;
    unsigned long long mask = 0;
    for (uint32_t p = low / side.span; p <= (high - 1) / side.span; ++p) mask |= 1ull << p;
    atomicOr(&active, mask);
  }
  __syncthreads();
  const uint64_t at = (uint64_t)blockIdx.x * 1024 + threadIdx.x * 4;
  if (at >= size) return;
  const uint32_t n = (uint32_t)min((uint64_t)4, size - at);
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint64_t left = active; left; left &= left - 1) {
    const float* from = side.planes + ((uint64_t)__builtin_ctzll(left) * a.by.adapters + adapter) * size + at;
    if (n == 4) {
      float more[4];
      __builtin_memcpy(more, from, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += more[e];
    } else {
      for (uint32_t e = 0; e < n; ++e) sum[e] += from[e];
    }
  }
  const float scale = side.scaled ? scale_of(a.by, adapter) : 1.0f;
  T* to = (T*)side.to + adapter * size + at;
  for (uint32_t e = 0; e < n; ++e) to[e] = (T)(sum[e] * scale);
}

// The splits of a shrink added up in order, where no expand does it on the way.
extern "C" __global__ __launch_bounds__(256) void mo_adapters_sum(const float* planes, float* to, uint64_t count, uint32_t splits) {
  const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= count) return;
  float sum = planes[at];
  for (uint32_t p = 1; p < splits; ++p) sum += planes[p * count + at];
  to[at] = sum;
}

// A weight turned, 32 x 32 through LDS.
template <class T>
__device__ __forceinline__ void turn(const Turn& a) {
  __shared__ T room[32][33];
  const bool second = blockIdx.x >= a.tiles[0];
  const uint32_t tile = blockIdx.x - (second ? a.tiles[0] : 0), rows = a.rows[second], cols = a.cols[second];
  const uint32_t across = (cols + 31) / 32, row0 = tile / across * 32, col0 = tile % across * 32;
  const uint32_t x = threadIdx.x % 32, y = threadIdx.x / 32;
  const uint64_t size = (uint64_t)rows * cols * blockIdx.y;
  const T* from = (const T*)a.from[second] + size;
  T* to = (T*)a.to[second] + size;
  for (uint32_t r = y; r < 32; r += 8)
    if (row0 + r < rows && col0 + x < cols) room[r][x] = from[(uint64_t)(row0 + r) * cols + col0 + x];
  __syncthreads();
  for (uint32_t r = y; r < 32; r += 8)
    if (col0 + r < cols && row0 + x < rows) to[(uint64_t)(col0 + r) * rows + row0 + x] = room[x][r];
}

#define MO_SHRINK(T, t, ranks, tiles)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_shrink_##t##_##ranks##_##tiles(Shrink a) {         \
    shrink<T, ranks, tiles>(a);                                                                                    \
  }
#define MO_EXPAND(T, t, rank, tiles)                                                                               \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_expand_##t##_##rank##_##tiles(Expand a) {          \
    expand<T, rank, tiles>(a);                                                                                     \
  }
#define MO_OUTER(T, t, ranks)                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_outer_##t##_##ranks(Outer a) { outer_sides<T, ranks>(a); }
#define MO_ADAPTERS(T, t)                                                                                          \
  MO_SHRINK(T, t, 1, 1)                                                                                            \
  MO_SHRINK(T, t, 1, 2)                                                                                            \
  MO_SHRINK(T, t, 2, 1)                                                                                            \
  MO_SHRINK(T, t, 2, 2)                                                                                            \
  MO_SHRINK(T, t, 4, 1)                                                                                            \
  MO_SHRINK(T, t, 4, 2)                                                                                            \
  MO_SHRINK(T, t, 8, 1)                                                                                            \
  MO_EXPAND(T, t, 16, 1)                                                                                           \
  MO_EXPAND(T, t, 16, 4)                                                                                           \
  MO_EXPAND(T, t, 32, 1)                                                                                           \
  MO_EXPAND(T, t, 32, 4)                                                                                           \
  MO_EXPAND(T, t, 64, 1)                                                                                           \
  MO_EXPAND(T, t, 64, 4)                                                                                           \
  MO_EXPAND(T, t, 128, 1)                                                                                          \
  MO_OUTER(T, t, 1)                                                                                                \
  MO_OUTER(T, t, 2)                                                                                                \
  MO_OUTER(T, t, 4)                                                                                                \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_join_##t(Outer a) { join<T>(a); }                  \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_turn_##t(Turn a) { turn<T>(a); }
MO_ADAPTERS(_Float16, f16)
MO_ADAPTERS(__bf16, bf16)
MO_ADAPTERS(float, f32)

}  // namespace
