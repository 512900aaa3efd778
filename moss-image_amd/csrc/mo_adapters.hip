// Low-rank adapters of many requests at once beside a shared projection, for gfx950.
//
//   h = x a_i^T,  y = result + c_i h b_i^T, i the adapter of the request that the row belongs to
//   backward, g the output's gradient:  d h = c_i g b_i,  d x = add + d h a_i,
//   d a_i = sum d h^T x,  d b_i = c_i sum g^T h over the rows of i's requests
// (one request with one adapter: the reference's LoRA linear, lora.py:60-86.)
//
// Three kernels: shrink (h and d h: rows against a weight's ranks, reduced over the features), expand (y and d x:
// reduced over the rank), outer (both weights' gradients: reduced over the rows). bfloat16 operands go into 16 x 16 x 32
// matrix instructions, and the fp32 numbers between the products in three bfloat16 parts, which are all of their 24 bits: what
// bounds these kernels is the tokens that they read and write. float16 and float32 go into the fp32 instructions, 16 x 16 x 4,
// where float16 parts would under- and overflow; at a sixteenth of the rate those are the bound from some 64 ranks on (17792 rows
// of 8192 and 3072 both ways, 64 ranks: 490 us by operations, 300 by bytes in float16; measured for 4608 rows 320 us, bfloat16 with 32
// ranks 137).
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

__device__ __forceinline__ uint32_t wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x / 64); }

// ---- operands of the matrix instructions: eight values a lane, 32 of the reduced dimension a fragment ----

struct Eight32 {
  float v[8];
};

template <class T>
struct Path {  // fp32 instructions: lane (i, k) has values k * 8 to k * 8 + 7, one instruction for each of the eight
  typedef Eight32 Fragment;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ Fragment of(const Eight<T>& v) {
    Fragment f;
    widen(f.v, v);
    return f;
  }
  static __device__ __forceinline__ void split(Fragment (&to)[1], const float (&v)[8], float = 1.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) to[0].v[i] = v[i];
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
  static constexpr int kParts = 3;
  static __device__ __forceinline__ Fragment of(const Eight<__bf16>& v) { return __builtin_bit_cast(Fragment, v); }
  // fp32 numbers as sums of three bfloat16 ones: the upper half of the number (cut, so that nothing overflows), that of
  // the rest, and `last` times what is left, eight bits each: none is lost. What is not finite has no rest. (A number of few bits
  // has parts of zero, which make NaN of an infinity on the other side.)
  static __device__ __forceinline__ void split(Fragment (&to)[3], const float (&v)[8], float last = 1.0f) {
    uint32_t words[3][4];
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = v[i];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      uint32_t bits[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bits[i] = __builtin_bit_cast(uint32_t, p == 2 ? rest[i] * last : rest[i]);
        rest[i] -= __builtin_bit_cast(float, bits[i] & 0xffff0000u);
        if (p == 0) rest[i] = (bits[i] & 0x7f800000u) == 0x7f800000u ? 0.0f : rest[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) words[p][i] = __builtin_amdgcn_perm(bits[2 * i + 1], bits[2 * i], 0x07060302u);
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) to[p] = __builtin_bit_cast(Fragment, words[p]);
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

// Rows `low` to `high` - 1 of one piece; none where the slot is between two pairs. The pieces are the requests, and before
// and behind them the rows that are in none.
struct Tile {
  uint32_t low, high, piece;
};

// The rows of a slot. What the lanes look at is read at once, so that this waits for memory once.
template <uint32_t kRows>
__device__ __forceinline__ Tile tile_of(const Requests& by, uint32_t slot) {
  const uint32_t pieces = by.requests + 2;
  auto border = [&](uint32_t s) { return s == 0 ? 0u : s >= pieces ? by.rows : begins(by, s - 1); };
  uint32_t low = 0, high = pieces - 1;  // the last piece whose first slot is not past this one
  while (high - low >= 64) {
    const uint32_t middle = (low + high + 1) / 2;
    if (border(middle) / kRows + middle <= slot)
      low = middle;
    else
      high = middle - 1;
  }
  const uint32_t mine = min(low + threadIdx.x % 64, high), from = border(mine), to = border(mine + 1);
  const bool reached = low + threadIdx.x % 64 <= high && from / kRows + mine <= slot;
  const int at = __popcll(__ballot(reached)) - 1;
  Tile t;
  t.piece = __builtin_amdgcn_readfirstlane(low) + at;
  const uint32_t first = (slot - t.piece) * kRows;
  t.low = max((uint32_t)__builtin_amdgcn_readlane(from, at), first);
  t.high = min((uint32_t)__builtin_amdgcn_readlane(to, at), first + kRows);
  return t;
}
// Its adapter: another wait, so asked for after what does not need it.
__device__ __forceinline__ uint32_t adapter_of(const Requests& by, const Tile& t) {
  if (t.piece == 0 || t.piece == by.requests + 1) return kNone;
  return __builtin_amdgcn_readfirstlane(adapter_of(by, t.piece - 1));
}

// ---- shrink ------------------------------------------------------------------------------------------

// A workgroup has 16 rows, all ranks and one split of the features; its eight waves take 128 features in turn and
// add up through LDS. A wave reads 256 bytes of each row side by side (64 bytes a row, as the instructions want them, came
// at 4.2 TB/s where this comes at 5.4) and turns them through its own part of LDS, eight values at a time; those of
// row r lie at (place ^ r), so that neither writing nor reading meets a bank twice. The rows are the instruction's
// columns, so a lane ends with four neighbouring ranks of a row. Nothing is loaded ahead: sixteen waves a CU are enough.
// Bound by the way to memory and back: bfloat16, 16 ranks, 4608 rows of 3072 (28 MB) in 11.5 us, 2.5 TB/s. More than 64 ranks of float32,
// or of float16 in odd sizes, leave no registers for all (268 to 432 bytes a lane in scratch): 4608 rows of 8192, 128 ranks, float32 265 us.
template <class T, int kRanks, bool kOdd>
__device__ __forceinline__ void shrink(const Shrink& a) {
  typedef Path<T> P;
  constexpr uint32_t kPitch = kRanks * 16 + 4;
  union Room {
    Eight<T> stage[8][16][16];
    float sums[8][16][kPitch];
    __device__ Room() {}
  };
  __shared__ Room room;
  const Tile tile = tile_of<16>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = wave_of(), i = lane % 16, k = lane / 16;
  f32x4 sum[kRanks];
#pragma unroll
  for (int r = 0; r < kRanks; ++r) sum[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t adapter = adapter_of(a.by, tile);
  if (adapter != kNone) {
    const uint32_t stride = (uint32_t)a.x_stride, rows = tile.high - tile.low;
    const Window<T, kOdd> x((const T*)a.x + tile.low * a.x_stride, (rows - 1) * stride + a.features);
    const Window<T, kOdd> w((const T*)a.w + (uint64_t)(a.by_request ? tile.piece - 1 : adapter) * rank * a.features, rank * a.features);
    const uint32_t first = blockIdx.y * a.span, last = min(a.features, first + a.span);
    for (uint32_t at = first + wave * 128; at < last; at += 1024) {
      Eight<T> xs[4], ws[4][kRanks];
      const uint32_t n = at + i * 8 >= last ? 0 : min(8u, last - at - i * 8);
#pragma unroll
      for (uint32_t t = 0; t < 4; ++t) xs[t] = x.read(t * 4 * stride + at, k * stride + i * 8, t * 4 + k < rows ? n : 0);
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t from = at + u * 32 + k * 8, m = from >= last ? 0 : min(8u, last - from);
#pragma unroll
        for (uint32_t r = 0; r < kRanks; ++r)
          ws[u][r] = w.read(r * 16 * a.features + at + u * 32, i * a.features + k * 8, r * 16 + i < rank ? m : 0);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) room.stage[wave][t * 4 + k][i ^ (t * 4 + k)] = xs[t];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const typename P::Fragment f = P::of(room.stage[wave][i][(u * 4 + k) ^ i]);
#pragma unroll
        for (int r = 0; r < kRanks; ++r) P::multiply(sum[r], P::of(ws[u][r]), f);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRanks; ++r) *(f32x4*)&room.sums[wave][i][r * 16 + k * 4] = sum[r];
  __syncthreads();
  const float scale = a.scaled && adapter != kNone ? scale_of(a.by, adapter) : 1.0f;
  float* to = a.to + ((uint64_t)blockIdx.y * a.by.rows + tile.low) * rank;
  for (uint32_t e = threadIdx.x; e < (tile.high - tile.low) * (kRanks * 16); e += 512) {
    const uint32_t row = e / (kRanks * 16), j = e % (kRanks * 16);
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) total += room.sums[u][row][j];
    if (j < rank) to[(uint64_t)row * rank + j] = total * scale;
  }
}

// The same for many rows in long requests: a wave has 16 rows of its own and the weight, which is read for each tile and
// with many ranks would be more than the rows themselves, comes to LDS once for all eight waves, one step ahead. Bound by
// memory: bfloat16, 16 ranks, 4608 rows of 16384 (151 MB) in 42.5 us, 3.6 TB/s; 64 ranks, 17792 rows of 8192 (292 MB) in 65, 4.5 TB/s.
template <class T, int kRanks>
__device__ __forceinline__ void shrink_tall(const Shrink& a) {
  typedef Path<T> P;
  constexpr uint32_t kRows = 128;
  __shared__ Eight<T> stage[8][16][16], weight[2][kRanks * 16][16];
  const Tile tile = tile_of<kRows>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = wave_of(), i = lane % 16, k = lane / 16;
  f32x4 sum[kRanks];
#pragma unroll
  for (int r = 0; r < kRanks; ++r) sum[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t low = tile.low + wave * 16, rows = low >= tile.high ? 0 : min(16u, tile.high - low);
  const uint32_t adapter = adapter_of(a.by, tile);
  if (adapter != kNone) {
    const uint32_t stride = (uint32_t)a.x_stride;
    const Window<T, false> x((const T*)a.x + (rows ? low : tile.low) * a.x_stride, rows ? (rows - 1) * stride + a.features : 0);
    const Window<T, false> w((const T*)a.w + (uint64_t)(a.by_request ? tile.piece - 1 : adapter) * rank * a.features, rank * a.features);
    const uint32_t first = blockIdx.y * a.span, last = min(a.features, first + a.span);
    Eight<T> xs[4], ws[(kRanks + 1) / 2];
    // a thread's eight columns of four rows, and of every 32nd rank
    const uint32_t wide = threadIdx.x % 16, tall = threadIdx.x / 16;
    auto load = [&](uint32_t at) {
#pragma unroll
      for (uint32_t t = 0; t < 4; ++t)
        xs[t] = x.read(t * 4 * stride + at, k * stride + i * 8, t * 4 + k < rows && at + i * 8 < last ? 8 : 0);
#pragma unroll
      for (uint32_t t = 0; t < (kRanks + 1) / 2; ++t)
        ws[t] = w.read(t * 32 * a.features + at, tall * a.features + wide * 8, t * 32 + tall < rank && at + wide * 8 < last ? 8 : 0);
    };
    load(first);
    uint32_t turn = 0;
    for (uint32_t at = first; at < last; at += 128, turn ^= 1) {
#pragma unroll
      for (int t = 0; t < 4; ++t) stage[wave][t * 4 + k][i ^ (t * 4 + k)] = xs[t];
#pragma unroll
      for (uint32_t t = 0; t < (kRanks + 1) / 2; ++t)
        if (t * 32 + tall < kRanks * 16) weight[turn][t * 32 + tall][wide ^ tall % 16] = ws[t];
      __syncthreads();  // the other buffer has been read by all when they come here again
      if (at + 128 < last) load(at + 128);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const typename P::Fragment f = P::of(stage[wave][i][(u * 4 + k) ^ i]);
#pragma unroll
        for (int r = 0; r < kRanks; ++r) P::multiply(sum[r], P::of(weight[turn][r * 16 + i][(u * 4 + k) ^ i]), f);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (i >= rows) return;
  const float scale = a.scaled && adapter != kNone ? scale_of(a.by, adapter) : 1.0f;
  float* to = a.to + ((uint64_t)blockIdx.y * a.by.rows + low + i) * rank;
#pragma unroll
  for (int r = 0; r < kRanks; ++r) {
    const uint32_t j = r * 16 + k * 4;
    if (j < rank) {  // a multiple of eight ranks
      const f32x4 v = sum[r] * scale;
      __builtin_memcpy(to + j, &v, 16);
    }
  }
}

// ---- expand ------------------------------------------------------------------------------------------

// Where a value of a narrow matrix lies turned, for the instructions of an outer: fp32 [rows / 8][rank][8 rows], so that a
// fragment is read from neighbouring places.
__device__ __forceinline__ uint64_t turned_at(uint32_t rank, uint32_t j, uint32_t row) {
  return ((uint64_t)(row / 8) * rank + j) * 8 + row % 8;
}

// A workgroup has 16 rows, whose h stays in registers, and `cols` columns, of which a wave takes 128 at a time. The
// columns are the instructions' rows, so a lane ends with four neighbouring columns of a row; through the wave's own
// part of LDS they come to lanes that read and write 256 bytes of a row side by side. With ranks up to 16 the first two
// parts of h lie beside each other in one fragment, the third's halves in another (beside zeros an infinite v would
// give NaN). (32 rows, which read v half as often, were slower: 4608 rows, 16 ranks, 3072 columns 25.5 us for 21.2.) Bound by memory: 16 ranks, 4608 rows of 16384 (302 MB, read and written) in 61 us, 4.9 TB/s; of 3072
// (57 MB, and 23 of h's 13 planes, which each of six workgroups beside another adds up) in 20.7, 3.8 TB/s.
template <class T, int kRank, bool kOdd>
__device__ __forceinline__ void expand(const Expand& a) {
  typedef Path<T> P;
  constexpr bool kBeside = kRank == 16 && P::kParts == 3;
  constexpr int kSteps = kRank < 32 ? 1 : kRank / 32, kParts = kBeside ? 2 : P::kParts;
  __shared__ float room[4][16][132];
  float(*shared)[132] = room[0];  // before the waves use their parts
  const Tile tile = tile_of<16>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = wave_of(), i = lane % 16, k = lane / 16;
  const uint32_t first = blockIdx.y * a.cols, end = min(a.features, first + a.cols);
  const uint32_t stride = (uint32_t)a.base_stride, rows = tile.high - tile.low;
  // a lane's rows (k, and every fourth after it) and columns where memory is read and written
  const Window<T, kOdd> base((const T*)a.base + tile.low * a.base_stride, a.base ? (rows - 1) * stride + a.features : 0);
  const Window<T, kOdd> to((const T*)a.to + (uint64_t)tile.low * a.features, rows * a.features);
  Eight<T> in[4];
  auto count = [&](uint32_t at) { return at + i * 8 >= end ? 0 : min(8u, end - at - i * 8); };
  auto read_base = [&](uint32_t at) {
#pragma unroll
    for (uint32_t t = 0; t < 4; ++t) {
      if (kOdd && !a.base)
        in[t] = Eight<T>{};
      else
        in[t] = base.read(t * 4 * stride + at, k * stride + i * 8, t * 4 + k < rows ? count(at) : 0);
    }
  };
  // the first step's loads are on their way while h's are waited for
  uint32_t at = first + wave * 128;
  read_base(at);
  const uint32_t adapter = adapter_of(a.by, tile);
  const bool has = adapter != kNone;
  const Window<T, kOdd> v((const T*)a.v + (uint64_t)(!has ? 0 : a.by_request ? tile.piece - 1 : adapter) * a.features * rank, a.features * rank);
  Eight<T> vs[8][kSteps];
  auto read_v = [&](uint32_t at) {
#pragma unroll
    for (uint32_t c = 0; c < 8; ++c)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t j = kBeside ? k % 2 * 8 : s * 32 + k * 8, n = j >= rank ? 0 : min(8u, rank - j);
        vs[c][s] = v.read((at + c * 16) * rank, i * rank + j, at + c * 16 + i < a.features ? n : 0);
      }
  };
  if (has) read_v(at);
  typename P::Fragment h[kParts][kSteps];
  float scale = 0.0f;
  if (has) {
    scale = a.scaled ? scale_of(a.by, adapter) : 1.0f;
    // h's splits added up, a part of the tile a thread, and from LDS to the lanes that need it
    const uint32_t row = threadIdx.x / 16;
    for (uint32_t j0 = threadIdx.x % 16 * 4; j0 < kRank; j0 += 64) {
      f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (row < rows) {
        const float* from = a.h + (uint64_t)(tile.low + row) * rank + j0;
#pragma unroll 4
        for (uint32_t p = 0; p < a.splits; ++p, from += (uint64_t)a.by.rows * rank) {
          f32x4 more = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if (!kOdd && j0 < rank) __builtin_memcpy(&more, from, 16);
          if (kOdd) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
              if (j0 + e < rank) more[e] = from[e];
          }
          sum = p ? sum + more : more;
        }
        if (blockIdx.y == 0) {
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            if (j0 + e >= rank) continue;
            if (a.h_sum) a.h_sum[(uint64_t)(tile.low + row) * rank + j0 + e] = sum[e];
            if (a.turned) a.turned[turned_at(rank, j0 + e, tile.low + row)] = sum[e];
          }
        }
      }
      *(f32x4*)&shared[row][j0] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint32_t j = kBeside ? k % 2 * 8 : s * 32 + k * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = j < kRank ? shared[i][j + e] : 0.0f;
      typename P::Fragment parts[P::kParts];
      P::split(parts, v, kBeside ? 0.5f : 1.0f);
      if (kBeside) {
        h[0][s] = k < 2 ? parts[0] : parts[P::kParts / 2];
        h[kParts - 1][s] = parts[P::kParts - 1];
      } else {
#pragma unroll
        for (int p = 0; p < kParts; ++p) h[p][s] = parts[p];
      }
    }
    __syncthreads();
  } else if (blockIdx.y == 0 && a.h_sum) {
    for (uint32_t e = threadIdx.x; e < (tile.high - tile.low) * rank; e += 256) a.h_sum[(uint64_t)tile.low * rank + e] = 0.0f;
  }
  while (at < end) {
    if (has) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int p = 0; p < kParts; ++p) P::multiply(sum, P::of(vs[c][s]), h[p][s]);
        *(f32x4*)&room[wave][i][c * 16 + k * 4] = sum;
      }
      __builtin_amdgcn_wave_barrier();
    }
    // the next step's loads go out before this one's writes, which a wait for later loads would wait for too
    if (has && at + 512 < end) read_v(at + 512);
    Eight<T> results[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      float out[8];
      widen(out, in[u]);
      if (has) {
        float more[8];
        __builtin_memcpy(more, __builtin_assume_aligned(&room[wave][u * 4 + k][i * 8], 16), 32);
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] += scale * more[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) results[u].v[e] = (T)out[e];
    }
    if (at + 512 < end) read_base(at + 512);
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
      to.write(results[u], u * 4 * a.features + at, k * a.features + i * 8, u * 4 + k < rows ? count(at) : 0);
    __builtin_amdgcn_wave_barrier();
    at += 512;
  }
}

// The same for more than 16 ranks and many rows: a wave has 32 rows of its own, all four waves take the same columns,
// and v's part of them, as large as the rows' own at 64 ranks, comes to LDS once, a step ahead in registers. Bound by memory,
// of which h's planes are a part, since every workgroup beside another reads them: bfloat16, 64 ranks, 17792 rows of 8192 (583 MB, and 109 of
// planes for eight workgroups) in 121 us, 5.7 TB/s; of 3072 (219 MB, and 82 of planes for six) in 59, 5.1 TB/s.
template <class T, int kRank>
__device__ __forceinline__ void expand_tall(const Expand& a) {
  typedef Path<T> P;
  constexpr uint32_t kRows = 128, kChunks = kRank / 8, kMine = 128 * kChunks / 256;
  constexpr int kSteps = kRank / 32;
  __shared__ float room[4][16][132];
  __shared__ Eight<T> weight[128][kChunks];
  const Tile tile = tile_of<kRows>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = wave_of(), i = lane % 16, k = lane / 16;
  const uint32_t first = blockIdx.y * a.cols, end = min(a.features, first + a.cols);
  const uint32_t low = tile.low + wave * 32, rows = low >= tile.high ? 0 : min(32u, tile.high - low);
  const uint32_t stride = (uint32_t)a.base_stride;
  const uint64_t from = rows ? low : tile.low;  // a wave without rows reads and writes none
  const Window<T, false> base((const T*)a.base + from * a.base_stride, a.base && rows ? (rows - 1) * stride + a.features : 0);
  const Window<T, false> to((const T*)a.to + from * a.features, rows * a.features);
  Eight<T> in[8];
  auto count = [&](uint32_t at) { return at + i * 8 < end ? 8u : 0u; };
  auto read_base = [&](uint32_t at, int t) {
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t row = t * 16 + u * 4;
      in[t * 4 + u] = base.read(row * stride + at, k * stride + i * 8, row + k < rows ? count(at) : 0);
    }
  };
  read_base(first, 0);
  read_base(first, 1);
  const uint32_t adapter = adapter_of(a.by, tile);
  const bool has = adapter != kNone;
  const Window<T, false> v((const T*)a.v + (uint64_t)(!has ? 0 : a.by_request ? tile.piece - 1 : adapter) * a.features * rank, a.features * rank);
  Eight<T> mine[kMine];
  auto read_v = [&](uint32_t at) {
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
      const uint32_t place = e * 256 + threadIdx.x, n = place / kChunks, j = place % kChunks * 8;
      mine[e] = v.read(at * rank, n * rank + j, j < rank && at + n < a.features ? 8 : 0);
    }
  };
  typename P::Fragment h[P::kParts][kSteps][2];
  float scale = 0.0f;
  if (has) {
    read_v(first);
    scale = a.scaled ? scale_of(a.by, adapter) : 1.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t j = s * 32 + k * 8, row = t * 16 + i;
        float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (row < rows && j < rank) {
          const float* p = a.h + (uint64_t)(low + row) * rank + j;
          widen(sum, load8(p));
#pragma unroll 2
          for (uint32_t split = 1; split < a.splits; ++split) {
            float more[8];
            widen(more, load8(p + (uint64_t)split * a.by.rows * rank));
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += more[e];
          }
          if (blockIdx.y == 0) {
            if (a.h_sum) store8(a.h_sum + (uint64_t)(low + row) * rank + j, sum);
            if (a.turned) {
#pragma unroll
              for (uint32_t e = 0; e < 8; ++e) a.turned[turned_at(rank, j + e, low + row)] = sum[e];
            }
          }
        }
        typename P::Fragment parts[P::kParts];
        P::split(parts, sum);
#pragma unroll
        for (int p = 0; p < P::kParts; ++p) h[p][s][t] = parts[p];
      }
  } else if (blockIdx.y == 0 && a.h_sum) {
    for (uint32_t e = threadIdx.x; e < (tile.high - tile.low) * rank; e += 256) a.h_sum[(uint64_t)tile.low * rank + e] = 0.0f;
  }
  for (uint32_t at = first; at < end; at += 128) {
    const bool more_cols = at + 128 < end;
    if (has) {
      __syncthreads();  // the last step's part has been read
#pragma unroll
      for (uint32_t e = 0; e < kMine; ++e) {
        const uint32_t place = e * 256 + threadIdx.x, n = place / kChunks, chunk = place % kChunks;
        weight[n][chunk ^ n % kChunks] = mine[e];
      }
      __syncthreads();
      if (more_cols) read_v(at + 128);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (has) {
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) {
          const uint32_t n = c * 16 + i;
          f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (uint32_t s = 0; s < kSteps; ++s) {
            const typename P::Fragment f = P::of(weight[n][(s * 4 + k) ^ n % kChunks]);
#pragma unroll
            for (int p = 0; p < P::kParts; ++p) P::multiply(sum, f, h[p][s][t]);
          }
          *(f32x4*)&room[wave][i][c * 16 + k * 4] = sum;
        }
        __builtin_amdgcn_wave_barrier();
      }
      Eight<T> results[4];
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        float out[8];
        widen(out, in[t * 4 + u]);
        if (has) {
          float more[8];
          __builtin_memcpy(more, __builtin_assume_aligned(&room[wave][u * 4 + k][i * 8], 16), 32);
#pragma unroll
          for (int e = 0; e < 8; ++e) out[e] += scale * more[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) results[u].v[e] = (T)out[e];
      }
      if (more_cols) read_base(at + 128, t);  // before the writes, which a wait for later loads would wait for too
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t row = t * 16 + u * 4;
        to.write(results[u], row * a.features + at, k * a.features + i * 8, row + k < rows ? count(at) : 0);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// A forward pass of few rows in one launch: a workgroup has 16 rows and 1024 columns, 128 a wave, and makes its own h over
// all features, its waves by turns of 128, added up in one order. What it reads of b and the base arrives meanwhile, and a
// comes from the caches after its first reading. Bound by the way to memory and back: 16 rows of 3072 with 16 adapters of
// 16 ranks in bfloat16 8.4 us (3.4 MB), in two launches 9.4.
template <class T, int kRanks>
__device__ __forceinline__ void few(const Few& f) {
  typedef Path<T> P;
  const Shrink& a = f.in;
  const Expand& b = f.out;
  constexpr uint32_t kRank = kRanks * 16, kPitch = kRank + 4;
  constexpr bool kBeside = kRanks == 1 && P::kParts == 3;
  constexpr int kSteps = kRank < 32 ? 1 : kRank / 32, kParts = kBeside ? 2 : P::kParts;
  union Room {
    Eight<T> stage[8][16][16];
    float sums[8][16][kPitch];
    float out[8][16][132];
    __device__ Room() {}
  };
  __shared__ Room room;
  __shared__ float h[16][kPitch];
  const Tile tile = tile_of<16>(a.by, blockIdx.x);
  if (tile.low >= tile.high) return;
  const uint32_t rank = a.by.rank, lane = threadIdx.x % 64, wave = wave_of(), i = lane % 16, k = lane / 16;
  const uint32_t rows = tile.high - tile.low, x_stride = (uint32_t)a.x_stride, stride = (uint32_t)b.base_stride;
  const uint32_t at = blockIdx.y * 1024 + wave * 128, count = at + i * 8 < b.features ? 8 : 0;
  const Window<T, false> base((const T*)b.base + tile.low * b.base_stride, (rows - 1) * stride + b.features);
  const Window<T, false> to((const T*)b.to + (uint64_t)tile.low * b.features, rows * b.features);
  Eight<T> in[4];
#pragma unroll
  for (uint32_t u = 0; u < 4; ++u) in[u] = base.read(u * 4 * stride + at, k * stride + i * 8, u * 4 + k < rows ? count : 0);
  const uint32_t adapter = adapter_of(a.by, tile);
  const bool has = adapter != kNone;
  Eight<T> vs[8][kSteps];
  f32x4 sum[kRanks];
#pragma unroll
  for (int r = 0; r < kRanks; ++r) sum[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (has) {
    const Window<T, false> v((const T*)b.v + (uint64_t)adapter * b.features * rank, b.features * rank);
#pragma unroll
    for (uint32_t c = 0; c < 8; ++c)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t j = kBeside ? k % 2 * 8 : s * 32 + k * 8;
        vs[c][s] = v.read((at + c * 16) * rank, i * rank + j, j < rank && at + c * 16 + i < b.features ? 8 : 0);
      }
    const Window<T, false> x((const T*)a.x + tile.low * a.x_stride, (rows - 1) * x_stride + a.features);
    const Window<T, false> w((const T*)a.w + (uint64_t)adapter * rank * a.features, rank * a.features);
    for (uint32_t from = wave * 128; from < a.features; from += 1024) {
      Eight<T> xs[4], ws[4][kRanks];
#pragma unroll
      for (uint32_t t = 0; t < 4; ++t)
        xs[t] = x.read(t * 4 * x_stride + from, k * x_stride + i * 8, t * 4 + k < rows && from + i * 8 < a.features ? 8 : 0);
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
        for (uint32_t r = 0; r < kRanks; ++r)
          ws[u][r] = w.read(r * 16 * a.features + from + u * 32, i * a.features + k * 8,
                            r * 16 + i < rank && from + u * 32 + k * 8 < a.features ? 8 : 0);
#pragma unroll
      for (int t = 0; t < 4; ++t) room.stage[wave][t * 4 + k][i ^ (t * 4 + k)] = xs[t];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const typename P::Fragment of = P::of(room.stage[wave][i][(u * 4 + k) ^ i]);
#pragma unroll
        for (int r = 0; r < kRanks; ++r) P::multiply(sum[r], P::of(ws[u][r]), of);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRanks; ++r) *(f32x4*)&room.sums[wave][i][r * 16 + k * 4] = sum[r];
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < 16 * kRank; e += 512) {
    const uint32_t row = e / kRank, j = e % kRank;
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) total += room.sums[u][row][j];
    h[row][j] = j < rank ? total : 0.0f;  // past the rank the sum is of zeros times the tokens, NaN for infinite ones
    if (blockIdx.y == 0 && row < rows && j < rank) a.to[(uint64_t)(tile.low + row) * rank + j] = total;
  }
  __syncthreads();
  if (has) {
    typename P::Fragment hs[kParts][kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint32_t j = kBeside ? k % 2 * 8 : s * 32 + k * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = j < kRank ? h[i][j + e] : 0.0f;
      typename P::Fragment parts[P::kParts];
      P::split(parts, v, kBeside ? 0.5f : 1.0f);
      if (kBeside) {
        hs[0][s] = k < 2 ? parts[0] : parts[P::kParts / 2];
        hs[kParts - 1][s] = parts[P::kParts - 1];
      } else {
#pragma unroll
        for (int p = 0; p < kParts; ++p) hs[p][s] = parts[p];
      }
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      f32x4 part = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int p = 0; p < kParts; ++p) P::multiply(part, P::of(vs[c][s]), hs[p][s]);
      *(f32x4*)&room.out[wave][i][c * 16 + k * 4] = part;
    }
    __builtin_amdgcn_wave_barrier();
  }
  const float scale = has ? scale_of(a.by, adapter) : 0.0f;
#pragma unroll
  for (uint32_t u = 0; u < 4; ++u) {
    float out[8];
    widen(out, in[u]);
    if (has) {
      float more[8];
      __builtin_memcpy(more, __builtin_assume_aligned(&room.out[wave][u * 4 + k][i * 8], 16), 32);
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] += scale * more[e];
    }
    Eight<T> result;
#pragma unroll
    for (int e = 0; e < 8; ++e) result.v[e] = (T)out[e];
    to.write(result, u * 4 * b.features + at, k * b.features + i * 8, u * 4 + k < rows ? count : 0);
  }
}

// ---- outer -------------------------------------------------------------------------------------------

// A workgroup has 128 columns, 64 ranks at most and an adapter's rows in one split; its waves take 32 rows in turn and
// add up through LDS. A lane reads eight neighbouring columns of eight rows, and column q of all lanes makes the operand of
// instruction q: the rows, which are reduced, lie beside each other in a lane without a way through LDS. A step's rows
// begin at a multiple of 32; those that are not the request's count as zeros on both sides (they may be infinite). bfloat16:
// 16 ranks, 4608 rows of 16384 and, in 8 bits, 3072 (166 MB) in 31 us, 5.3 TB/s, bound by memory; 64 ranks, 17792 rows of 8192 and
// 3072 (401 MB) in 142, 2.8 TB/s, where the sums leave registers for two waves a SIMD (seven more values go to scratch), too few to
// cover the loads, of which none is asked for a step ahead.
template <class T, int kRanks, bool kKept, bool kOdd>
__device__ __forceinline__ void outer(const Requests& by, const Side& a, uint32_t tile, f32x4* room) {
  typedef Path<T> P;
  const uint32_t lane = threadIdx.x % 64, wave = wave_of(), i = lane % 16, k = lane / 16;
  const uint32_t split = blockIdx.y, adapter = blockIdx.z % by.adapters, rank0 = blockIdx.z / by.adapters * (kRanks * 16);
  const uint32_t col = tile * kOuterCols + i * 8, count = col >= a.cols ? 0 : min(8u, a.cols - col);
  const uint32_t from = split * a.span, to = min(by.rows, from + a.span);
  f32x4 sum[kRanks][8];
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int q = 0; q < 8; ++q) sum[r][q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // The wave's steps of 32 rows: the adapter's requests, 64 looked at at once, and in each every fourth step, from
  // another wave on for the next request.
  uint32_t s0 = 0, low = 0, high = 0, pieces = 0, row0 = 0, first = 0, last = 0;
  uint64_t found = 0;
  auto look = [&]() {
    const uint32_t s = s0 + lane;
    low = high = 0;
    if (s < by.requests && adapter_of(by, s) == adapter) {
      low = max(begins(by, s), from);
      high = min(begins(by, s + 1), to);
    }
    found = __ballot(low < high);
    s0 += 64;
  };
  auto next = [&]() {
    row0 += 128;
    while (row0 >= last) {
      while (!found && s0 < by.requests) look();
      if (!found) break;
      const int at = __builtin_ctzll(found);
      found &= found - 1;
      first = __builtin_amdgcn_readlane(low, at);
      row0 = first / 32 * 32 + (wave - pieces) % 4 * 32;
      last = __builtin_amdgcn_readlane(high, at);
      ++pieces;
    }
  };

  next();
  while (row0 < last) {
    // of the step's rows, which are the request's
    const uint32_t low_in = first > row0 ? first - row0 : 0, rows = min(32u, last - row0);
    auto in_step = [&](uint32_t row) { return row >= low_in && row < rows; };
    Eight<T> wide[8];
    if (kKept) {
      const uint32_t pitch = a.groups * kGroup, left = pitch - tile * kOuterCols;
      const Window<int8_t, false> values((const int8_t*)a.wide + (uint64_t)row0 * pitch + tile * kOuterCols, (rows - 1) * pitch + left);
      const Window<uint8_t, false> exponents(a.exponents + (uint64_t)row0 * a.groups + tile * (kOuterCols / kGroup),
                                             (rows - 1) * a.groups + left / kGroup);
      uint2 q[8];
      uint32_t x[8];
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) {
        const bool in = count && in_step(k * 8 + e);
        typedef uint32_t Pair __attribute__((ext_vector_type(2)));
        const Pair pair = __builtin_amdgcn_raw_buffer_load_b64(values.buffer, in ? k * 8 * pitch + i * 8 : kNowhere, e * pitch, 0);
        q[e] = uint2{pair.x, pair.y};
        x[e] = __builtin_amdgcn_raw_buffer_load_b8(exponents.buffer, in ? k * 8 * a.groups + i / 4 : kNowhere, e * a.groups, 0);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) wide[e] = P::decoded(q[e], x[e]);
    } else {
      const uint32_t stride = (uint32_t)a.stride;
      const Window<T, kOdd> from((const T*)a.wide + row0 * a.stride + tile * kOuterCols, (rows - 1) * stride + a.cols - tile * kOuterCols);
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) wide[e] = from.read(e * stride, k * 8 * stride + i * 8, in_step(k * 8 + e) ? count : 0);
    }
    const uint32_t octet = by.rank * 8;
    const Window<float, false> narrow0(a.narrow + (uint64_t)(row0 / 8) * octet, 4 * octet);
    Eight<float> narrow[kRanks];
#pragma unroll
    for (uint32_t r = 0; r < kRanks; ++r)
      narrow[r] = narrow0.read((rank0 + r * 16) * 8, k * octet + i * 8, rank0 + r * 16 + i < by.rank ? 8 : 0);
    if (low_in || rows < 32) {
#pragma unroll
      for (uint32_t r = 0; r < kRanks; ++r)
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) narrow[r].v[e] = in_step(k * 8 + e) ? narrow[r].v[e] : 0.0f;
    }
    if constexpr (kRanks <= 2 || P::kParts == 1) {  // one column's operand at a time
      typename P::Fragment parts[kRanks][P::kParts];
#pragma unroll
      for (int r = 0; r < kRanks; ++r) P::split(parts[r], narrow[r].v);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const typename P::Fragment f = P::column(wide, q);
#pragma unroll
        for (int r = 0; r < kRanks; ++r)
#pragma unroll
          for (int p = 0; p < P::kParts; ++p) P::multiply(sum[r][q], parts[r][p], f);
      }
    } else {  // one narrow operand's parts at a time: those of all would not fit in registers
      typename P::Fragment columns[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) columns[q] = P::column(wide, q);
#pragma unroll
      for (int r = 0; r < kRanks; ++r) {
        typename P::Fragment parts[P::kParts];
        P::split(parts, narrow[r].v);
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
          for (int p = 0; p < P::kParts; ++p) P::multiply(sum[r][q], parts[p], columns[q]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    next();
  }
  const bool any = pieces != 0;
  if (!any && a.splits > 1) return;  // nothing reads this plane

  // waves 2 and 3 to 0 and 1, then 1 to 0; whole vectors, since the loop above would hold the sums once more where they
  // are taken apart
#pragma unroll
  for (uint32_t apart = 2; apart; apart /= 2) {
    f32x4* spot = room + (wave % apart) * kRanks * 8 * 64 + lane;
    __syncthreads();
    if (wave >= apart && wave < 2 * apart) {
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int q = 0; q < 8; ++q) spot[(r * 8 + q) * 64] = sum[r][q];
    }
    __syncthreads();
    if (wave < apart) {
#pragma unroll
      for (int r = 0; r < kRanks; ++r)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          sum[r][q] += spot[(r * 8 + q) * 64];
          if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // not all of them in registers at once
        }
    }
  }
  if (wave || !count) return;
  const bool alone = a.splits == 1;
  const float scale = alone && a.scaled ? scale_of(by, adapter) : 1.0f;
  const uint64_t size = (uint64_t)a.cols * by.rank;
  float* plane = a.planes + ((uint64_t)split * by.adapters + adapter) * size;
  T* out = (T*)a.to + adapter * size;
#pragma unroll
  for (int r = 0; r < kRanks; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t j = rank0 + r * 16 + k * 4 + e;
      __builtin_amdgcn_sched_barrier(0);
      if (j >= by.rank) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = sum[r][q][e] * scale;
      if (a.turned) {
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) {
          if (q >= count) continue;
          const uint64_t at = (uint64_t)(col + q) * by.rank + j;
          if (alone)
            out[at] = (T)v[q];
          else
            plane[at] = v[q];
        }
      } else {
        const uint64_t at = (uint64_t)j * a.cols + col;
        if (alone)
          store8<kOdd>(out + at, v, count);
        else
          store8<kOdd>(plane + at, v, count);
      }
    }
}

template <class T, int kRanks, bool kOdd>
__device__ __forceinline__ void outer_sides(const Outer& a) {
  __shared__ f32x4 room[2 * kRanks * 8 * 64];
  const bool second = blockIdx.x >= a.side[0].tiles;
  const Side& side = a.side[second];
  if (blockIdx.y >= side.splits) return;
  const uint32_t tile = blockIdx.x - (second ? a.side[0].tiles : 0);
  if (side.exponents)
    outer<T, kRanks, true, kOdd>(a.by, side, tile, room);
  else
    outer<T, kRanks, false, kOdd>(a.by, side, tile, room);
}

// The planes of a gradient's splits that have rows of the adapter, added up in order. Bound by the time to memory and back:
// 16 ranks of 19456 columns, three planes (3.7 MB) in 4.5 us; one plane asked for after the other took 5.9.
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
  const uint64_t all = active;
  uint64_t left = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(all >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)all);
  while (left) {  // eight planes asked for at a time
    float more[8][4];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) more[u][e] = 0.0f;
      if (!left) continue;
      const float* from = side.planes + ((uint64_t)__builtin_ctzll(left) * a.by.adapters + adapter) * size + at;
      left &= left - 1;
      if (n == 4)
        __builtin_memcpy(more[u], from, 16);
      else
#pragma unroll
        for (uint32_t e = 0; e < 3; ++e)
          if (e < n) more[u][e] = from[e];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += more[u][e];
  }
  const float scale = side.scaled ? scale_of(a.by, adapter) : 1.0f;
  T* to = (T*)side.to + adapter * size + at;
  for (uint32_t e = 0; e < n; ++e) to[e] = (T)(sum[e] * scale);
}

// A weight turned, 32 x 32 through LDS; behind the weights' tiles a narrow matrix, the sum of its splits. 4.7 us for 16 ranks of
// 19456 columns and 4608 rows, a launch's latency; it saves the products reads of 2 bytes from each of many lines.
template <class T>
__device__ __forceinline__ void turn(const Turn& a) {
  const uint32_t x = threadIdx.x % 32, y = threadIdx.x / 32;
  uint32_t tile = blockIdx.x;
  if (tile < a.tiles[0] + a.tiles[1]) {
    __shared__ T room[32][33];
    const bool second = tile >= a.tiles[0];
    tile -= second ? a.tiles[0] : 0;
    const uint32_t rows = a.rows[second], cols = a.cols[second];
    const uint32_t across = (cols + 31) / 32, row0 = tile / across * 32, col0 = tile % across * 32;
    for (uint32_t place = blockIdx.y; place < a.places; place += gridDim.y) {
      uint32_t adapter = place;
      if (a.by_request) {
        adapter = begins(a.by, place) < begins(a.by, place + 1) ? adapter_of(a.by, place) : kNone;
        if (adapter == kNone) continue;  // nothing reads its place
      }
      const uint64_t size = (uint64_t)rows * cols;
      const T* from = (const T*)a.from[second] + size * adapter;
      T* to = (T*)a.to[second] + size * place;
      __syncthreads();
      for (uint32_t r = y; r < 32; r += 8)
        if (row0 + r < rows && col0 + x < cols) room[r][x] = from[(uint64_t)(row0 + r) * cols + col0 + x];
      __syncthreads();
      for (uint32_t r = y; r < 32; r += 8)
        if (col0 + r < cols && row0 + x < rows) to[(uint64_t)(col0 + r) * rows + row0 + x] = room[x][r];
    }
    return;
  }
  if (blockIdx.y) return;
  __shared__ float room[32][33];
  tile -= a.tiles[0] + a.tiles[1];
  const uint32_t across = (a.rank + 31) / 32, row0 = tile / across * 32, col0 = tile % across * 32;
  for (uint32_t r = y; r < 32; r += 8) {
    if (row0 + r >= a.count || col0 + x >= a.rank) continue;
    const uint64_t at = (uint64_t)(row0 + r) * a.rank + col0 + x;
    float sum = a.narrow[at];
    for (uint32_t p = 1; p < a.splits; ++p) sum += a.narrow[(uint64_t)p * a.count * a.rank + at];
    room[r][x] = sum;
  }
  __syncthreads();
  for (uint32_t r = y; r < 32; r += 8)
    if (col0 + r < a.rank && row0 + x < a.count) a.turned[turned_at(a.rank, col0 + r, row0 + x)] = room[x][r];
}

// Names: type, ranks; "tall": tiles of 128 rows; "odd": features or a rank that are no multiples of eight, or addresses off the
// 4-byte grid.
// Waves a SIMD asked for where the compiler would take registers for one less: an expand of 16 ranks (4608 rows of 3072 bfloat16
// 21.0 us, 23.4 with three), an outer of 32 (three of its values go to scratch; 4608 rows of 8192 and 3072 27.1 us).
#define MO_SHRINK(T, t, ranks)                                                                                     \
  extern "C" __global__ __launch_bounds__(512) void mo_adapters_shrink_##t##_##ranks(Shrink a) {                   \
    shrink<T, ranks, false>(a);                                                                                    \
  }                                                                                                                \
  extern "C" __global__ __launch_bounds__(512) void mo_adapters_shrink_##t##_##ranks##_odd(Shrink a) {             \
    shrink<T, ranks, true>(a);                                                                                     \
  }
#define MO_TALL(T, t, ranks)                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void mo_adapters_shrink_##t##_##ranks##_tall(Shrink a) {            \
    shrink_tall<T, ranks>(a);                                                                                      \
  }
#define MO_EXPAND(T, t, rank)                                                                                      \
  extern "C" __global__ __launch_bounds__(256, rank == 16 && sizeof(T) == 2 ? 4 : 1)                     \
  void mo_adapters_expand_##t##_##rank(Expand a) {                                                                 \
    expand<T, rank, false>(a);                                                                                     \
  }                                                                                                                \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_expand_##t##_##rank##_odd(Expand a) {              \
    expand<T, rank, true>(a);                                                                                      \
  }
#define MO_EXPAND_TALL(T, t, rank)                                                                                 \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_expand_##t##_##rank##_tall(Expand a) {             \
    expand_tall<T, rank>(a);                                                                                       \
  }
#define MO_FEW(T, t, ranks)                                                                                        \
  extern "C" __global__ __launch_bounds__(512) void mo_adapters_few_##t##_##ranks(Few f) { few<T, ranks>(f); }
#define MO_OUTER(T, t, ranks)                                                                                      \
  extern "C" __global__ __launch_bounds__(256, ranks == 2 && sizeof(T) == 2 ? 3 : 2) void mo_adapters_outer_##t##_##ranks(Outer a) {                     \
    outer_sides<T, ranks, false>(a);                                                                               \
  }                                                                                                                \
  extern "C" __global__ __launch_bounds__(256, 2) void mo_adapters_outer_##t##_##ranks##_odd(Outer a) {               \
    outer_sides<T, ranks, true>(a);                                                                                \
  }
#define MO_ADAPTERS(T, t)                                                                                          \
  MO_SHRINK(T, t, 1)                                                                                               \
  MO_SHRINK(T, t, 2)                                                                                               \
  MO_SHRINK(T, t, 4)                                                                                               \
  MO_SHRINK(T, t, 8)                                                                                               \
  MO_TALL(T, t, 1)                                                                                                 \
  MO_TALL(T, t, 2)                                                                                                 \
  MO_TALL(T, t, 4)                                                                                                 \
  MO_EXPAND(T, t, 16)                                                                                              \
  MO_EXPAND(T, t, 32)                                                                                              \
  MO_EXPAND(T, t, 64)                                                                                              \
  MO_EXPAND(T, t, 128)                                                                                             \
  MO_EXPAND_TALL(T, t, 128)                                                                                        \
  MO_FEW(T, t, 1)                                                                                                  \
  MO_FEW(T, t, 2)                                                                                                  \
  MO_OUTER(T, t, 1)                                                                                                \
  MO_OUTER(T, t, 2)                                                                                                \
  MO_OUTER(T, t, 4)                                                                                                \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_join_##t(Outer a) { join<T>(a); }                  \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_turn_##t(Turn a) { turn<T>(a); }
MO_ADAPTERS(_Float16, f16)
MO_ADAPTERS(__bf16, bf16)
MO_ADAPTERS(float, f32)
MO_EXPAND_TALL(__bf16, bf16, 32)
MO_EXPAND_TALL(float, f32, 32)
MO_EXPAND_TALL(__bf16, bf16, 64)
MO_EXPAND_TALL(float, f32, 64)
MO_FEW(_Float16, f16, 4)
MO_FEW(__bf16, bf16, 4)
MO_TALL(_Float16, f16, 8)
MO_TALL(__bf16, bf16, 8)

}  // namespace
