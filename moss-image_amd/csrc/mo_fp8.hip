// 8-bit floating point with a scale for each 128 values, for gfx950: quantizing, reading back, and the
// products of block-scaled operands on the f8f6f4 matrix instructions.
//
//   stored value  q = e4m3(x / s), s = 2^e the smallest power of two, from 2^-126 on, with
//                 max |x| <= 448 s over the group; read back as q s (exact in fp32 and bf16)
//   groups        128 values along a row, 128 along a column, or a 128 x 128 block of a weight
//   product       C[m][n] = sum_k A[m][k] a(m, k / 128) B[n][k] b(n, k / 128) (+ bias[n]), fp32 sums
//
// A power of two as scale costs the quantizer at most one bit of range and nothing of precision, is
// found from the bits of the group's maximum (no logarithm, no division), and is what the scaled matrix
// instructions take: v_mfma_scale_f32_32x32x64_f8f6f4 multiplies each 32 values of an operand's row by
// 2^(byte - 127) on the way in (the E8M0 form), so a scaled product takes no more instructions than an
// unscaled one. Weights whose block scales are arbitrary fp32 numbers are multiplied in as fp32 for each
// 128 of the reduction.
//
// What the matrix instructions on e4m3 add is not exact to fp32: of neighbouring products inside one
// instruction, bits under about 2^-15 of the largest are dropped (measured: 65536 + 1 gives 65536, and
// Gaussian operands come out 1.5e-5 off, in the scaled, the unscaled and the 16-deep form alike). There, that
// is a hundredth of a bf16 rounding and a tenth of an fp16 one, and stays for 16-bit outputs; where products of
// a strong channel cancel, what is lost is relative to them and can be more than the output's own rounding. An
// fp32 output is asked for its fp32 sums: those kernels decode the operands to bf16, exact for values from
// 2^-126 on, and use the bf16 instructions (half the rate, 6e-8 off).
//
// A group with an infinity or a NaN gets the scale byte 255, which reads back as NaN throughout and
// makes NaN of every output that it takes part in.
//
// MFMA 32x32x64 lane layout (checked on the device): lane l holds 32 bytes of row l % 32 of either
// operand, reduction indices 32 * (l / 32) + j, and that slice's scale byte; D register r of lane l is
// row 8 * (r / 4) + 4 * (l / 32) + r % 4 of the first operand, row l % 32 of the second. The order of
// the reduction inside a group is free as long as both operands agree. The weights are the first
// operand here, so a lane holds runs of four neighbouring output features of one token.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "mo_fp8.h"

namespace {

using mo_fp8::ProductArgs;
using mo_fp8::kBF16;
using mo_fp8::kF32;
using mo_fp8::kGroup;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---- element types -------------------------------------------------------------------------------

template <class T>
struct Bits {};  // eight values of T as loaded: 16 or 32 bytes

template <>
struct Bits<__bf16> {
  u32x4 w;
  __device__ __forceinline__ void load(const void* p) { w = *(const u32x4*)p; }
  __device__ __forceinline__ void zero() { w = u32x4{}; }
  __device__ __forceinline__ float get(int i) const {
    return __builtin_bit_cast(float, i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
};

template <>
struct Bits<_Float16> {
  u32x4 w;
  __device__ __forceinline__ void load(const void* p) { w = *(const u32x4*)p; }
  __device__ __forceinline__ void zero() { w = u32x4{}; }
  __device__ __forceinline__ float get(int i) const {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]));
  }
};

template <>
struct Bits<float> {
  f32x4 lo, hi;
  __device__ __forceinline__ void load(const void* p) {
    lo = ((const f32x4*)p)[0];
    hi = ((const f32x4*)p)[1];
  }
  __device__ __forceinline__ void zero() { lo = hi = f32x4{}; }
  __device__ __forceinline__ float get(int i) const { return i < 4 ? lo[i & 3] : hi[i & 3]; }
};

__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// The scale byte of a group from the bits of its largest magnitude m (IEEE order is integer order, and
// an infinity or a NaN is above every number): 448 = 1.75 * 2^8, so 2^(exponent(m) - 8) holds m when
// its fraction is at most 1.75, and twice that otherwise.
__device__ __forceinline__ uint32_t scale_byte(uint32_t m) {
  if (m >= 0x7f800000u) return 255u;
  const int e = (int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(e < 1 ? 1 : e);
}

// 1 / scale as a factor: exact, and the product with it is exact unless it falls under 2^-126, where e4m3
// is zero anyway. NaN for the byte 255.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 255u ? 0x7fc00000u : (254u - byte) << 23);
}

__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __builtin_bit_cast(float, byte == 255u ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u);
}

// Four floats to four e4m3 bytes, to nearest with ties to even (the hardware conversion; its inputs are
// within 448 here, so nothing saturates).
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return (uint32_t)r;
}

// Maximum over the 16 lanes of a DPP row.
template <int kRor>
__device__ __forceinline__ uint32_t ror16(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 | kRor, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, ror16<8>(v));
  v = max(v, ror16<4>(v));
  v = max(v, ror16<2>(v));
  return max(v, ror16<1>(v));
}

// ---- quantizing -----------------------------------------------------------------------------------
//
// A workgroup takes a tile of 128 x 128 values, once, into registers: thread (g, c) holds rows 8 g to
// 8 g + 7 of columns 8 c to 8 c + 7 (kPer = 8; with kPer = 1, for few rows, one row, 16 a workgroup: eight times
// the workgroups, 333 x 3072 in 3.5 us instead of 5.7). A row's 16 threads are one DPP row, so its maximum takes four DPP
// steps; a column's maximum is taken over the thread's own rows, the four row groups of its wave, and
// the waves through LDS. Bound by memory: 17792 x 12288 bf16 both ways in 162 us (5.4 TB/s read and written), rows
// alone 119 (5.5), columns alone 123. The columns' bytes are turned in LDS and leave as whole 128-byte lines.

enum { kRows = 1, kColumns = 2, kBlock = 4 };

template <class T, int kForm, int kPer>
__device__ __forceinline__ void quantize_tile(const T* __restrict__ x, uint64_t rows, uint32_t cols, uint64_t stride,
                                              uint8_t* __restrict__ row_values, uint8_t* __restrict__ row_scales,
                                              uint8_t* __restrict__ col_values, uint8_t* __restrict__ col_scales) {
  constexpr int kLine = kGroup + 16;  // bytes between a turned column and the next
  __shared__ uint32_t part[4][kGroup];
  __shared__ __attribute__((aligned(16))) uint8_t turned[kForm & kColumns ? kGroup * kLine : 16];
  const uint32_t tiles_c = (cols + kGroup - 1) / kGroup;
  const uint64_t tile_r = blockIdx.x / tiles_c;
  const uint32_t tile_c = blockIdx.x % tiles_c;
  const int tid = threadIdx.x, c = tid & 15, g = tid >> 4, wave = tid >> 6;
  const uint64_t row0 = tile_r * 16 * kPer + kPer * g;
  const uint32_t col0 = tile_c * kGroup + 8 * c;
  const bool in_cols = col0 < cols;  // cols is a multiple of 16: a thread's eight are in or out

  static_assert(kPer == 8 || kForm == kRows, "groups down the columns take whole tiles");
  Bits<T> v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (in_cols && row0 + i < rows)
      v[i].load(x + (row0 + i) * stride + col0);
    else
      v[i].zero();
  }

  if (kForm & kRows) {
    const uint64_t pitch = (rows + 15) & ~(uint64_t)15;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i].get(j)));
      const uint32_t byte = scale_byte(max16(m));
      const float inv = inverse_scale(byte);
      if (row0 + i < rows) {
        if (in_cols) {
          u32x2 w;
          w[0] = pack4(v[i].get(0) * inv, v[i].get(1) * inv, v[i].get(2) * inv, v[i].get(3) * inv);
          w[1] = pack4(v[i].get(4) * inv, v[i].get(5) * inv, v[i].get(6) * inv, v[i].get(7) * inv);
          *(u32x2*)(row_values + (row0 + i) * cols + col0) = w;
        }
        if (c == 0) row_scales[tile_c * pitch + row0 + i] = (uint8_t)byte;
      }
    }
  }

  if constexpr ((kForm & (kColumns | kBlock)) != 0) {
    uint32_t m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m[j] = max(m[j], abs_bits(v[i].get(j)));
      m[j] = max(m[j], (uint32_t)__shfl_xor((int)m[j], 16));
      m[j] = max(m[j], (uint32_t)__shfl_xor((int)m[j], 32));
    }
    if ((tid & 48) == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) part[wave][8 * c + j] = m[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      m[j] = max(max(part[0][8 * c + j], part[1][8 * c + j]), max(part[2][8 * c + j], part[3][8 * c + j]));
    if (kForm & kBlock) {
      uint32_t all = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) all = max(all, m[j]);
      const uint32_t byte = scale_byte(max16(all));
      const float inv = inverse_scale(byte);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!in_cols || row0 + i >= rows) continue;
        u32x2 w;
        w[0] = pack4(v[i].get(0) * inv, v[i].get(1) * inv, v[i].get(2) * inv, v[i].get(3) * inv);
        w[1] = pack4(v[i].get(4) * inv, v[i].get(5) * inv, v[i].get(6) * inv, v[i].get(7) * inv);
        *(u32x2*)(row_values + (row0 + i) * cols + col0) = w;
      }
      if (tid == 0) row_scales[tile_r * tiles_c + tile_c] = (uint8_t)byte;
    } else {
      const uint64_t pitch = (rows + kGroup - 1) / kGroup * kGroup;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t byte = scale_byte(m[j]);
        const float inv = inverse_scale(byte);
        u32x2 w;
        w[0] = pack4(v[0].get(j) * inv, v[1].get(j) * inv, v[2].get(j) * inv, v[3].get(j) * inv);
        w[1] = pack4(v[4].get(j) * inv, v[5].get(j) * inv, v[6].get(j) * inv, v[7].get(j) * inv);
        *(u32x2*)(turned + (8 * c + j) * kLine + 8 * g) = w;
        if (g == 0 && in_cols) col_scales[tile_r * cols + col0 + j] = (uint8_t)byte;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = (tid >> 3) + 32 * i, piece = tid & 7;
        if (tile_c * kGroup + col < cols)
          *(u32x4*)(col_values + (uint64_t)(tile_c * kGroup + col) * pitch + tile_r * kGroup + 16 * piece) =
              *(const u32x4*)(turned + col * kLine + 16 * piece);
      }
    }
  }
}

#define MO_QUANTIZE(name, T, form, per)                                                                            \
  extern "C" __global__ __launch_bounds__(256) void mo_fp8_quantize_##name(                                   \
      const T* x, uint64_t rows, uint32_t cols, uint64_t stride, uint8_t* row_values, uint8_t* row_scales,    \
      uint8_t* col_values, uint8_t* col_scales) {                                                             \
    quantize_tile<T, form, per>(x, rows, cols, stride, row_values, row_scales, col_values, col_scales);            \
  }
#define MO_QUANTIZE_FORMS(t, T)                     \
  MO_QUANTIZE(rows_##t, T, kRows, 8)                \
  MO_QUANTIZE(few_##t, T, kRows, 1)                 \
  MO_QUANTIZE(columns_##t, T, kColumns, 8)          \
  MO_QUANTIZE(both_##t, T, kRows | kColumns, 8)     \
  MO_QUANTIZE(weight_##t, T, kBlock, 8)
MO_QUANTIZE_FORMS(f16, _Float16)
MO_QUANTIZE_FORMS(bf16, __bf16)
MO_QUANTIZE_FORMS(f32, float)

// ---- reading back ---------------------------------------------------------------------------------

// Four outputs to memory in the type of `kind`; `n` of them exist.
__device__ __forceinline__ void store4(void* base, uint64_t at, f32x4 v, uint32_t kind) {
  if (kind == kF32) {
    *(f32x4*)((float*)base + at) = v;
  } else if (kind == kBF16) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    bf16x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (__bf16)v[i];
    *(bf16x4*)((__bf16*)base + at) = o;
  } else {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    f16x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (_Float16)v[i];
    *(f16x4*)((_Float16*)base + at) = o;
  }
}

__device__ __forceinline__ float load1(const void* base, uint64_t at, uint32_t kind) {
  return kind == kF32 ? ((const float*)base)[at] : kind == kBF16 ? (float)((const __bf16*)base)[at]
                                                                 : (float)((const _Float16*)base)[at];
}

// One lane reads eight values and their scale and writes eight products, 16 bytes (or twice that) in a row with
// its neighbours': bound by memory, 17792 x 12288 to bf16 in 115 us (5.7 TB/s). d: chunks of eight in a row, and its divisor while all chunks are under
// 2^31 (m 0: a 64-bit division). Output rows that are not whole chunks go out value by value.
extern "C" __global__ __launch_bounds__(256) void mo_fp8_decode_kernel(
    const uint8_t* __restrict__ values, uint64_t pitch, const void* __restrict__ scales, uint32_t f32_scales,
    uint64_t scale_row, uint64_t scale_col, uint32_t shift, void* __restrict__ out, uint32_t kind, uint64_t rows,
    uint32_t cols, mo_fp8::Divisor chunks) {
  const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t row = chunks.m ? (__umulhi(chunks.m, (uint32_t)at) + (uint32_t)at) >> chunks.s : at / chunks.d;
  const uint32_t col = (uint32_t)(at - row * chunks.d) * 8;
  if (row >= rows) return;
  const u32x2 w = *(const u32x2*)(values + row * pitch + col);
  const uint64_t s = (row >> shift) * scale_row + col / kGroup * scale_col;
  const float scale = f32_scales ? ((const float*)scales)[s] : scale_value(((const uint8_t*)scales)[s]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    v[4 * i] = lo[0] * scale, v[4 * i + 1] = lo[1] * scale, v[4 * i + 2] = hi[0] * scale, v[4 * i + 3] = hi[1] * scale;
  }
  const uint64_t to = row * cols + col;
  if (cols % 8) {
    for (uint32_t j = 0; j < 8 && col + j < cols; ++j) {
      if (kind == kF32)
        ((float*)out)[to + j] = v[j];
      else if (kind == kBF16)
        ((__bf16*)out)[to + j] = (__bf16)v[j];
      else
        ((_Float16*)out)[to + j] = (_Float16)v[j];
    }
  } else if (kind == kF32) {
    *(f32x4*)((float*)out + to) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)((float*)out + to + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else if (kind == kBF16) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (__bf16)v[j];
    *(bf16x8*)((__bf16*)out + to) = o;
  } else {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    f16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (_Float16)v[j];
    *(f16x8*)((_Float16*)out + to) = o;
  }
}

// ---- products -------------------------------------------------------------------------------------

// ---- tiles in LDS ----
//
// A workgroup owns a tile of kBM tokens x kBN features, shared out over WM x WN waves of TM x TN MFMA tiles
// of 32 x 32 (the weights are the first MFMA operand). The reduction advances a group of 128 a step: kBM +
// kBN rows of 128 bytes, one cache line each (half lines come at half the rate), go straight from memory
// into LDS by the buffer-load DMA path, with no register on the way, into one of two buffers; the rows'
// scale bytes go with them. A step is two halves of 64. While a half's MFMAs run, the other half's
// fragments are read into the registers as those come free. After the first half every wave has read all it
// wants of this step's buffer and the next step's DMA has landed (it had a whole step to): the one barrier
// of a step sits there, and the second half refills the buffer with the step after next.
//   LDS rows of 128 bytes keep 16-byte piece c of row r at c ^ (r / 2 % 8): 16 lanes of a read then fall on
//   the 64 banks without a conflict (rows of one parity share a half of the banks), and a DMA instruction
//   still fills eight whole rows.
// The scales lie group by group, a byte a row, so that a step's are one dense piece. What lies past the rows
// or the reduction reads as zero.
//
// An input gradient reads the weight as it is stored, [reduction][features]: kTrans keeps 128 rows of kBN
// features in LDS and reads fragments with ds_read_b64_tr_b8, which hands each lane of 16 eight bytes of one
// column (16 lanes transpose 8 rows x 16 bytes). The rows' 32-byte units are XOR-swizzled by row, so that the
// 8 rows of a read lie on distinct banks.
//
// fp32 block scales (kBlockFloats): a wave's features lie in one block, so a step has one scale s = f 2^e, f
// in [1, 2). The instructions take 2^e; the accumulators are held in units of f, multiplied by f(before) /
// f(now) before a step's first products and by f once at the end. That keeps every factor between 1/2 and 2,
// needs no second set of accumulators, and its multiplications run in the shadow of the MFMAs. Scales under
// 2^-126 count as zero, an infinite one as NaN.
//
// kWide (fp32 outputs): operands decoded to bf16 in registers, the power-of-two scales with them.
// Large tile, 8192 x 8192 from 8192: 418 to 425 us, 2.6 PFLOP/s; the instructions alone reach 3.84 on such bytes,
// held to 1.9 GHz by power, and are busy 66 % of the cycles here. Eight waves of 128 x 64 with the scales group by
// group: 404 us at best, four waves of 128 x 128 without 490. fp32 scales: 16384 rows of 3072 from 12288 604 us.
// Tiles are numbered in groups of kGroupM row tiles and then by XCD, so that the workgroups of one XCD
// (blockIdx % 8) share rows and columns in its L2 (groups of 4, 8, 16 row tiles: 4608 rows of 24576 from 3072
// 318, 325, 346 us; the other large calls differ by 1 %).

#define MO_LDS __attribute__((address_space(3)))
typedef __amdgpu_buffer_rsrc_t rsrc_t;

// Raw buffer descriptors (gfx9 word 3 = 0x00020000): a read whose vector and scalar offsets add up to
// num_records or more returns zero and moves no data (into LDS, the zero is written), a write there is
// dropped. The scalar offset must not pass num_records itself: the check subtracts it.
constexpr uint32_t kOob = 0x80000000u;
__device__ __forceinline__ rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)bytes, 0x00020000);
}
// s_waitcnt immediate (gfx9): at most n vector-memory operations outstanding, and all LDS operations done.
constexpr int wait_vm(int n) { return (n & 0xF) | ((n >> 4) << 14) | (0x7 << 4); }

constexpr int kGroupM = 4, kXcds = 8;

template <int WM, int WN, int TM, int TN>
struct Tile {
  static constexpr int kWM = WM, kTM = TM, kTN = TN, kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kBM = 32 * WM * TM, kBN = 32 * WN * TN;
  static constexpr int kDmaA = kBM / 8 / kWaves, kDmaB = kBN / 8 / kWaves;  // 1 KiB pieces a wave and step
  static_assert(kBM % (16 * kWaves) == 0 && kBN % (16 * kWaves) == 0, "pairs of DMA pieces divide over the waves");
  static_assert(kBM <= 256 && kBN <= 256 && kWaves >= 2, "one DMA instruction brings an operand's scales");
};

// How B's scales come: a byte or an fp32 number a block of 128 x 128, or a byte a row.
enum { kBlockBytes = 0, kRowBytes = 1, kBlockFloats = 2 };

// Eight e4m3 bytes times a power of two as bf16: exact (four significant bits), or rounded towards zero
// under 2^-126.
__device__ __forceinline__ bf16x8 widen(int lo, int hi, float power) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// acc (+)= the products of one fragment pair (64 of the reduction), under the scale bytes sb and sa.
template <bool kWide>
__device__ __forceinline__ f32x16 products(i32x8 fb, i32x8 fa, f32x16 acc, int sb, int sa) {
  if (!kWide) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb, fa, acc, 0, 0, 0, sb, 0, sa);
  const float pb = __builtin_bit_cast(float, sb << 23), pa = __builtin_bit_cast(float, sa << 23);
#pragma unroll
  for (int q = 0; q < 4; ++q)
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(fb[2 * q], fb[2 * q + 1], pb), widen(fa[2 * q], fa[2 * q + 1], pa),
                                                  acc, 0, 0, 0);
  return acc;
}

template <class G, int kScales, bool kWide, bool kTrans>
__device__ __forceinline__ void product_tile(const ProductArgs& p) {
  constexpr int kBM = G::kBM, kBN = G::kBN, kTM = G::kTM, kTN = G::kTN, kDmaA = G::kDmaA, kDmaB = G::kDmaB;
  // distinct objects, chosen at compile time: the compiler then knows which reads a DMA in flight can reach
  __shared__ __attribute__((aligned(1024))) uint8_t a_0[kBM * kGroup], a_1[kBM * kGroup];
  __shared__ __attribute__((aligned(1024))) uint8_t b_0[kBN * kGroup], b_1[kBN * kGroup];
  __shared__ __attribute__((aligned(256))) uint8_t sa_0[256], sa_1[256], sb_0[256], sb_1[256], nowhere[256];
  typedef MO_LDS uint8_t* lp;
  struct Buffer {
    lp a, b, sa, sb;
  };
  const Buffer buf0 = {(lp)a_0, (lp)b_0, (lp)sa_0, (lp)sb_0}, buf1 = {(lp)a_1, (lp)b_1, (lp)sa_1, (lp)sb_1};

  const int lane = threadIdx.x & 63, lr = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % G::kWM, wn = wave / G::kWM;

  const int items = gridDim.x, tiles = items / p.splits;
  const int tiles_m = (int)((p.m + kBM - 1) / kBM), tiles_n = tiles / tiles_m;
  int t;
  {
    const int b = blockIdx.x, xcd = b % kXcds, idx = b / kXcds;
    const int per = items / kXcds, rem = items % kXcds;
    t = xcd < rem ? xcd * (per + 1) + idx : rem * (per + 1) + (xcd - rem) * per + idx;
  }
  const int split = t / tiles;
  t -= split * tiles;
  const uint32_t k_begin = split * p.split_steps * kGroup, k_end = min(p.r, k_begin + p.split_steps * kGroup);
  const int group_tiles = kGroupM * tiles_n, first_m = t / group_tiles * kGroupM;
  const int gm = min(tiles_m - first_m, kGroupM), in_group = t % group_tiles;
  const uint64_t m0 = (uint64_t)(first_m + in_group % gm) * kBM;
  const uint32_t n0 = (uint32_t)(in_group / gm) * kBN;

  const uint32_t rows_m = (uint32_t)min((uint64_t)kBM, p.m - m0), rows_n = min((uint32_t)kBN, p.n - n0);
  const rsrc_t ra = make_rsrc(p.a + m0 * p.a_pitch, (uint32_t)(rows_m * p.a_pitch));
  const rsrc_t rb = kTrans ? make_rsrc(p.b + n0, (uint32_t)(p.r * p.b_pitch - n0))
                           : make_rsrc(p.b + (uint64_t)n0 * p.b_pitch, (uint32_t)(rows_n * p.b_pitch));
  const uint8_t* b_scales = (const uint8_t*)p.b_scales;

  // DMA: piece j of wave w is rows 8 (w kDma + j) .. + 7; lane i fills position i % 8 of row i / 8. The
  // swizzle goes by row / 2 % 8, of which bit 2 is the piece's parity. The pieces' offsets are sums made
  // when they are wanted.
  const uint32_t dma_row = lane >> 3;
  uint32_t dma_k[2], a_off[2], b_off[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    dma_k[e] = 16 * ((lane & 7) ^ (4 * e + dma_row / 2));
    a_off[e] = (uint32_t)((wave * kDmaA * 8 + dma_row) * p.a_pitch + dma_k[e]);
    b_off[e] = (uint32_t)((wave * kDmaB * 8 + dma_row) * p.b_pitch + dma_k[e]);
  }
  // kTrans: piece j of wave w is 1024 / kBN rows of the reduction; unit(row): the row's swizzle
  auto unit = [](int row) { return kBN >= 256 ? row & 7 : kBN == 128 ? (row >> 1) & 3 : (row >> 2) & 1; };
  uint32_t t_off[kDmaB];
#pragma unroll
  for (int j = 0; j < kDmaB; ++j) {
    const int place = (wave * kDmaB + j) * 64 + lane, row = place / (kBN / 16);
    const int chunk = (place % (kBN / 16)) ^ (unit(row) << 1);
    t_off[j] = n0 + 16 * chunk < p.n ? (uint32_t)(row * p.b_pitch + 16 * chunk) : kOob;
  }
  const uint32_t last_group = (k_end - 1) / kGroup;
  const bool scales_of_a = wave == 0, scales_of_b = kScales == kRowBytes && wave == 1;
  auto dma = [&](const Buffer& to, uint32_t k) {
    const uint32_t group = min(k / kGroup, last_group);
    // a group's scales of the tile's rows (a word that begins within the rows is within the pitch)
    const rsrc_t rsa = make_rsrc(p.a_scales + (uint64_t)group * p.a_scale_pitch + m0, (rows_m + 3) & ~3u);
    const rsrc_t rsb = make_rsrc(b_scales + (uint64_t)group * p.b_scale_col + n0, (rows_n + 3) & ~3u);
    const int at_k = k < k_end ? (int)k : 0;
    // steps come in turn: from the one that the reduction ends in on, the pieces past its end read as zero
    // (an offset from kOob on stays past every descriptor: a tile's rows take less than 2^31 bytes)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool in = k + dma_k[e] < k_end;
      a_off[e] = in ? a_off[e] : kOob;
      b_off[e] = in ? b_off[e] : kOob;
    }
    // every wave issues the scales' pieces (a branch would cut the loop up), all but one of them zeros to nowhere
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (MO_LDS void*)(scales_of_a ? to.sa : (lp)nowhere), 4, scales_of_a ? 4 * lane : kOob, 0,
                                             0, 0);
    if (kScales == kRowBytes)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, (MO_LDS void*)(scales_of_b ? to.sb : (lp)nowhere), 4, scales_of_b ? 4 * lane : kOob, 0,
                                               0, 0);
#pragma unroll
    for (int j = 0; j < kDmaA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (MO_LDS void*)(to.a + (wave * kDmaA + j) * 1024), 16,
                                               a_off[j & 1] + 8 * j * (uint32_t)p.a_pitch, at_k, 0, 0);
#pragma unroll
    for (int j = 0; j < kDmaB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (MO_LDS void*)(to.b + (wave * kDmaB + j) * 1024), 16,
          kTrans ? (k < k_end ? t_off[j] : kOob)
                 : b_off[j & 1] + 8 * j * (uint32_t)p.b_pitch,
          kTrans ? at_k * (int)p.b_pitch : at_k, 0, 0);
  };

  f32x16 acc[kTN][kTM];
#pragma unroll
  for (int j = 0; j < kTN; ++j)
#pragma unroll
    for (int i = 0; i < kTM; ++i) acc[j][i] = f32x16{};

  // A block's scale byte is the same for all lanes, one a step: loaded two steps ahead.
  const uint32_t n_wave = n0 + 32 * wn * kTN;
  const uint32_t block_at = n_wave < p.n ? (n_wave >> 7) * p.b_scale_row : 0;
  auto load_block = [&](uint32_t k) {
    const uint64_t at = block_at + (uint64_t)min(k / kGroup, last_group) * p.b_scale_col;
    return kScales == kBlockFloats ? ((const int*)p.b_scales)[at] : (int)b_scales[at];
  };

  // a lane's 32 bytes of a half h are pieces 4 h + 2 half and the next of its row
  i32x8 fa[kTM], fb[2][kTN];
  int sa[2][kTM], sb[2][kTN];
  int at[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) at[h][e] = lr * (int)kGroup + 16 * ((4 * h + 2 * half + e) ^ (lr / 2 & 7));
  auto fragment = [&](const MO_LDS uint8_t* base, int h) {
    const u32x4 lo = *(const MO_LDS u32x4*)(base + at[h][0]), hi = *(const MO_LDS u32x4*)(base + at[h][1]);
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  auto read_a = [&](const Buffer& from, int i, int h) { fa[i] = fragment(from.a + (wm * kTM + i) * 32 * kGroup, h); };
  const int t_row = 32 * half + ((lane & 15) >> 1);
  auto read_b = [&](const Buffer& from, int h) {
#pragma unroll
    for (int j = 0; j < kTN; ++j) {
      if (kTrans) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = t_row + 8 * q, byte = 32 * (wn * kTN + j) + 16 * ((lane >> 4) & 1) + 8 * (lane & 1);
          const i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (MO_LDS i32x2*)(from.b + 64 * h * kBN + row * kBN + (byte ^ (unit(row) << 5))));
          fb[h][j][2 * q] = v[0], fb[h][j][2 * q + 1] = v[1];
        }
      } else {
        fb[h][j] = fragment(from.b + (wn * kTN + j) * 32 * kGroup, h);
      }
    }
  };
  auto read_scales = [&](const Buffer& from, int parity) {
#pragma unroll
    for (int i = 0; i < kTM; ++i) sa[parity][i] = from.sa[32 * (wm * kTM + i) + lr];
    if (kScales == kRowBytes) {
#pragma unroll
      for (int j = 0; j < kTN; ++j) sb[parity][j] = from.sb[32 * (wn * kTN + j) + lr];
    }
  };
  // kBlockFloats: the byte of the step's scale, and the accumulators' unit and its change
  int block_byte = 0, a_keep = 0xff;
  float in_units = 1.0f, change = 1.0f, poison = 0.0f;
  auto begin = [&](int parity) {
    if (kScales == kRowBytes) return;
    block_byte = sb[parity][0];
    if (kScales == kBlockFloats) {
      const int bits = sb[parity][0];
      block_byte = bits >> 23 & 0xff;
      a_keep = block_byte ? 0xff : 0;  // nothing: 2^-254 of the products
      const float f = block_byte ? __builtin_bit_cast(float, (bits & 0x807fffff) | 0x3f800000) : in_units;
      change = in_units / f;
      in_units = f;
    }
    if (kWide) poison = block_byte == 255 ? __builtin_nanf("") : poison;
  };
  // the MFMAs of half h, and behind each row of them the fragments of the half after
  auto multiply = [&](int h, int parity, const Buffer& then) {
    constexpr int kMfma = 0x008, kDsRead = 0x100;
    if (h == 0) begin(parity);
    read_b(then, h ^ 1);
    if (h == 1) read_scales(then, parity ^ 1);
#pragma unroll
    for (int i = 0; i < kTM; ++i) {
#pragma unroll
      for (int j = 0; j < kTN; ++j)
      {
        if (kScales == kBlockFloats && h == 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[j][i][e] *= change;
        }
        acc[j][i] = products<kWide>(fb[h][j], fa[i], acc[j][i], kScales == kRowBytes ? sb[parity][j] : block_byte,
                                    kScales == kBlockFloats ? sa[parity][i] & a_keep : sa[parity][i]);
      }
      read_a(then, i, h ^ 1);
    }
    if (!kWide && kScales != kBlockFloats) {
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kDsRead, (kTrans ? 4 : 2) * kTN, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, kTN - 1, 0);
#pragma unroll
      for (int i = 0; i < kTM; ++i) {
        __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kMfma, kTN, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto step = [&](int parity, const Buffer& now, const Buffer& next, uint32_t k) {
    multiply(0, parity, now);
    __builtin_amdgcn_s_waitcnt(wait_vm(0));
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    int after = 0;
    if (kScales != kRowBytes) after = load_block(k + 2 * kGroup);
    dma(now, k + 2 * kGroup);
    __builtin_amdgcn_s_setprio(1);  // past the barrier, a wave with its DMA issued goes before the other (1 to 6 %)
    multiply(1, parity, next);
    __builtin_amdgcn_s_setprio(0);
    if (kScales != kRowBytes) sb[parity][0] = after;
  };

  if (kScales != kRowBytes) sb[0][0] = load_block(k_begin), sb[1][0] = load_block(k_begin + kGroup);
  dma(buf0, k_begin);
  dma(buf1, k_begin + kGroup);
  __builtin_amdgcn_s_waitcnt(wait_vm(kDmaA + kDmaB + 1 + (kScales == kRowBytes ? 1 : 0)));
  __syncthreads();
  read_scales(buf0, 0);
  read_b(buf0, 0);
#pragma unroll
  for (int i = 0; i < kTM; ++i) read_a(buf0, i, 0);
  // steps in pairs, one a buffer; an odd count gets one more over zeros
  for (uint32_t k = k_begin; k < k_end; k += 2 * kGroup) {
    step(0, buf0, buf1, k);
    step(1, buf1, buf0, k + kGroup);
  }

  // Epilogue: 32 tokens by up to 128 bytes of features at a time through a part of LDS of the wave's own, so
  // that a store writes whole lines instead of pieces of 32 rows. 16-byte piece c of row r at c ^ (r % kPieces):
  // writes and reads spread over the banks.
  __builtin_amdgcn_s_waitcnt(wait_vm(0));
  __syncthreads();  // every wave has read its last fragments, every DMA has landed
  auto emit = [&](auto value_bytes, void* out, bool last) {
    constexpr int kBytes = decltype(value_bytes)::value;
    constexpr int kAcross = kBytes == 4 ? 1 : kTN < 2 ? kTN : 2;  // MFMA tiles of a line
    constexpr int kLine = 32 * kAcross * kBytes, kPieces = kLine / 16, kRowsAStore = 64 / kPieces;
    constexpr int kOwn = 32 * kLine, kValues = 16 / kBytes;
    static_assert(kOwn * G::kWaves <= (kBM + kBN) * (int)kGroup && kBM * kGroup % kOwn == 0, "a wave's part of a buffer");
    const int in_a = kBM * kGroup / kOwn;
    lp own = wave < in_a ? (lp)a_0 + wave * kOwn : (lp)b_0 + (wave - in_a) * kOwn;
    const int out_row = lane / kPieces, piece = lane % kPieces;
    const bool f16 = p.out_kind != kBF16;
    const rsrc_t ro = make_rsrc((uint8_t*)out + m0 * p.n * kBytes, (uint32_t)(rows_m * p.n * kBytes));
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j0 = 0; j0 < kTN; j0 += kAcross) {
        const uint32_t n_line = n_wave + 32 * j0;
#pragma unroll
        for (int j = 0; j < kAcross; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x16& w16 = acc[j0 + j][i];
            f32x4 o = {w16[4 * q], w16[4 * q + 1], w16[4 * q + 2], w16[4 * q + 3]};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (kScales == kBlockFloats) o[e] *= in_units;
              if (kWide && kScales != kRowBytes) o[e] += poison;
            }
            if (last && p.bias) {
              const uint32_t n = n_line + 32 * j + 8 * q + 4 * half;
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] += n < p.n ? load1(p.bias, n + e, p.bias_kind) : 0.0f;
            }
            if (kBytes == 4) {
              *(MO_LDS f32x4*)(own + lr * kLine + 16 * ((2 * q + half) ^ (lr % kPieces))) = o;
            } else {
              u32x2 w;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
                typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
                w[e] = f16 ? __builtin_bit_cast(uint32_t, f16x2{(_Float16)o[2 * e], (_Float16)o[2 * e + 1]})
                           : __builtin_bit_cast(uint32_t, bf16x2{(__bf16)o[2 * e], (__bf16)o[2 * e + 1]});
              }
              *(MO_LDS u32x2*)(own + lr * kLine + 16 * ((4 * j + q) ^ (lr % kPieces)) + 8 * half) = w;
            }
          }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 32; r += kRowsAStore) {
          const int row = r + out_row;
          const u32x4 w = *(const MO_LDS u32x4*)(own + row * kLine + 16 * (piece ^ (row % kPieces)));
          const uint32_t n = n_line + kValues * piece;
          const uint32_t to = ((uint32_t)(32 * (wm * kTM + i) + row) * p.n + n) * kBytes;
          __builtin_amdgcn_raw_buffer_store_b128(w, ro, (int)(n < p.n ? to : kOob), 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_wave_barrier();
      }
  };
  if (p.splits > 1)
    emit(std::integral_constant<int, 4>{}, p.planes + (uint64_t)split * p.m * p.n, false);
  else
    emit(std::integral_constant<int, kWide ? 4 : 2>{}, p.out, true);
}

// The sum of a call's planes, in the order of the reduction, + bias: four outputs a lane.
extern "C" __global__ __launch_bounds__(256) void mo_fp8_plane_sum(ProductArgs p) {
  const uint64_t count = p.m * p.n, at = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= count) return;  // a multiple of 16
  f32x4 v = *(const f32x4*)(p.planes + at);
  for (uint32_t s = 1; s < p.splits; ++s) v += *(const f32x4*)(p.planes + s * count + at);
  if (p.bias) {
    const uint32_t n = (uint32_t)(at % p.n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += load1(p.bias, n + e, p.bias_kind);
  }
  store4(p.out, at, v, p.out_kind);
}

#define MO_TILE_KERNEL(name, G, scales, wide, trans)                                                        \
  extern "C" __global__ __launch_bounds__(G::kThreads) void mo_fp8_product_##name(ProductArgs p) {          \
    product_tile<G, scales, wide, trans>(p);                                                                \
  }
#define MO_TILE(name, G)                                            \
  MO_TILE_KERNEL(name##_bytes, G, kBlockBytes, false, false)        \
  MO_TILE_KERNEL(name##_floats, G, kBlockFloats, false, false)      \
  MO_TILE_KERNEL(name##_rows, G, kRowBytes, false, false)           \
  MO_TILE_KERNEL(name##_bytes_t, G, kBlockBytes, false, true)       \
  MO_TILE_KERNEL(name##_floats_t, G, kBlockFloats, false, true)     \
  MO_TILE_KERNEL(name##_bytes_w, G, kBlockBytes, true, false)       \
  MO_TILE_KERNEL(name##_floats_w, G, kBlockFloats, true, false)     \
  MO_TILE_KERNEL(name##_rows_w, G, kRowBytes, true, false)          \
  MO_TILE_KERNEL(name##_bytes_tw, G, kBlockBytes, true, true)       \
  MO_TILE_KERNEL(name##_floats_tw, G, kBlockFloats, true, true)
typedef Tile<2, 4, 4, 2> Large;  // 256 x 256
typedef Tile<2, 2, 2, 2> Middle;  // 128 x 128
typedef Tile<2, 2, 1, 1> Small;  // 64 x 64
MO_TILE(large, Large)
MO_TILE(middle, Middle)
MO_TILE(small, Small)

}  // namespace
