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
// Gaussian operands come out 1.5e-5 off, in the scaled, the unscaled and the 16-deep form alike). That is
// a hundredth of a bf16 rounding and a tenth of an fp16 one, and stays for 16-bit outputs. An fp32 output
// is asked for its fp32 sums: those kernels decode the operands to bf16, which is exact, and use the bf16
// instructions (half the rate, 6e-8 off).
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

#include "mo_fp8.h"

namespace {

using mo_fp8::ProductArgs;
using mo_fp8::kBF16;
using mo_fp8::kF32;
using mo_fp8::kGroup;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
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
// 8 g + 7 of columns 8 c to 8 c + 7. A row's 16 threads are one DPP row, so its maximum takes four DPP
// steps; a column's maximum is taken over the thread's own rows, the four row groups of its wave, and
// the waves through LDS. The columns' bytes are turned in LDS and leave as whole 128-byte lines.

enum { kRows = 1, kColumns = 2, kBlock = 4 };

template <class T, int kForm>
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
  const uint64_t row0 = tile_r * kGroup + 8 * g;
  const uint32_t col0 = tile_c * kGroup + 8 * c;
  const bool in_cols = col0 < cols;  // cols is a multiple of 16: a thread's eight are in or out

  Bits<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (in_cols && row0 + i < rows)
      v[i].load(x + (row0 + i) * stride + col0);
    else
      v[i].zero();
  }

  if (kForm & kRows) {
    const uint32_t pitch = (tiles_c + 3) & ~3u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
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
        if (c == 0) row_scales[(row0 + i) * pitch + tile_c] = (uint8_t)byte;
      }
    }
  }

  if (kForm & (kColumns | kBlock)) {
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
      const uint64_t groups = (rows + kGroup - 1) / kGroup, pitch = groups * kGroup;
      const uint64_t scale_pitch = (groups + 3) & ~(uint64_t)3;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t byte = scale_byte(m[j]);
        const float inv = inverse_scale(byte);
        u32x2 w;
        w[0] = pack4(v[0].get(j) * inv, v[1].get(j) * inv, v[2].get(j) * inv, v[3].get(j) * inv);
        w[1] = pack4(v[4].get(j) * inv, v[5].get(j) * inv, v[6].get(j) * inv, v[7].get(j) * inv);
        *(u32x2*)(turned + (8 * c + j) * kLine + 8 * g) = w;
        if (g == 0 && in_cols) col_scales[(uint64_t)(col0 + j) * scale_pitch + tile_r] = (uint8_t)byte;
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

#define MO_QUANTIZE(name, T, form)                                                                            \
  extern "C" __global__ __launch_bounds__(256) void mo_fp8_quantize_##name(                                   \
      const T* x, uint64_t rows, uint32_t cols, uint64_t stride, uint8_t* row_values, uint8_t* row_scales,    \
      uint8_t* col_values, uint8_t* col_scales) {                                                             \
    quantize_tile<T, form>(x, rows, cols, stride, row_values, row_scales, col_values, col_scales);            \
  }
#define MO_QUANTIZE_FORMS(t, T)                     \
  MO_QUANTIZE(rows_##t, T, kRows)                   \
  MO_QUANTIZE(columns_##t, T, kColumns)             \
  MO_QUANTIZE(both_##t, T, kRows | kColumns)        \
  MO_QUANTIZE(weight_##t, T, kBlock)
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

// One lane reads 16 values and their scale and writes 16 products: bound by memory.
extern "C" __global__ __launch_bounds__(256) void mo_fp8_decode_kernel(
    const uint8_t* __restrict__ values, uint64_t pitch, const void* __restrict__ scales, uint32_t f32_scales,
    uint64_t scale_pitch, uint32_t shift, void* __restrict__ out, uint32_t kind, uint64_t rows, uint32_t cols) {
  const uint32_t chunks = (cols + 15) / 16;
  const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t row = at / chunks;
  const uint32_t col = (uint32_t)(at % chunks) * 16;
  if (row >= rows) return;
  const u32x4 w = *(const u32x4*)(values + row * pitch + col);
  const uint64_t s = (row >> shift) * scale_pitch + col / kGroup;
  const float scale = f32_scales ? ((const float*)scales)[s] : scale_value(((const uint8_t*)scales)[s]);
  const bool whole = col + 16 <= cols && cols % 4 == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    const f32x4 v = {lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
    if (whole) {
      store4(out, row * cols + col + 4 * i, v, kind);
    } else {
      for (int j = 0; j < 4; ++j) {
        if (col + 4 * i + j >= cols) break;
        const uint64_t o = row * cols + col + 4 * i + j;
        if (kind == kF32)
          ((float*)out)[o] = v[j];
        else if (kind == kBF16)
          ((__bf16*)out)[o] = (__bf16)v[j];
        else
          ((_Float16*)out)[o] = (_Float16)v[j];
      }
    }
  }
}

// out[c][r] = in[r][c], bytes; rows and cols multiples of 16. A tile of 128 x 128 through LDS.
extern "C" __global__ __launch_bounds__(256) void mo_fp8_transpose_kernel(const uint8_t* __restrict__ in,
                                                                          uint8_t* __restrict__ out, uint32_t rows,
                                                                          uint32_t cols) {
  constexpr int kLine = 128 + 4;
  __shared__ __attribute__((aligned(16))) uint8_t tile[128 * kLine];
  const uint32_t tiles_c = (cols + 127) / 128;
  const uint32_t r0 = blockIdx.x / tiles_c * 128, c0 = blockIdx.x % tiles_c * 128;
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t r = (tid >> 3) + 32 * i, c = (tid & 7) * 16;
    u32x4 v = {};
    if (r0 + r < rows && c0 + c < cols) v = *(const u32x4*)(in + (uint64_t)(r0 + r) * cols + c0 + c);
    uint32_t* to = (uint32_t*)(tile + r * kLine + c);
    to[0] = v[0], to[1] = v[1], to[2] = v[2], to[3] = v[3];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = (tid & 31) + 32 * i, r = (tid >> 5) * 16;
    if (c0 + c >= cols || r0 + r >= rows) continue;
    u32x4 v;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t x = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) x |= (uint32_t)tile[(r + 4 * w + b) * kLine + c] << (8 * b);
      v[w] = x;
    }
    *(u32x4*)(out + (uint64_t)(c0 + c) * rows + r0 + r) = v;
  }
}

// ---- products -------------------------------------------------------------------------------------

// Output of one 32 x 32 tile: a lane holds token m and features n0 + 8 (r / 4) + 4 (l / 32) + r % 4.
__device__ __forceinline__ void store_tile(const ProductArgs& p, f32x16 acc, uint64_t m, uint32_t n0, int half) {
  if (m >= p.m) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t n = n0 + 8 * q + 4 * half;
    if (n >= p.n) continue;  // p.n is a multiple of 16
    f32x4 v = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += load1(p.bias, n + i, p.out_kind);
    }
    store4(p.out, m * p.n + n, v, p.out_kind);
  }
}

// Eight e4m3 bytes times a power of two as bf16: exact (four significant bits).
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi, float scale) {
  bf16x8 o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)(i ? hi : lo), false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)(i ? hi : lo), true);
    o[4 * i] = (__bf16)(a[0] * scale), o[4 * i + 1] = (__bf16)(a[1] * scale);
    o[4 * i + 2] = (__bf16)(b[0] * scale), o[4 * i + 3] = (__bf16)(b[1] * scale);
  }
  return o;
}

// The plain kernel: four waves of one 32 x 32 tile each, operands straight from memory.
template <bool kF32Scales, bool kWide>
__device__ __forceinline__ void product_plain(const ProductArgs& p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 31, half = lane >> 5;
  const uint32_t tiles_n = (p.n + 63) / 64;
  const uint64_t m0 = (uint64_t)(blockIdx.x / tiles_n) * 64 + 32 * (wave & 1);
  const uint32_t n0 = blockIdx.x % tiles_n * 64 + 32 * (wave >> 1);
  const uint64_t m = m0 + lr;
  const uint32_t n = n0 + lr;
  const bool in_m = m < p.m, in_n = n < p.n;
  const uint8_t* a = p.a + (in_m ? m : 0) * p.a_pitch;
  const uint8_t* b = p.b + (uint64_t)(in_n ? n : 0) * p.b_pitch;
  f32x16 acc = {};
  for (uint32_t k0 = 0; k0 < p.r; k0 += kGroup) {
    const uint32_t group = k0 / kGroup;
    const int sa = in_m ? p.a_scales[m * p.a_scale_pitch + group] : 127;
    const uint64_t at = (uint64_t)((in_n ? n : 0) >> p.b_shift) * p.b_scale_row + (uint64_t)group * p.b_scale_col;
    const int sb = kF32Scales ? 127 : ((const uint8_t*)p.b_scales)[at];
    f32x16 sum = kF32Scales ? f32x16{} : acc;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x8 fa = {}, fb = {};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t k = k0 + 64 * h + 32 * half + 16 * c;
        u32x4 va = {}, vb = {};
        if (in_m && k < p.r) va = *(const u32x4*)(a + k);
        if (in_n && k < p.r) vb = *(const u32x4*)(b + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) fa[4 * c + i] = (int)va[i], fb[4 * c + i] = (int)vb[i];
      }
      if (kWide) {
        const float xa = scale_value((uint32_t)sa), xb = scale_value((uint32_t)sb);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(fb[2 * q], fb[2 * q + 1], xb),
                                                        widen(fa[2 * q], fa[2 * q + 1], xa), sum, 0, 0, 0);
      } else {
        sum = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb, fa, sum, 0, 0, 0, sb, 0, sa);
      }
    }
    if (kF32Scales) {
      const float s = ((const float*)p.b_scales)[(uint64_t)((n0 < p.n ? n0 : 0) >> p.b_shift) * p.b_scale_row +
                                                 (uint64_t)group * p.b_scale_col];
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += sum[i] * s;
    } else {
      acc = sum;
    }
  }
  store_tile(p, acc, m, n0, half);
}

#define MO_PLAIN(name, f32_scales, wide)                                                                 \
  extern "C" __global__ __launch_bounds__(256) void mo_fp8_product_plain##name(ProductArgs p) {          \
    product_plain<f32_scales, wide>(p);                                                                  \
  }
MO_PLAIN(, false, false)
MO_PLAIN(_f32, true, false)
MO_PLAIN(_wide, false, true)
MO_PLAIN(_wide_f32, true, true)

}  // namespace
