// Activations in 8 bits, shared by the kernels that write them and the backward kernels that read them.
//
//   For each 32 values of a row: e the smallest integer, from -126 on, with max |x| <= 127 2^e;
//   q = round(x 2^-e) to the nearest whole number, ties to even; x is read back as q 2^e.
//
// values int8 [rows][groups * 32] (zero past the row's end), exponents uint8 [rows][groups], e + 127. A
// group with an infinity or a NaN has exponent 255 and zeros, and reads back as NaN: 0 * inf. Where 64 2^e is past the
// type's largest value, |q| is at most 63, so that what is read back is finite. Powers of two make both
// directions exact but for the one rounding of q, so every implementation of the rule gives the same bits; a scale of
// max / 127 would be nearer by a factor between 1 and 2. Groups of 32: against 128 a strong channel spoils a
// quarter of the values around it, for 3 % of the bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mo_keep {

constexpr uint32_t kGroup = 32;  // values an exponent; a lane holds 8, so four neighbouring lanes a group

// Eight neighbouring values from anywhere that a T may lie: gfx950 takes 16-byte accesses at any address.
template <class T>
struct alignas(T) Eight {
  T v[8];
};
template <class T>
__device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
// The first n of them, the rest zero. Where sizes are multiples of eight, n is 8 or 0, and eight values are read all the
// same (p has to be readable). Odd sizes have kernels of their own: single values need an address each, and the
// registers for those would be taken from the others too.
template <bool kOdd, class T>
__device__ __forceinline__ Eight<T> load8(const T* p, uint32_t n) {
  if (!kOdd || n >= 8) {
    Eight<T> r = load8(p);
    if (!kOdd) {
      uint32_t word[sizeof(r) / 4];
      __builtin_memcpy(word, &r, sizeof(r));
#pragma unroll
      for (int i = 0; i < (int)(sizeof(r) / 4); ++i) word[i] = n ? word[i] : 0;
      __builtin_memcpy(&r, word, sizeof(r));
    }
    return r;
  }
  Eight<T> r;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : (T)0;
  return r;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&from)[8]) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = (T)from[i];
  __builtin_memcpy(p, &r, sizeof(r));
}
// The first n of them: 8 or 0 where sizes are multiples of eight.
template <bool kOdd, class T>
__device__ __forceinline__ void store8(T* p, const Eight<T>& from, uint32_t n) {
  if (n >= 8) {
    __builtin_memcpy(p, &from, sizeof(from));
    return;
  }
  if (!kOdd) return;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i)
    if (i < n) p[i] = from.v[i];
}
template <bool kOdd, class T>
__device__ __forceinline__ void store8(T* p, const float (&from)[8], uint32_t n) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = (T)from[i];
  store8<kOdd>(p, r, n);
}
template <class T>
__device__ __forceinline__ void widen(float (&to)[8], const Eight<T>& from) {
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = (float)from.v[i];
}

// A part of memory that all lanes share: its address stays in scalar registers, a lane has 32-bit offsets (the host keeps
// rows near enough for that), and what a lane should not read or write it asks for past the end, where reads
// give zeros and writes are dropped. Odd sizes, or addresses off the 4-byte grid, go by each lane's own address, the last of a row
// value by value.
constexpr uint32_t kNowhere = 0x80000000u;  // no window is as long

template <class T, bool kOdd>
struct Window {
  T* at;
  __amdgpu_buffer_rsrc_t buffer;
  // `count` elements from `p`
  __device__ __forceinline__ Window(const T* p, uint32_t count)
      : at(const_cast<T*>(p)),
        buffer(__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, (int)(count * sizeof(T)), 0x00020000)) {}
  // the first n (8 or 0, unless kOdd) of eight elements, `shared` + `own` from the beginning; the rest are zero
  __device__ __forceinline__ Eight<T> read(uint32_t shared, uint32_t own, uint32_t n) const {
    if (kOdd) return load8<true>(at + shared + (n ? own : 0), n);
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    Words words[sizeof(Eight<T>) / 16];
    const uint32_t offset = n ? own * (uint32_t)sizeof(T) : kNowhere;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(Eight<T>) / 16; ++i)
      words[i] = __builtin_amdgcn_raw_buffer_load_b128(buffer, offset + i * 16, shared * (uint32_t)sizeof(T), 0);
    return __builtin_bit_cast(Eight<T>, words);
  }
  __device__ __forceinline__ void write(const Eight<T>& v, uint32_t shared, uint32_t own, uint32_t n) const {
    if (kOdd) {
      store8<true>(at + shared + (n ? own : 0), v, n);
      return;
    }
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    struct All {
      Words words[sizeof(Eight<T>) / 16];
    };
    const All all = __builtin_bit_cast(All, v);
    // No scalar offset: with one, the compiler lets the next instruction overwrite the registers that a 16-byte store has
    // yet to read (it counts that case as safe), and single values came out as addresses here.
    const uint32_t offset = (n ? own * (uint32_t)sizeof(T) : kNowhere) + shared * (uint32_t)sizeof(T);
#pragma unroll
    for (uint32_t i = 0; i < sizeof(Eight<T>) / 16; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(all.words[i], buffer, offset + i * 16, 0, 0);
  }
};
// The same of a type known at run time (MO_DTYPE_*).
template <bool kOdd>
__device__ __forceinline__ void load8_kind(float (&to)[8], const void* base, uint64_t at, uint32_t kind, uint32_t n) {
  if (kind == 2)
    widen(to, load8<kOdd>((const float*)base + at, n));
  else if (kind == 1)
    widen(to, load8<kOdd>((const __bf16*)base + at, n));
  else
    widen(to, load8<kOdd>((const _Float16*)base + at, n));
}
__device__ __forceinline__ void store_kind(void* base, uint64_t at, uint32_t kind, float v) {
  if (kind == 2)
    ((float*)base)[at] = v;
  else if (kind == 1)
    ((__bf16*)base)[at] = (__bf16)v;
  else
    ((_Float16*)base)[at] = (_Float16)v;
}

// The exponent byte under which 64 2^e is past the type's largest value.
template <class T>
constexpr uint32_t kTopExponent = 249;
template <>
constexpr uint32_t kTopExponent<_Float16> = 137;

template <int kControl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kControl, 0xf, 0xf, true);
}

// A lane's eight values (past the row's end: zeros) to 8 bits, the group's exponent in all four of its lanes.
template <class T>
__device__ __forceinline__ uint2 encode(const float (&v)[8], uint32_t& exponent) {
  uint32_t peak = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) peak = max(peak, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  peak = max(peak, dpp<0xB1>(peak));  // swapped neighbours
  peak = max(peak, dpp<0x4E>(peak));  // swapped pairs
  uint2 out = {0, 0};
  if (peak >= 0x7f800000u) {
    exponent = 255;
    return out;
  }
  const int e = (int)(peak >> 23) - 6 + ((peak & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  exponent = (uint32_t)max(e, 1);
  const float inverse = __builtin_bit_cast(float, (254u - exponent) << 23);
  const float most = exponent == kTopExponent<T> ? 63.0f : 127.0f;
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = (uint32_t)(int)fminf(fmaxf(rintf(v[i] * inverse), -most), most) & 0xffu;
  out.x = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
  out.y = q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24;
  return out;
}

__device__ __forceinline__ void decode(float (&to)[8], uint2 values, uint32_t exponent) {
  const float scale = __builtin_bit_cast(float, exponent << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) to[i] = (float)(int8_t)((i < 4 ? values.x : values.y) >> (8 * (i & 3))) * scale;
}

}  // namespace mo_keep
