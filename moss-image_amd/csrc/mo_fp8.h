// Shared by the device and host sides of the 8-bit floating-point products (mo_fp8.hip, mo_fp8.cpp).
#pragma once
#include <stdint.h>

namespace mo_fp8 {

constexpr uint32_t kGroup = 128;                   // values that share a scale
constexpr uint32_t kF16 = 0, kBF16 = 1, kF32 = 2;  // MO_DTYPE_*

// Division of a number under 2^31 by a fixed one: (n + n m / 2^32) >> s (mo_layout.h makes m and s).
struct Divisor {
  uint32_t d, m, s;
};

// C[m][n] = sum_k A[m][k] B[n][k] under their scales (+ bias[n]); pitches in bytes, scale strides in
// elements. B's scale of (n, group) is at n / 128 * b_scale_row + group * b_scale_col where a scale covers a
// block of 128 x 128, at n + group * b_scale_col in the kernels that take one a row (b_scale_row unused).
struct ProductArgs {
  const uint8_t* a;
  const uint8_t* b;
  const uint8_t* a_scales;  // one byte a row and group: group * a_scale_pitch + row
  const void* b_scales;     // bytes, or fp32 for the floats kernels
  const void* bias;         // of bias_kind, or null
  void* out;                // [m][n]
  uint64_t m, a_pitch, b_pitch;
  uint32_t n, r;
  uint32_t a_scale_pitch, b_scale_row, b_scale_col;
  uint32_t out_kind, bias_kind;
  // the reduction shared out over workgroups: each takes split_steps groups of it and leaves fp32 sums in its
  // plane, [splits][m][n]; out and bias are then the sum kernel's. splits 1: planes is null
  uint32_t splits, split_steps;
  float* planes;
};

}  // namespace mo_fp8
