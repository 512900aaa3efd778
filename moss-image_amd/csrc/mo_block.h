// Shared by the device and host sides of the norms (mo_norm.hip, mo_norm.cpp) and of the gated activation and
// the activations in 8 bits (mo_gated.hip, mo_gated.cpp).
#pragma once
#include <stdint.h>

namespace mo_block {

constexpr uint32_t kMaxDim = 16384;  // values a row of a norm: 512 lanes of 32

// Division of a number under 2^31 by a fixed one: (n + n m / 2^32) >> s (mo_layout.h makes m and s).
struct Divisor {
  uint32_t d, m, s;
};

struct NormArgs {
  const void* x;                 // [rows][dim] of the call's type, or 8-bit values [rows][groups * 32]
  const uint8_t* x_exponents;    // backward from 8 bits: [rows][groups]
  const void* grad;              // backward: the output's gradient
  void* out;                     // forward: the output; backward: the input's gradient
  float* stats;                  // [rows][2]: mean, 1 / deviation
  const void *weight, *bias;     // [dim] or null
  const void *scale, *shift;     // [samples][dim] or null
  int8_t* kept;                  // forward: the input in 8 bits, or null
  uint8_t* kept_exponents;
  const int64_t* cu;             // [samples + 1]: where each sample's rows begin and end; null: rows / samples each
  float* partial;                // backward: [slots][2][pitch] sums of grad * normalised and of grad
  float* sample_sums;            // [samples][2][pitch], where more than one sample makes a weight's gradient
  void *weight_grad, *bias_grad, *scale_grad, *shift_grad;
  uint64_t x_stride, grad_stride, scale_stride, shift_stride;  // elements between rows
  uint32_t rows, dim, samples, groups, pitch;
  uint32_t lanes, per, chunk;    // lanes a row, rows side by side in a workgroup, rows one after the other
  uint32_t weight_kind, scale_kind;  // MO_DTYPE_*
  uint32_t layer;
  float eps;
  Divisor by_share;              // rows a sample, where cu is null
};

struct GatedArgs {
  const void *up, *gate;         // [rows][cols] each, or 8-bit values [rows][groups * 32]
  const uint8_t *up_exponents, *gate_exponents;
  const void* grad;              // backward: [rows][cols]
  void *out, *out_gate;          // forward: the output; backward: the gradients of up and gate
  int8_t *kept_up, *kept_gate;   // forward: up and gate in 8 bits, or null
  uint8_t *kept_up_exponents, *kept_gate_exponents;
  uint64_t up_stride, gate_stride, grad_stride, out_stride;  // elements between rows
  uint64_t values_stride, exponents_stride;                  // bytes between rows of what is in 8 bits
  uint32_t rows, cols, lanes;    // lanes a row: four for each 32 columns
  uint32_t silu;
  Divisor by_lanes;
};

struct KeepArgs {
  const void* x;
  void* out;
  int8_t* values;
  uint8_t* exponents;
  uint64_t stride;               // elements between rows of x or out
  uint32_t rows, cols, groups, lanes;
  Divisor by_lanes;
};

}  // namespace mo_block
