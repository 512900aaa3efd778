// Shared by the device and host sides of the rotary positions (mo_rotary.hip, mo_rotary.cpp).
#pragma once
#include <stdint.h>

namespace mo_rotary {

constexpr uint32_t kMaxHead = 512;
constexpr uint32_t kMaxBlocks = 1024;  // workgroups a side of a backward call with a norm: partial sums kept

// Division of a number under 2^31 by a fixed one: (n + n m / 2^32) >> s (mo_layout.h makes m and s).
struct Divisor {
  uint32_t d, m, s;
};

// One side (queries or keys): tensors [batch][tokens][heads][head_dim], the last dimension dense.
struct Side {
  const void* x;       // input (null in a backward call without a norm)
  const void* grad;    // backward: the output's gradient
  void* out;           // forward: the output; backward: the input's gradient
  const void* weight;  // the norm's, [head_dim], or null
  float* partial;      // backward with a norm: [blocks][head_dim] sums of the weight's gradient
  void* weight_grad;   // [head_dim], in the weight's type
  int64_t x_batch, x_token, x_head;  // strides in elements
  int64_t g_batch, g_token, g_head;
  uint32_t heads, blocks;  // heads 0: no such side
  Divisor by_heads;
};

struct Args {
  Side side[2];
  const void* table;  // [batch or 1][tokens][rotary_dim]: sines, then cosines
  uint64_t table_batch;  // stride in elements, 0 where one table serves every batch entry
  uint32_t batch, tokens, head_dim, rotary_dim;
  uint32_t table_kind, weight_kind;  // MO_DTYPE_*
  uint32_t interleaved;
  float eps;
  Divisor by_tokens;
};

}  // namespace mo_rotary
