// Shared by the device and host sides of the low-rank adapters (mo_adapters.hip, mo_adapters.cpp).
#pragma once
#include <stdint.h>

#include "mo_block.h"

namespace mo_adapters {

constexpr uint32_t kMaxRank = 128;

struct Args {
  const void* x;               // [rows][in] of the call's type, or 8-bit values [rows][groups * 32]
  const uint8_t* x_exponents;  // [rows][groups], or null
  const void* result;          // forward: [rows][out], the shared projection's
  void* y;                     // forward: [rows][out]
  const void *a, *b;           // [adapters][rank][in], [adapters][out][rank]
  const float* scale;          // [adapters], or null: 1; times factor
  const int64_t* cu;           // [requests + 1], or null: rows / requests each
  const int64_t* index;        // [requests]: the adapter of each, any other number: none; null: 0, or the request's own
  float* hidden;               // [rows][rank]: x a^T
  const void* grad;            // backward: [rows][out]
  const void* add;             // [rows][in] or null
  void *dx, *da, *db;
  float* back;                 // [rows][rank]: scale grad b
  uint64_t x_stride, result_stride, grad_stride, add_stride;  // elements between rows
  uint32_t rows, requests, adapters, rank, in, out, groups;
  float factor;
  mo_block::Divisor by_share;  // rows a request, where cu is null
};

}  // namespace mo_adapters
