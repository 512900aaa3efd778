// Shared by the device and host sides of the low-rank adapters (mo_adapters.hip, mo_adapters.cpp).
#pragma once
#include <stdint.h>

#include "mo_block.h"

namespace mo_adapters {

constexpr uint32_t kMaxRank = 128;
constexpr uint64_t kMaxRows = 1ull << 26;    // less
constexpr uint64_t kMaxStride = 1ull << 22;  // elements between rows
constexpr uint32_t kMaxSplits = 64;   // of the rows of a weight's gradient: a bit each in a mask
constexpr uint32_t kOuterCols = 128;  // columns a workgroup of a weight's gradient

// Which rows have which adapter.
struct Requests {
  const int64_t* cu;      // [requests + 1], or null: rows / requests each
  const int64_t* index;   // [requests]: the adapter of each, any other number: none; null: 0, or the request's own
  const float* scale;     // [adapters], or null: 1; times factor
  float factor;
  uint32_t rows, requests, adapters, rank, share;
};

// to[row][j] = sum over the features of x[row][k] w_i[j][k].
struct Shrink {
  Requests by;
  const void* x;          // [rows][features]
  const void* w;          // [adapters][rank][features]
  float* to;              // [splits][rows][rank]
  uint64_t x_stride;
  uint32_t features, span;  // features a split, a multiple of 128
  uint32_t scaled;        // times the adapter's scale
  uint32_t by_request;    // w is [requests] of them: the request's place holds its adapter's
};

// to[row][n] = base[row][n] + s sum over the rank of h[row][j] v_i[n][j], h the sum of its splits.
struct Expand {
  Requests by;
  const float* h;         // [splits][rows][rank]
  float* h_sum;           // [rows][rank] or null
  float* turned;          // h turned, for an outer, or null
  const void* v;          // [adapters][features][rank]
  const void* base;       // [rows][features], or null: 0
  void* to;
  uint64_t base_stride;
  uint32_t features, splits, cols;  // columns a workgroup, a multiple of 512
  uint32_t scaled;
  uint32_t by_request;    // v is, as above
};

// Both for a forward pass of few rows.
struct Few {
  Shrink in;
  Expand out;
};

// One gradient of a weight: sum over an adapter's rows of narrow[row][j] wide[row][c].
struct Side {
  const void* wide;          // [rows][cols], or 8-bit values [rows][groups * 32]
  const uint8_t* exponents;  // [rows][groups], or null
  const float* narrow;       // turned: [rows / 8][rank][8]
  float* planes;             // [splits][adapters][cols * rank] sums over a split's rows, where there are several
  void* to;                  // [adapters][rank][cols], or turned: [adapters][cols][rank]; null: not wanted
  uint64_t stride;
  uint32_t cols, groups, tiles, splits, span;  // span: rows a split, a multiple of 32
  uint32_t turned, scaled;
};
struct Outer {
  Requests by;
  Side side[2];
};

// Copies of both weights, each [places] matrices turned, and of a narrow matrix for an outer: the sum of its splits,
// turned, [rows / 8][rank][8].
struct Turn {
  Requests by;
  const void* from[2];
  void* to[2];
  uint32_t rows[2], cols[2], tiles[2];  // of `from`; tiles of 32 x 32, 0: not wanted
  const float* narrow;                  // [splits][count][rank]
  float* turned;
  uint32_t places, by_request, count, rank, splits;  // places: the adapters, or the requests
};

}  // namespace mo_adapters
