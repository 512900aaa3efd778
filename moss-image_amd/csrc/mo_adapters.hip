// Low-rank adapters of many requests at once beside a shared projection, for gfx950.
//
//   h = x a_i^T,  y = result + c_i h b_i^T, i the adapter of the request that the row belongs to
//   backward, g the output's gradient:  d h = c_i g b_i,  d x = add + d h a_i,
//   d a_i = sum d h^T x,  d b_i = c_i sum g^T h over the rows of i's requests
// (one request with one adapter: the reference's LoRA linear, lora.py:60-86.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mo_adapters.h"
#include "mo_keep.h"

namespace {

using mo_adapters::Args;
using namespace mo_keep;

constexpr uint32_t kNone = 0xffffffffu;

__device__ __forceinline__ uint32_t divide(uint32_t n, const mo_block::Divisor& by) {
  return (__umulhi(by.m, n) + n) >> by.s;
}

__device__ __forceinline__ uint32_t adapter_of(const Args& a, uint32_t row) {
  uint32_t request;
  if (!a.cu) {
    request = divide(row, a.by_share);
  } else {
    uint32_t low = 0, high = a.requests;  // the number of requests that end at or before the row
    while (low < high) {
      const uint32_t mid = (low + high) / 2;
      if (a.cu[mid + 1] <= (int64_t)row)
        low = mid + 1;
      else
        high = mid;
    }
    if (low == a.requests || a.cu[low] > (int64_t)row) return kNone;
    request = low;
  }
  if (!a.index) return a.adapters == 1 ? 0 : request;
  const int64_t i = a.index[request];
  return i < 0 || i >= (int64_t)a.adapters ? kNone : (uint32_t)i;
}

__device__ __forceinline__ float scale_of(const Args& a, uint32_t adapter) { return a.scale ? a.scale[adapter] * a.factor : a.factor; }

template <class T>
__device__ __forceinline__ float x_value(const Args& a, uint32_t row, uint32_t c) {
  if (!a.x_exponents) return (float)((const T*)a.x)[row * a.x_stride + c];
  const uint32_t e = a.x_exponents[(uint64_t)row * a.groups + c / kGroup];
  return (float)((const int8_t*)a.x)[(uint64_t)row * a.groups * kGroup + c] * __builtin_bit_cast(float, e << 23);
}

// A wave a row and a rank: hidden (forward) or back (backward).
template <class T, bool kBackward>
__device__ __forceinline__ void shrink(const Args& a) {
  const uint64_t item = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const uint32_t row = (uint32_t)(item / a.rank), j = (uint32_t)(item % a.rank), lane = threadIdx.x % 64;
  if (row >= a.rows) return;
  const uint32_t i = adapter_of(a, row);
  float sum = 0.0f;
  if (i != kNone) {
    if (kBackward)
      for (uint32_t o = lane; o < a.out; o += 64)
        sum += (float)((const T*)a.grad)[row * a.grad_stride + o] * (float)((const T*)a.b)[((uint64_t)i * a.out + o) * a.rank + j];
    else
      for (uint32_t c = lane; c < a.in; c += 64)
        sum += x_value<T>(a, row, c) * (float)((const T*)a.a)[((uint64_t)i * a.rank + j) * a.in + c];
  }
  for (int s = 1; s < 64; s *= 2) sum += __shfl_xor(sum, s);
  if (lane == 0) (kBackward ? a.back : a.hidden)[(uint64_t)row * a.rank + j] = kBackward && i != kNone ? sum * scale_of(a, i) : sum;
}

// A lane a value: y (forward) or dx (backward).
template <class T, bool kBackward>
__device__ __forceinline__ void expand(const Args& a) {
  const uint32_t cols = kBackward ? a.in : a.out;
  const uint64_t item = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = (uint32_t)(item / cols), c = (uint32_t)(item % cols);
  if (row >= a.rows) return;
  const uint32_t i = adapter_of(a, row);
  float sum = 0.0f;
  if (i != kNone) {
    for (uint32_t j = 0; j < a.rank; ++j)
      sum += (kBackward ? a.back : a.hidden)[(uint64_t)row * a.rank + j] *
             (float)(kBackward ? ((const T*)a.a)[((uint64_t)i * a.rank + j) * a.in + c]
                               : ((const T*)a.b)[((uint64_t)i * a.out + c) * a.rank + j]);
    if (!kBackward) sum *= scale_of(a, i);
  }
  if (kBackward)
    ((T*)a.dx)[(uint64_t)row * cols + c] = (T)((a.add ? (float)((const T*)a.add)[row * a.add_stride + c] : 0.0f) + sum);
  else
    ((T*)a.y)[(uint64_t)row * cols + c] = (T)((float)((const T*)a.result)[row * a.result_stride + c] + sum);
}

// A lane a value of da or db, over all rows.
template <class T, bool kB>
__device__ __forceinline__ void outer(const Args& a) {
  const uint32_t cols = kB ? a.out : a.in;
  const uint64_t item = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t c = (uint32_t)(item % cols), j = (uint32_t)(item / cols % a.rank);
  const uint64_t i = item / cols / a.rank;
  if (i >= a.adapters) return;
  float sum = 0.0f;
  for (uint32_t request = 0; request < a.requests; ++request) {
    int64_t low = a.cu ? a.cu[request] : (int64_t)request * a.by_share.d, high = a.cu ? a.cu[request + 1] : low + a.by_share.d;
    low = low < 0 ? 0 : low;
    high = high > (int64_t)a.rows ? (int64_t)a.rows : high;
    const int64_t which = a.index ? a.index[request] : a.adapters == 1 ? 0 : (int64_t)request;
    if (which != (int64_t)i) continue;
    for (int64_t row = low; row < high; ++row)
      sum += kB ? a.hidden[row * a.rank + j] * (float)((const T*)a.grad)[row * a.grad_stride + c]
                : a.back[row * a.rank + j] * x_value<T>(a, (uint32_t)row, c);
  }
  if (kB)
    ((T*)a.db)[(i * a.out + c) * a.rank + j] = (T)(sum * scale_of(a, (uint32_t)i));
  else
    ((T*)a.da)[(i * a.rank + j) * a.in + c] = (T)sum;
}

#define MO_ADAPTERS(T, t)                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_hidden_##t(Args a) { shrink<T, false>(a); }       \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_back_##t(Args a) { shrink<T, true>(a); }          \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_y_##t(Args a) { expand<T, false>(a); }            \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_dx_##t(Args a) { expand<T, true>(a); }            \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_da_##t(Args a) { outer<T, false>(a); }            \
  extern "C" __global__ __launch_bounds__(256) void mo_adapters_db_##t(Args a) { outer<T, true>(a); }
MO_ADAPTERS(_Float16, f16)
MO_ADAPTERS(__bf16, bf16)
MO_ADAPTERS(float, f32)

}  // namespace
