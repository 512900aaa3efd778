// Host side of the 8-bit floating-point operators (csrc/mo_fp8.hip): argument checks, module loading
// from the embedded gfx950 code object, workspace layouts and launches. C ABI: mo_fp8_*.
#include "mo_fp8.h"

#include <hip/hip_runtime_api.h>

#include <map>
#include <mutex>
#include <string>

#include "../../include/moss_offload.h"

extern "C" const unsigned char mo_fp8_code[];

namespace mo {
int set_error(int code, const std::string& msg);
int set_hip_error(int e, const char* what);
}  // namespace mo

namespace {

using mo_fp8::kGroup;
using mo_fp8::ProductArgs;

enum Form { kFormRows, kFormColumns, kFormBoth, kFormWeight, kForms };
const char* const kFormNames[kForms] = {"rows", "columns", "both", "weight"};
const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

// How the second operand's scales come: a byte or an fp32 number a block of 128 x 128, or a byte a row.
enum { kScaleBytes = MO_FP8_SCALE_E8M0, kScaleFloats = MO_FP8_SCALE_F32, kScaleRows = 2 };
const char* const kScaleNames[3] = {"bytes", "floats", "rows"};

struct Module {
  hipModule_t module = nullptr;
  int cus = 0;
  hipFunction_t quantize[kForms][3] = {};
  hipFunction_t decode = nullptr, transpose = nullptr;
  hipFunction_t large[3][2][2] = {};  // [scales][fp32 output][transposed]
  hipFunction_t plain[2][2] = {};  // [fp32 output][fp32 scales]
};

std::mutex g_mu;
std::map<int, Module> g_modules;

int load_module(Module* out) {
  int device = 0;
  hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) return mo::set_hip_error((int)e, "hipGetDevice");
  std::lock_guard<std::mutex> lock(g_mu);
  auto it = g_modules.find(device);
  if (it == g_modules.end()) {
    Module m;
    if ((e = hipModuleLoadData(&m.module, mo_fp8_code)) != hipSuccess)
      return mo::set_hip_error((int)e, "hipModuleLoadData (fp8 code object)");
    if ((e = hipDeviceGetAttribute(&m.cus, hipDeviceAttributeMultiprocessorCount, device)) != hipSuccess)
      return mo::set_hip_error((int)e, "hipDeviceGetAttribute (CU count)");
    auto get = [&](hipFunction_t* fn, const std::string& name) {
      return (e = hipModuleGetFunction(fn, m.module, name.c_str())) == hipSuccess;
    };
    bool ok = get(&m.decode, "mo_fp8_decode_kernel") && get(&m.transpose, "mo_fp8_transpose_kernel") &&
              get(&m.plain[0][0], "mo_fp8_product_plain") && get(&m.plain[0][1], "mo_fp8_product_plain_f32") &&
              get(&m.plain[1][0], "mo_fp8_product_plain_wide") && get(&m.plain[1][1], "mo_fp8_product_plain_wide_f32");
    for (int f = 0; f < kForms; ++f)
      for (int t = 0; t < 3; ++t)
        ok = ok && get(&m.quantize[f][t], std::string("mo_fp8_quantize_") + kFormNames[f] + "_" + kTypeNames[t]);
    for (int k = 0; k < 3; ++k)
      for (int wide = 0; wide < 2; ++wide)
        for (int trans = 0; trans < (k == kScaleRows ? 1 : 2); ++trans) {
          std::string name = std::string("mo_fp8_product_large_") + kScaleNames[k];
          if (trans || wide) name += std::string("_") + (trans ? "t" : "") + (wide ? "w" : "");
          ok = ok && get(&m.large[k][wide][trans], name);
        }
    if (!ok) return mo::set_hip_error((int)e, "hipModuleGetFunction (fp8)");
    it = g_modules.emplace(device, m).first;
  }
  *out = it->second;
  return 0;
}

// No exception crosses the boundary (a failed allocation in a map or a message is what could).
template <class F>
int guarded(F&& body) {
  try {
    return body();
  } catch (...) {
    return mo::set_error(MO_E_HOST_OOM, "no host memory");  // short: needs no allocation itself
  }
}

uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t align(uint64_t bytes) { return (bytes + 255) & ~uint64_t(255); }
uint64_t scale_pitch(uint64_t rows) { return (rows + 15) & ~uint64_t(15); }  // bytes of a group's scales

int launch(hipFunction_t fn, uint64_t blocks, uint32_t threads, void** params, uint64_t stream, const char* what) {
  if (blocks == 0 || blocks >= (1ull << 31)) return mo::set_error(MO_E_INVALID, std::string(what) + ": grid too large");
  const hipError_t e =
      hipModuleLaunchKernel(fn, (uint32_t)blocks, 1, 1, threads, 1, 1, 0, (hipStream_t)stream, params, nullptr);
  return e == hipSuccess ? 0 : mo::set_hip_error((int)e, what);
}

int check_matrix(uint64_t x, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t stride) {
  if (!x) return mo::set_error(MO_E_INVALID, "null matrix pointer");
  if (dtype > MO_DTYPE_F32) return mo::set_error(MO_E_INVALID, "unknown element type");
  if (rows == 0 || cols == 0) return mo::set_error(MO_E_INVALID, "empty matrix");
  if (cols % 16 || cols > (1u << 20)) return mo::set_error(MO_E_INVALID, "features must be multiples of 16, at most 2^20");
  if (rows >= (1ull << 31)) return mo::set_error(MO_E_INVALID, "too many rows");
  if (stride < cols || stride >= (1ull << 40)) return mo::set_error(MO_E_INVALID, "row stride out of range");
  if (x % 16 || stride * kTypeBytes[dtype] % 16)
    return mo::set_error(MO_E_INVALID, "matrix rows must be 16-byte aligned");
  return 0;
}

int quantize(const Module& m, Form form, uint64_t x, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t stride,
             uint64_t rv, uint64_t rs, uint64_t cv, uint64_t cs, uint64_t stream) {
  const void *X = (const void*)x, *RV = (const void*)rv, *RS = (const void*)rs, *CV = (const void*)cv,
             *CS = (const void*)cs;
  void* params[] = {&X, &rows, &cols, &stride, &RV, &RS, &CV, &CS};
  return launch(m.quantize[form][dtype], div_up(rows, kGroup) * div_up(cols, kGroup), 256, params, stream,
                "fp8 quantize launch");
}

// Whether a call of `rows` runs on the tiles (below, on the plain kernel, whose second operand lies along the
// reduction).
bool tiles(uint64_t rows) { return rows > 256; }

int product(const Module& m, const ProductArgs& p, int scales, bool trans, uint64_t stream) {
  ProductArgs args = p;
  void* params[] = {&args};
  const bool wide = p.out_kind == MO_DTYPE_F32;
  if (tiles(p.m))
    return launch(m.large[scales][wide][trans], div_up(p.m, 256) * div_up(p.n, 256), 512, params, stream,
                  "fp8 product launch");
  return launch(m.plain[wide][scales == kScaleFloats], div_up(p.m, 64) * div_up(p.n, 64), 256, params, stream,
                "fp8 product launch");
}

int check_weight(uint64_t w, uint64_t scale, uint32_t kind, uint32_t in_f, uint32_t out_f) {
  if (!w || !scale) return mo::set_error(MO_E_INVALID, "null weight or scale pointer");
  if (kind != MO_FP8_SCALE_E8M0 && kind != MO_FP8_SCALE_F32) return mo::set_error(MO_E_INVALID, "unknown scale type");
  if (in_f == 0 || out_f == 0) return mo::set_error(MO_E_INVALID, "empty weight");
  if (in_f % 16 || out_f % 16 || in_f > (1u << 20) || out_f > (1u << 20))
    return mo::set_error(MO_E_INVALID, "features must be multiples of 16, at most 2^20 (got " + std::to_string(in_f) +
                                           ", " + std::to_string(out_f) + ")");
  // 32-bit buffer offsets
  if ((uint64_t)in_f * out_f >= (1ull << 31)) return mo::set_error(MO_E_INVALID, "weight too large (2^31 values or more)");
  if (w % 16 || (kind == MO_FP8_SCALE_F32 && scale % 4))
    return mo::set_error(MO_E_INVALID, "misaligned weight or scale pointer");
  return 0;
}

int check_output(uint64_t out, uint32_t dtype, uint64_t bias) {
  if (!out) return mo::set_error(MO_E_INVALID, "null output pointer");
  if (dtype > MO_DTYPE_F32) return mo::set_error(MO_E_INVALID, "unknown output type");
  if (out % 16 || bias % kTypeBytes[dtype]) return mo::set_error(MO_E_INVALID, "misaligned output or bias pointer");
  return 0;
}

// Activations of a product: a matrix to quantize, or values [rows][cols] with scales already (scales != 0).
int check_operand(uint64_t x, uint64_t scales, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t stride) {
  if (!scales) return check_matrix(x, dtype, rows, cols, stride);
  if (!x || x % 16 || scales % 4) return mo::set_error(MO_E_INVALID, "null or misaligned quantized operand");
  if (rows == 0 || rows >= (1ull << 31)) return mo::set_error(MO_E_INVALID, "empty matrix, or too many rows");
  return 0;
}

int check_workspace(uint64_t workspace, uint64_t bytes, uint64_t needed) {
  if (needed == 0) return 0;
  if (!workspace || workspace % 256) return mo::set_error(MO_E_INVALID, "workspace must be 256-byte aligned device memory");
  if (bytes < needed) return mo::set_error(MO_E_INVALID, "workspace smaller than mo_fp8_workspace_bytes");
  return 0;
}

// Bytes of a quantized operand in a workspace: values, then scales.
uint64_t row_bytes(uint64_t rows, uint64_t cols) { return align(rows * cols) + align(div_up(cols, kGroup) * scale_pitch(rows)); }
uint64_t col_bytes(uint64_t rows, uint64_t cols) {
  return align(cols * div_up(rows, kGroup) * kGroup) + align(div_up(rows, kGroup) * cols);
}

uint64_t workspace_of(uint32_t op, uint64_t rows, uint64_t in_f, uint64_t out_f, bool quantized) {
  if (op == MO_FP8_FORWARD) return quantized ? 0 : row_bytes(rows, in_f);
  if (op == MO_FP8_BACKWARD) return (quantized ? 0 : row_bytes(rows, out_f)) + align(in_f * out_f);
  if (op == MO_FP8_WEIGHT) return quantized ? 0 : col_bytes(rows, out_f) + col_bytes(rows, in_f);
  return 0;
}

}  // namespace

extern "C" {

uint64_t mo_fp8_workspace_bytes(uint32_t op, uint64_t rows, uint32_t in_features, uint32_t out_features,
                                uint32_t quantized) {
  return rows ? workspace_of(op, rows, in_features, out_features, quantized != 0) : 0;
}

int mo_fp8_quantize(uint64_t x, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t row_stride, uint64_t row_values,
                    uint64_t row_scales, uint64_t col_values, uint64_t col_scales, uint64_t stream) {
  return guarded([&]() -> int {
    if (int rc = check_matrix(x, dtype, rows, cols, row_stride)) return rc;
    if (!row_values != !row_scales || !col_values != !col_scales || (!row_values && !col_values))
      return mo::set_error(MO_E_INVALID, "values and scales come in pairs, one at least");
    if ((row_values | col_values) % 16) return mo::set_error(MO_E_INVALID, "values must be 16-byte aligned");
    Module m;
    if (int rc = load_module(&m)) return rc;
    const Form form = !col_values ? kFormRows : !row_values ? kFormColumns : kFormBoth;
    return quantize(m, form, x, dtype, rows, cols, row_stride, row_values, row_scales, col_values, col_scales, stream);
  });
}

int mo_fp8_quantize_weight(uint64_t w, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t row_stride,
                           uint64_t values, uint64_t scales, uint64_t stream) {
  return guarded([&]() -> int {
    if (int rc = check_matrix(w, dtype, rows, cols, row_stride)) return rc;
    if (!values || !scales || values % 16) return mo::set_error(MO_E_INVALID, "null or misaligned output");
    Module m;
    if (int rc = load_module(&m)) return rc;
    return quantize(m, kFormWeight, w, dtype, rows, cols, row_stride, values, scales, 0, 0, stream);
  });
}

int mo_fp8_decode(uint64_t values, uint64_t pitch, uint64_t scales, uint32_t scale_kind, uint64_t scale_row,
                  uint64_t scale_col, uint32_t block_rows, uint64_t out, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t stream) {
  return guarded([&]() -> int {
    if (!values || !scales || !out) return mo::set_error(MO_E_INVALID, "null pointer");
    if (rows == 0 || cols == 0) return mo::set_error(MO_E_INVALID, "empty matrix");
    if (scale_kind != MO_FP8_SCALE_E8M0 && scale_kind != MO_FP8_SCALE_F32)
      return mo::set_error(MO_E_INVALID, "unknown scale type");
    if (block_rows != 1 && block_rows != kGroup) return mo::set_error(MO_E_INVALID, "a scale covers 1 or 128 rows");
    if (dtype > MO_DTYPE_F32) return mo::set_error(MO_E_INVALID, "unknown output type");
    if (values % 16 || pitch % 16 || pitch < cols || out % 16 || (scale_kind == MO_FP8_SCALE_F32 && scales % 4))
      return mo::set_error(MO_E_INVALID, "misaligned pointer, or pitch out of range");
    if (rows >= (1ull << 31)) return mo::set_error(MO_E_INVALID, "too many rows");
    Module m;
    if (int rc = load_module(&m)) return rc;
    const void *V = (const void*)values, *S = (const void*)scales;
    void* O = (void*)out;
    uint32_t shift = block_rows == 1 ? 0 : 7;
    void* params[] = {&V, &pitch, &S, &scale_kind, &scale_row, &scale_col, &shift, &O, &dtype, &rows, &cols};
    return launch(m.decode, div_up(rows * div_up(cols, 16), 256), 256, params, stream, "fp8 decode launch");
  });
}

int mo_fp8_linear_forward(uint64_t x, uint64_t x_scales, uint32_t dtype, uint64_t rows, uint32_t in_features,
                          uint64_t row_stride, uint64_t w, uint64_t w_scale, uint32_t scale_kind,
                          uint32_t out_features, uint64_t bias, uint64_t y, uint32_t y_dtype, uint64_t workspace,
                          uint64_t workspace_bytes, uint64_t stream) {
  return guarded([&]() -> int {
    if (int rc = check_weight(w, w_scale, scale_kind, in_features, out_features)) return rc;
    if (int rc = check_operand(x, x_scales, dtype, rows, in_features, row_stride)) return rc;
    if (int rc = check_output(y, y_dtype, bias)) return rc;
    const uint64_t needed = workspace_of(MO_FP8_FORWARD, rows, in_features, out_features, x_scales != 0);
    if (int rc = check_workspace(workspace, workspace_bytes, needed)) return rc;
    Module m;
    if (int rc = load_module(&m)) return rc;
    if (!x_scales) {
      const uint64_t scales = workspace + align(rows * in_features);
      if (int rc = quantize(m, kFormRows, x, dtype, rows, in_features, row_stride, workspace, scales, 0, 0, stream))
        return rc;
      x = workspace, x_scales = scales;
    }
    ProductArgs p = {};
    p.a = (const uint8_t*)x, p.a_scales = (const uint8_t*)x_scales, p.a_pitch = in_features;
    p.a_scale_pitch = (uint32_t)scale_pitch(rows);
    p.b = (const uint8_t*)w, p.b_scales = (const void*)w_scale, p.b_pitch = in_features;
    p.b_scale_row = (uint32_t)div_up(in_features, kGroup), p.b_scale_col = 1, p.b_shift = 7;
    p.bias = (const void*)bias, p.out = (void*)y, p.out_kind = y_dtype;
    p.m = rows, p.n = out_features, p.r = in_features;
    return product(m, p, (int)scale_kind, false, stream);
  });
}

int mo_fp8_linear_backward(uint64_t dy, uint64_t dy_scales, uint32_t dtype, uint64_t rows, uint32_t in_features,
                           uint32_t out_features, uint64_t row_stride, uint64_t w, uint64_t w_scale,
                           uint32_t scale_kind, uint64_t dx, uint32_t dx_dtype, uint64_t workspace,
                           uint64_t workspace_bytes, uint64_t stream) {
  return guarded([&]() -> int {
    if (int rc = check_weight(w, w_scale, scale_kind, in_features, out_features)) return rc;
    if (int rc = check_operand(dy, dy_scales, dtype, rows, out_features, row_stride)) return rc;
    if (int rc = check_output(dx, dx_dtype, 0)) return rc;
    const uint64_t needed = workspace_of(MO_FP8_BACKWARD, rows, in_features, out_features, dy_scales != 0);
    if (int rc = check_workspace(workspace, workspace_bytes, needed)) return rc;
    Module m;
    if (int rc = load_module(&m)) return rc;
    const bool trans = tiles(rows);
    if (!trans) {  // the weight with the reduction (out_features) contiguous
      const void* in = (const void*)w;
      void* out = (void*)workspace;
      uint32_t r = out_features, c = in_features;
      void* params[] = {&in, &out, &r, &c};
      if (int rc = launch(m.transpose, div_up(r, 128) * div_up(c, 128), 256, params, stream, "fp8 transpose launch"))
        return rc;
    }
    if (!dy_scales) {
      const uint64_t values = workspace + align((uint64_t)in_features * out_features);
      const uint64_t scales = values + align(rows * out_features);
      if (int rc = quantize(m, kFormRows, dy, dtype, rows, out_features, row_stride, values, scales, 0, 0, stream))
        return rc;
      dy = values, dy_scales = scales;
    }
    ProductArgs p = {};
    p.a = (const uint8_t*)dy, p.a_scales = (const uint8_t*)dy_scales, p.a_pitch = out_features;
    p.a_scale_pitch = (uint32_t)scale_pitch(rows);
    p.b = trans ? (const uint8_t*)w : (const uint8_t*)workspace;
    p.b_scales = (const void*)w_scale, p.b_pitch = trans ? in_features : out_features;
    p.b_scale_row = 1, p.b_scale_col = (uint32_t)div_up(in_features, kGroup), p.b_shift = 7;
    p.out = (void*)dx, p.out_kind = dx_dtype;
    p.m = rows, p.n = in_features, p.r = out_features;
    return product(m, p, (int)scale_kind, trans, stream);
  });
}

int mo_fp8_weight_gradient(uint64_t dy, uint64_t dy_scales, uint32_t dy_dtype, uint64_t dy_stride, uint64_t x,
                           uint64_t x_scales, uint32_t x_dtype, uint64_t x_stride, uint64_t rows,
                           uint32_t in_features, uint32_t out_features, uint64_t dw, uint32_t dw_dtype,
                           uint64_t workspace, uint64_t workspace_bytes, uint64_t stream) {
  return guarded([&]() -> int {
    if (in_features == 0 || out_features == 0 || in_features % 16 || out_features % 16 || in_features > (1u << 20) ||
        out_features > (1u << 20))
      return mo::set_error(MO_E_INVALID, "features must be multiples of 16, at most 2^20");
    if (!dy_scales != !x_scales) return mo::set_error(MO_E_INVALID, "both operands are quantized, or neither");
    if (int rc = check_operand(dy, dy_scales, dy_dtype, rows, out_features, dy_stride)) return rc;
    if (int rc = check_operand(x, x_scales, x_dtype, rows, in_features, x_stride)) return rc;
    if (int rc = check_output(dw, dw_dtype, 0)) return rc;
    const uint64_t needed = workspace_of(MO_FP8_WEIGHT, rows, in_features, out_features, dy_scales != 0);
    if (int rc = check_workspace(workspace, workspace_bytes, needed)) return rc;
    Module m;
    if (int rc = load_module(&m)) return rc;
    const uint64_t padded = div_up(rows, kGroup) * kGroup;
    if (padded * 256 >= (1ull << 31))  // 32-bit buffer offsets over a tile's rows
      return mo::set_error(MO_E_INVALID, "too many rows for one weight gradient (2^23 - 128 at most)");
    if (!dy_scales) {
      const uint64_t dv = workspace, ds = dv + align(out_features * padded);
      const uint64_t xv = workspace + col_bytes(rows, out_features), xs = xv + align(in_features * padded);
      if (int rc = quantize(m, kFormColumns, dy, dy_dtype, rows, out_features, dy_stride, 0, 0, dv, ds, stream))
        return rc;
      if (int rc = quantize(m, kFormColumns, x, x_dtype, rows, in_features, x_stride, 0, 0, xv, xs, stream)) return rc;
      dy = dv, dy_scales = ds, x = xv, x_scales = xs;
    }
    ProductArgs p = {};
    p.a = (const uint8_t*)dy, p.a_scales = (const uint8_t*)dy_scales, p.a_pitch = padded;
    p.a_scale_pitch = out_features;
    p.b = (const uint8_t*)x, p.b_scales = (const void*)x_scales, p.b_pitch = padded;
    p.b_scale_row = 1, p.b_scale_col = in_features, p.b_shift = 0;
    p.out = (void*)dw, p.out_kind = dw_dtype;
    p.m = out_features, p.n = in_features, p.r = (uint32_t)padded;
    return product(m, p, kScaleRows, false, stream);
  });
}

}  // extern "C"
