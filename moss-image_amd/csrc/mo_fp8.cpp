// Host side of the 8-bit floating-point operators (csrc/mo_fp8.hip): argument checks, module loading
// from the embedded gfx950 code object, workspace layouts and launches. C ABI: mo_fp8_*.
#include "mo_fp8.h"

#include <hip/hip_runtime_api.h>

#include <map>
#include <mutex>
#include <string>

#include "../../include/moss_offload.h"
#include "mo_layout.h"

extern "C" const unsigned char mo_fp8_code[];

namespace mo {
int set_error(int code, const std::string& msg);
int set_hip_error(int e, const char* what);
}  // namespace mo

namespace {

using mo_fp8::kGroup;
using mo_fp8::ProductArgs;

enum Form { kFormRows, kFormFew, kFormColumns, kFormBoth, kFormWeight, kForms };
const char* const kFormNames[kForms] = {"rows", "few", "columns", "both", "weight"};
const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

// How the second operand's scales come: a byte or an fp32 number a block of 128 x 128, or a byte a row.
enum { kScaleBytes = MO_FP8_SCALE_E8M0, kScaleFloats = MO_FP8_SCALE_F32, kScaleRows = 2 };
const char* const kScaleNames[3] = {"bytes", "floats", "rows"};

// The tiles (mo_fp8.hip): edge, workgroups that fit a CU, and what the cost model knows of them on an MI355X,
// in us, for 16-bit outputs, 16-bit outputs with fp32 block scales, and fp32 outputs: a call's fixed part, what
// a further round of workgroups adds of it, and a step of 128 of the reduction with one workgroup on a CU and
// with all that fit. Fitted to 12 400 timed calls (110 shapes of 1 to 17 792 rows, every tile, 1 to 32
// splits, eight kinds of operands, replayed back to back). Of the launches timed for a shape, the one that these
// numbers choose takes 1 % longer than the fastest on average, 4 % at the ninetieth percentile, 29 % at worst (199
// rows of 3072 from 24576), a split call's time with the 2.4 us that kSumFixed counts for the host. Inputs that come
// from memory take longer than replays do: 3072 x 3072 fp32 from 1333 is 34 here and 44 in a program's trace.
struct Cost {
  double fixed, again, alone, together;
};
struct TileShape {
  const char* name;
  uint32_t edge, threads;
  int resident;
  Cost cost[3];  // [kCostNarrow ..]
};
enum { kCostNarrow, kCostFloats, kCostWide };
constexpr int kTiles = 3;
constexpr TileShape kTileShapes[kTiles] = {
    {"large", 256, 512, 1, {{6.2, 0.86, 1.10, 1.10}, {7.0, 0.79, 1.48, 1.48}, {6.4, 0.79, 2.27, 2.27}}},
    {"middle", 128, 256, 2, {{4.1, 0.63, 0.54, 0.91}, {4.5, 0.46, 0.78, 1.19}, {4.5, 0.19, 0.91, 1.64}}},
    {"small", 64, 256, 4, {{3.1, 0.31, 0.32, 0.92}, {3.2, 0.32, 0.37, 1.00}, {3.2, 0.19, 0.44, 1.21}}},
};
// The sum of a split call's planes: fixed (1.1 on the GPU; the launch takes the host 3.4, which calls this short
// wait for), a plane, a MB of planes.
constexpr double kSumFixed = 3.5, kSumPlane = 0.26, kSumMb = 0.32;
constexpr uint32_t kMaxSplits = 32, kMinSplitSteps = 2;
constexpr uint64_t kMaxPlanes = 1ull << 31;  // bytes

struct Module {
  hipModule_t module = nullptr;
  int cus = 0;
  hipFunction_t quantize[kForms][3] = {};
  hipFunction_t decode = nullptr, sum = nullptr;
  hipFunction_t product[kTiles][3][2][2] = {};  // [tile][scales][fp32 output][weight as stored]
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
    bool ok = get(&m.decode, "mo_fp8_decode_kernel") && get(&m.sum, "mo_fp8_plane_sum");
    for (int f = 0; f < kForms; ++f)
      for (int t = 0; t < 3; ++t)
        ok = ok && get(&m.quantize[f][t], std::string("mo_fp8_quantize_") + kFormNames[f] + "_" + kTypeNames[t]);
    for (int tile = 0; tile < kTiles; ++tile)
      for (int k = 0; k < 3; ++k)
        for (int wide = 0; wide < 2; ++wide)
          for (int trans = 0; trans < (k == kScaleRows ? 1 : 2); ++trans) {
            std::string name = std::string("mo_fp8_product_") + kTileShapes[tile].name + "_" + kScaleNames[k];
            if (trans || wide) name += std::string("_") + (trans ? "t" : "") + (wide ? "w" : "");
            ok = ok && get(&m.product[tile][k][wide][trans], name);
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
  // rows alone, fewer tiles than fill the CUs four at a time: 16 rows a workgroup
  if (form == kFormRows && div_up(rows, kGroup) * div_up(cols, kGroup) < 4ull * m.cus) form = kFormFew;
  return launch(m.quantize[form][dtype], div_up(rows, form == kFormFew ? 16 : kGroup) * div_up(cols, kGroup), 256, params, stream,
                "fp8 quantize launch");
}

// A product's launches: rows [row0, row0 + rows) on `tile`, the reduction in `splits` of `split_steps` groups.
struct Part {
  uint64_t row0, rows;
  int tile;
  uint32_t splits, split_steps;
};
struct Plan {
  int parts;
  Part part[2];
};

// Modelled time (us) of a call whose reduction is shared out over `splits` workgroups a tile, `per` steps each.
double cost_of(const TileShape& t, const Cost& c, uint64_t rows, uint64_t cols, uint32_t splits, uint32_t per, int cus) {
  const uint64_t each = div_up(div_up(rows, t.edge) * div_up(cols, t.edge) * splits, (uint64_t)cus);
  const uint64_t full = each / t.resident, left = each % t.resident;
  const uint32_t steps = (per + 1) & ~1u;  // the loop runs steps in pairs
  double step = (double)full * c.together;
  if (left) step += c.alone + (t.resident > 1 ? (c.together - c.alone) * (double)(left - 1) / (t.resident - 1) : 0.0);
  double us = c.fixed * (1 + c.again * (double)(full + (left > 0) - 1)) + steps * step;
  if (splits > 1) us += kSumFixed + kSumPlane * splits + kSumMb * (double)splits * (double)rows * (double)cols * 4e-6;
  return us;
}

// The cheapest tile and splits for `rows` rows from row0 on; *us: the modelled time.
Part part_of(uint64_t row0, uint64_t rows, uint64_t cols, uint32_t steps, int kind, int cus, double* us) {
  Part best{row0, rows, 0, 1, steps};
  *us = 0;
  for (int i = 0; i < kTiles; ++i) {
    const TileShape& t = kTileShapes[i];
    uint32_t tried = 0;
    for (uint32_t want = 1; want <= kMaxSplits; ++want) {
      if (want > 1 && (steps / want < kMinSplitSteps || want * rows * cols * 4 > kMaxPlanes)) break;
      const uint32_t per = (uint32_t)div_up(steps, want), splits = (uint32_t)div_up(steps, per);
      if (splits == tried) continue;
      tried = splits;
      const double c = cost_of(t, t.cost[kind], rows, cols, splits, per, cus);
      if (*us == 0 || c < *us) best = Part{row0, rows, i, splits, per}, *us = c;
    }
  }
  return best;
}

// One launch, or two: the rows that fill whole rounds of the CUs with large tiles, and the rest on what suits
// them. A last round that few tiles are left for costs as much as a full one (17792 rows of 3072 from 12288 are
// 840 tiles, 3.3 rounds).
Plan plan_of(uint64_t rows, uint64_t cols, uint32_t steps, int kind, int cus) {
  double whole;
  Plan plan{1, {part_of(0, rows, cols, steps, kind, cus, &whole), {}}};
  const TileShape& t = kTileShapes[0];
  const uint64_t tiles_m = div_up(rows, t.edge), tiles_n = div_up(cols, t.edge);
  const uint64_t rounds = tiles_m * tiles_n / (uint64_t)cus, fill = rounds * (uint64_t)cus / tiles_n;
  if (fill == 0 || fill >= tiles_m) return plan;
  double rest;
  const uint64_t head = fill * t.edge;
  const Part tail = part_of(head, rows - head, cols, steps, kind, cus, &rest);
  if (cost_of(t, t.cost[kind], head, cols, 1, steps, cus) + rest < whole)
    plan = Plan{2, {Part{0, head, 0, 1, steps}, tail}};
  return plan;
}

int cost_kind(int scales, uint32_t out_kind) {
  return out_kind == MO_DTYPE_F32 ? kCostWide : scales == kScaleFloats ? kCostFloats : kCostNarrow;
}

uint64_t plane_bytes(const Plan& p, uint64_t cols) {  // only the last part is split
  const Part& last = p.part[p.parts - 1];
  return last.splits > 1 ? align(last.splits * last.rows * cols * 4) : 0;
}

// `planes`: room for the plan's plane_bytes.
int product(const Module& m, const Plan& plan, const ProductArgs& whole, int scales, bool trans, uint64_t planes,
            uint64_t stream) {
  for (int i = 0; i < plan.parts; ++i) {
    const Part& part = plan.part[i];
    const TileShape& t = kTileShapes[part.tile];
    ProductArgs p = whole;
    p.a += part.row0 * p.a_pitch, p.a_scales += part.row0;
    p.out = (uint8_t*)p.out + part.row0 * p.n * kTypeBytes[p.out_kind];
    p.m = part.rows, p.splits = part.splits, p.split_steps = part.split_steps;
    p.planes = part.splits > 1 ? (float*)planes : nullptr;
    void* params[] = {&p};
    if (int rc = launch(m.product[part.tile][scales][p.out_kind == MO_DTYPE_F32][trans],
                        div_up(p.m, t.edge) * div_up(p.n, t.edge) * part.splits, t.threads, params, stream,
                        "fp8 product launch"))
      return rc;
    if (part.splits == 1) continue;
    if (int rc = launch(m.sum, div_up(p.m * p.n / 4, 256), 256, params, stream, "fp8 plane sum launch")) return rc;
  }
  return 0;
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

int check_output(uint64_t out, uint32_t dtype, uint64_t bias = 0, uint32_t bias_dtype = 0) {
  if (!out) return mo::set_error(MO_E_INVALID, "null output pointer");
  if (dtype > MO_DTYPE_F32) return mo::set_error(MO_E_INVALID, "unknown output type");
  if (out % 16 || bias % kTypeBytes[bias_dtype]) return mo::set_error(MO_E_INVALID, "misaligned output or bias pointer");
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

// A call's plan and its workspace: the operands it quantizes, then its planes.
struct Room {
  Plan plan;
  uint64_t operands, planes;
  uint64_t bytes() const { return operands + planes; }
};

Room room_of(uint32_t op, uint64_t rows, uint64_t in_f, uint64_t out_f, bool quantized, uint32_t scale_kind,
             uint32_t out_kind, int cus) {
  Room r = {};
  const uint64_t m = op == MO_FP8_WEIGHT ? out_f : rows, n = op == MO_FP8_FORWARD ? out_f : in_f;
  const uint64_t reduction = op == MO_FP8_FORWARD ? in_f : op == MO_FP8_BACKWARD ? out_f : rows;
  if (!quantized) {
    if (op == MO_FP8_FORWARD) r.operands = row_bytes(rows, in_f);
    if (op == MO_FP8_BACKWARD) r.operands = row_bytes(rows, out_f);
    if (op == MO_FP8_WEIGHT) r.operands = col_bytes(rows, out_f) + col_bytes(rows, in_f);
  }
  const int scales = op == MO_FP8_WEIGHT ? kScaleRows : (int)scale_kind;
  r.plan = plan_of(m, n, (uint32_t)div_up(reduction, kGroup), cost_kind(scales, out_kind), cus);
  r.planes = plane_bytes(r.plan, n);
  return r;
}

}  // namespace

extern "C" {

uint64_t mo_fp8_workspace_bytes(uint32_t op, uint64_t rows, uint32_t in_features, uint32_t out_features,
                                uint32_t quantized, uint32_t scale_kind, uint32_t out_dtype) {
  if (op > MO_FP8_WEIGHT || rows == 0 || rows >= (1ull << 31) || in_features == 0 || out_features == 0 ||
      in_features > (1u << 20) || out_features > (1u << 20) || scale_kind > MO_FP8_SCALE_F32 || out_dtype > MO_DTYPE_F32)
    return 0;
  uint64_t bytes = 0;
  const int rc = guarded([&]() -> int {
    Module m;
    if (int bad = load_module(&m)) return bad;
    bytes = room_of(op, rows, in_features, out_features, quantized != 0, scale_kind, out_dtype, m.cus).bytes();
    return 0;
  });
  return rc ? MO_FP8_NO_SIZE : bytes;
}

int mo_fp8_plan(uint64_t rows, uint32_t cols, uint32_t reduction, uint32_t scale_kind, uint32_t out_dtype, uint32_t cus,
                uint32_t* plan) {
  if (!plan) return mo::set_error(MO_E_INVALID, "null output pointer");
  if (rows == 0 || rows >= (1ull << 31) || cols == 0 || reduction == 0 || cus == 0)
    return mo::set_error(MO_E_INVALID, "empty shape, or too many rows");
  if (scale_kind > MO_FP8_SCALE_F32 || out_dtype > MO_DTYPE_F32) return mo::set_error(MO_E_INVALID, "unknown type");
  const Plan p = plan_of(rows, cols, (uint32_t)div_up(reduction, kGroup), cost_kind((int)scale_kind, out_dtype), (int)cus);
  for (int i = 0; i < 2; ++i) {
    const Part& part = p.part[i];
    const bool on = i < p.parts;
    plan[4 * i] = on ? (uint32_t)part.rows : 0, plan[4 * i + 1] = on ? kTileShapes[part.tile].edge : 0;
    plan[4 * i + 2] = on ? part.splits : 0, plan[4 * i + 3] = on ? part.split_steps : 0;
  }
  return 0;
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
    const uint32_t across = (uint32_t)div_up(cols, 8);
    const uint64_t total = rows * across;
    const mo::FastDiv f = mo::make_fastdiv(across);
    mo_fp8::Divisor chunks = {f.d, total + 255 < (1ull << 31) ? f.m : 0u, f.s};
    void* params[] = {&V, &pitch, &S, &scale_kind, &scale_row, &scale_col, &shift, &O, &dtype, &rows, &cols, &chunks};
    return launch(m.decode, div_up(total, 256), 256, params, stream, "fp8 decode launch");
  });
}

int mo_fp8_linear_forward(uint64_t x, uint64_t x_scales, uint32_t dtype, uint64_t rows, uint32_t in_features,
                          uint64_t row_stride, uint64_t w, uint64_t w_scale, uint32_t scale_kind,
                          uint32_t out_features, uint64_t bias, uint64_t y, uint32_t y_dtype, uint64_t workspace,
                          uint64_t workspace_bytes, uint64_t stream) {
  return guarded([&]() -> int {
    if (int rc = check_weight(w, w_scale, scale_kind, in_features, out_features)) return rc;
    if (int rc = check_operand(x, x_scales, dtype, rows, in_features, row_stride)) return rc;
    const bool wide_bias = y_dtype & MO_FP8_BIAS_F32;
    y_dtype &= ~(uint32_t)MO_FP8_BIAS_F32;
    const uint32_t bias_dtype = wide_bias ? (uint32_t)MO_DTYPE_F32 : y_dtype > MO_DTYPE_F32 ? 0 : y_dtype;
    if (int rc = check_output(y, y_dtype, bias, bias_dtype)) return rc;
    Module m;
    if (int rc = load_module(&m)) return rc;
    const Room room =
        room_of(MO_FP8_FORWARD, rows, in_features, out_features, x_scales != 0, scale_kind, y_dtype, m.cus);
    if (int rc = check_workspace(workspace, workspace_bytes, room.bytes())) return rc;
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
    p.b_scale_row = (uint32_t)div_up(in_features, kGroup), p.b_scale_col = 1;
    p.bias = (const void*)bias, p.bias_kind = bias_dtype, p.out = (void*)y, p.out_kind = y_dtype;
    p.m = rows, p.n = out_features, p.r = in_features;
    return product(m, room.plan, p, (int)scale_kind, false, workspace + room.operands, stream);
  });
}

int mo_fp8_linear_backward(uint64_t dy, uint64_t dy_scales, uint32_t dtype, uint64_t rows, uint32_t in_features,
                           uint32_t out_features, uint64_t row_stride, uint64_t w, uint64_t w_scale,
                           uint32_t scale_kind, uint64_t dx, uint32_t dx_dtype, uint64_t workspace,
                           uint64_t workspace_bytes, uint64_t stream) {
  return guarded([&]() -> int {
    if (int rc = check_weight(w, w_scale, scale_kind, in_features, out_features)) return rc;
    if (int rc = check_operand(dy, dy_scales, dtype, rows, out_features, row_stride)) return rc;
    if (int rc = check_output(dx, dx_dtype)) return rc;
    Module m;
    if (int rc = load_module(&m)) return rc;
    const Room room =
        room_of(MO_FP8_BACKWARD, rows, in_features, out_features, dy_scales != 0, scale_kind, dx_dtype, m.cus);
    if (int rc = check_workspace(workspace, workspace_bytes, room.bytes())) return rc;
    if (!dy_scales) {
      const uint64_t values = workspace, scales = workspace + align(rows * out_features);
      if (int rc = quantize(m, kFormRows, dy, dtype, rows, out_features, row_stride, values, scales, 0, 0, stream))
        return rc;
      dy = values, dy_scales = scales;
    }
    ProductArgs p = {};
    p.a = (const uint8_t*)dy, p.a_scales = (const uint8_t*)dy_scales, p.a_pitch = out_features;
    p.a_scale_pitch = (uint32_t)scale_pitch(rows);
    p.b = (const uint8_t*)w, p.b_scales = (const void*)w_scale, p.b_pitch = in_features;  // as stored
    p.b_scale_row = 1, p.b_scale_col = (uint32_t)div_up(in_features, kGroup);
    p.out = (void*)dx, p.out_kind = dx_dtype;
    p.m = rows, p.n = in_features, p.r = out_features;
    return product(m, room.plan, p, (int)scale_kind, true, workspace + room.operands, stream);
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
    if (int rc = check_output(dw, dw_dtype)) return rc;
    const uint64_t padded = div_up(rows, kGroup) * kGroup;
    if (padded * 256 >= (1ull << 31))  // 32-bit buffer offsets over a tile's rows
      return mo::set_error(MO_E_INVALID, "too many rows for one weight gradient (2^23 - 128 at most)");
    Module m;
    if (int rc = load_module(&m)) return rc;
    const Room room = room_of(MO_FP8_WEIGHT, rows, in_features, out_features, dy_scales != 0, MO_FP8_SCALE_E8M0,
                              dw_dtype, m.cus);
    if (int rc = check_workspace(workspace, workspace_bytes, room.bytes())) return rc;
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
    p.b_scale_col = in_features;  // one scale a row
    p.out = (void*)dw, p.out_kind = dw_dtype;
    p.m = out_features, p.n = in_features, p.r = (uint32_t)padded;
    return product(m, room.plan, p, kScaleRows, false, workspace + room.operands, stream);
  });
}

}  // extern "C"
