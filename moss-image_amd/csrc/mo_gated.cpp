// Host side of the gated activation and of activations in 8 bits (csrc/mo_gated.hip): argument checks and launches.
// C ABI: mo_gated_*, mo_keep_*.
#include "mo_block.h"
#include "mo_layout.h"
#include "mo_module.h"

extern "C" const unsigned char mo_gated_code[];

namespace {

const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

mo::Kernels& kernels() {
  static mo::Kernels k(mo_gated_code);
  return k;
}

int bad(const char* what) { return mo::set_error(MO_E_INVALID, what); }

// Four lanes for each 32 columns; false where the lanes are too many to count.
bool shares(uint64_t rows, uint32_t cols, uint32_t* lanes, mo_block::Divisor* by) {
  *lanes = (cols + 31) / 32 * 4;
  const mo::FastDiv f = mo::make_fastdiv(*lanes);
  *by = {f.d, f.m, f.s};
  return rows * *lanes < (1ull << 31) - 256;
}

int gated(const mo_gated_call* c, bool backward, uint64_t stream) {
  if (!c) return bad("null call");
  if (c->dtype > MO_DTYPE_F32) return bad("unknown element type");
  if (c->rows == 0 || c->rows >= (1ull << 31) || c->cols == 0 || c->cols >= (1u << 30)) return bad("no rows or columns, or too many");
  const uint32_t size = kTypeBytes[c->dtype];
  if (!c->up || !c->gate || !c->out || c->out % size) return bad("null or misaligned operands");
  const bool kept = c->up_exponents || c->gate_exponents;
  if (kept && (!backward || !c->up_exponents || !c->gate_exponents)) return bad("up and gate are both in 8 bits, backward, or neither");
  if (kept ? c->up % 8 || c->gate % 8 || c->values_stride % 8 : c->up % size || c->gate % size) return bad("misaligned operands");
  const bool keep = !backward && (c->kept_up || c->kept_gate);
  if (keep && (!c->kept_up || !c->kept_gate || !c->kept_up_exponents || !c->kept_gate_exponents || c->kept_up % 8 ||
               c->kept_gate % 8 || c->values_stride % 8))
    return bad("null or misaligned 8-bit outputs");
  if (backward && (!c->grad || c->grad % size || !c->out_gate || c->out_gate % size)) return bad("null or misaligned gradients");
  const uint64_t groups = (c->cols + 31) / 32;
  if (c->rows > 1 && ((!kept && (c->up_stride < c->cols || c->gate_stride < c->cols)) || c->out_stride < c->cols ||
                      (backward && c->grad_stride < c->cols) ||
                      ((kept || keep) && (c->values_stride < groups * 32 || c->exponents_stride < groups))))
    return bad("rows overlap");
  mo_block::GatedArgs a = {};
  a.up = (const void*)c->up, a.gate = (const void*)c->gate;
  a.up_exponents = (const uint8_t*)c->up_exponents, a.gate_exponents = (const uint8_t*)c->gate_exponents;
  a.grad = (const void*)c->grad, a.out = (void*)c->out, a.out_gate = (void*)c->out_gate;
  a.kept_up = (int8_t*)c->kept_up, a.kept_gate = (int8_t*)c->kept_gate;
  a.kept_up_exponents = (uint8_t*)c->kept_up_exponents, a.kept_gate_exponents = (uint8_t*)c->kept_gate_exponents;
  a.up_stride = c->up_stride, a.gate_stride = c->gate_stride, a.grad_stride = c->grad_stride, a.out_stride = c->out_stride;
  a.values_stride = c->values_stride, a.exponents_stride = c->exponents_stride;
  a.rows = (uint32_t)c->rows, a.cols = c->cols, a.silu = c->silu;
  if (!shares(c->rows, c->cols, &a.lanes, &a.by_lanes)) return bad("too many values");
  const bool eights = kept || keep, singly = c->cols % 8 != 0;
  auto name = [&]() {
    return std::string("mo_gated_") + (backward ? "backward_" : "forward_") + (kept ? "kept_" : keep ? "keep_" : "") +
           kTypeNames[c->dtype] + (singly ? "_odd" : "");
  };
  hipFunction_t kernel = nullptr;
  if (int rc = kernels().get(((backward * 2 + eights) * 3 + (int)c->dtype) * 2 + singly, name, &kernel)) return rc;
  void* params[] = {&a};
  const uint64_t items = c->rows * a.lanes;
  return mo::launch(kernel, (uint32_t)((items + 255) / 256), 1, 1, 256, stream, params, "gated activation launch");
}

int keep(uint64_t x, uint64_t values, uint64_t exponents, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t stride,
         bool restore, uint64_t stream) {
  if (!x || !values || !exponents) return bad("null pointer");
  if (dtype > MO_DTYPE_F32) return bad("unknown element type");
  if (rows == 0 || rows >= (1ull << 31) || cols == 0 || cols >= (1u << 30)) return bad("no rows or columns, or too many");
  if (x % kTypeBytes[dtype] || values % 8) return bad("misaligned pointer");
  if (rows > 1 && stride < cols) return bad("rows overlap");
  mo_block::KeepArgs a = {};
  a.x = (const void*)x, a.out = (void*)x, a.values = (int8_t*)values, a.exponents = (uint8_t*)exponents;
  a.stride = stride, a.rows = (uint32_t)rows, a.cols = cols, a.groups = (cols + 31) / 32;
  if (!shares(rows, cols, &a.lanes, &a.by_lanes)) return bad("too many values");
  const bool singly = cols % 8 != 0;
  auto name = [&]() {
    return std::string(restore ? "mo_keep_restore_" : "mo_keep_pack_") + kTypeNames[dtype] + (singly ? "_odd" : "");
  };
  hipFunction_t kernel = nullptr;
  if (int rc = kernels().get(24 + (restore * 3 + (int)dtype) * 2 + singly, name, &kernel)) return rc;
  void* params[] = {&a};
  const uint64_t items = rows * a.lanes;
  return mo::launch(kernel, (uint32_t)((items + 255) / 256), 1, 1, 256, stream, params, "8-bit activations launch");
}

}  // namespace

extern "C" {

int mo_gated_forward(const mo_gated_call* call, uint64_t stream) {
  return mo::guarded([&]() -> int { return gated(call, false, stream); });
}

int mo_gated_backward(const mo_gated_call* call, uint64_t stream) {
  return mo::guarded([&]() -> int { return gated(call, true, stream); });
}

int mo_keep_pack(uint64_t x, uint32_t dtype, uint64_t rows, uint32_t cols, uint64_t row_stride, uint64_t values,
                 uint64_t exponents, uint64_t stream) {
  return mo::guarded([&]() -> int { return keep(x, values, exponents, dtype, rows, cols, row_stride, false, stream); });
}

int mo_keep_restore(uint64_t values, uint64_t exponents, uint64_t out, uint32_t dtype, uint64_t rows, uint32_t cols,
                    uint64_t row_stride, uint64_t stream) {
  return mo::guarded([&]() -> int { return keep(out, values, exponents, dtype, rows, cols, row_stride, true, stream); });
}

}  // extern "C"
