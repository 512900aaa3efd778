// Host side of the norms (csrc/mo_norm.hip): argument checks, how rows are shared out, launches. C ABI: mo_norm_*.
#include "mo_block.h"
#include "mo_layout.h"
#include "mo_module.h"

extern "C" const unsigned char mo_norm_code[];

namespace {

using mo_block::NormArgs;

const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

mo::Kernels& kernels() {
  static mo::Kernels k(mo_norm_code);
  return k;
}

uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// How a call's rows are shared out: `lanes` of 8 values (kIter times) a row, `per` rows side by side in a workgroup,
// `chunk` rows one after the other.
struct Plan {
  uint32_t lanes, per, chunk, iter, groups;
  uint64_t slots;  // backward: pairs of a group of rows and a sample that have a place for sums
};

// Whether every eight neighbouring values lie in a row and on the 4-byte grid: dim is a multiple of eight, and so on. Other calls have
// kernels in which each lane reads its eight at an address of its own, and the last of a row value by value (4608 rows of 2047 bfloat16
// 17.2 and 32.2 us, of 2048 10.9 and 17.2).
bool odd(const mo_norm_call& c) {
  const uint64_t size = kTypeBytes[c.dtype];
  uint64_t off = c.dim % 8;
  for (uint64_t p : {c.x_exponents ? 0 : c.x, c.grad, c.out}) off |= p % 4;
  if (c.rows > 1) off |= (c.x_exponents ? 0 : c.x_stride * size % 4) | c.grad_stride * size % 4;
  return off != 0;
}

Plan plan_of(const mo_norm_call& c, bool backward) {
  Plan p = {};
  const uint64_t held = div_up(c.dim, 8);
  // 8 values a lane up to 512 lanes, more past that; 5 to 7 waves of 8 values were slower than 3 or 4 of 16 (17792 rows of
  // 3072 bfloat16, forward and backward: 41.8 and 78.1 us against 37.1 and 74.6), 8 waves faster (4608 of 4096: 13.8 and 28.5
  // against 15.1 and 30.8)
  p.iter = held > 1024 ? 4 : held > 512 || (held > 256 && held <= 448) ? 2 : 1;
  p.lanes = (uint32_t)div_up(div_up(held, p.iter), 64) * 64;
  // rows of a wave four to a workgroup: 17792 of 256 7.4 and 23.3 us, one to a workgroup 10.2 and 26.1
  p.per = p.lanes == 64 ? 4 : 1;
  // Forward: enough workgroups for several on every CU (half as many: 4608 rows of 3072 14.8 us for 12.9; twice: 3584 17.9
  // for 14.5). Backward each leaves sums of dim values, so fewer: two a CU, or one where a workgroup is large (twice as many
  // of those: 4608 rows of 8192 58.9 us for 47.7, of 12288 102 for 92; half as many of the others: 17792 of 3072 92 for 74.6),
  // and of two rows at least (333 rows of 3072: 16.0 us for 12.0).
  const uint64_t most = !backward ? 1024 : p.lanes == 512 || p.iter == 4 || p.per > 1 ? 256 : 512;
  p.chunk = (uint32_t)div_up(c.rows, most * p.per);
  if (p.chunk > 1 || backward) p.chunk += p.chunk % 2;  // whole batches of two rows
  p.groups = (uint32_t)div_up(c.rows, p.chunk);
  p.slots = (uint64_t)p.groups + (c.samples ? c.samples - 1 : 0);
  return p;
}

uint32_t pitch_of(const mo_norm_call& c) { return (c.dim + 7) / 8 * 8; }
bool wants_sums(const mo_norm_call& c) { return c.weight_grad || c.bias_grad || c.scale_grad || c.shift_grad; }
bool wants_sample_sums(const mo_norm_call& c) { return c.samples > 1 && (c.weight_grad || c.bias_grad); }

uint64_t workspace_bytes(const mo_norm_call& c, const Plan& p) {
  uint64_t floats = 0;
  if (wants_sums(c)) floats += p.slots * 2 * pitch_of(c);
  if (wants_sample_sums(c)) floats += (uint64_t)c.samples * 2 * pitch_of(c);
  return (floats * 4 + 255) & ~uint64_t(255);
}

int check(const mo_norm_call* c, bool backward) {
  auto bad = [](const char* what) { return mo::set_error(MO_E_INVALID, what); };
  if (!c) return bad("null call");
  if (c->dtype > MO_DTYPE_F32 || c->weight_dtype > MO_DTYPE_F32 || c->scale_dtype > MO_DTYPE_F32)
    return bad("unknown element type");
  if (c->rows == 0 || c->rows >= (1ull << 31) || c->dim == 0 || c->dim > mo_block::kMaxDim)
    return bad("rows must be 1 to 2^31 - 1 and dim 1 to 16384");
  const uint32_t size = kTypeBytes[c->dtype];
  if (!c->x || !c->out || c->out % size) return bad("null or misaligned rows");
  if (c->x_exponents ? !backward || c->x % 8 != 0 : c->x % size != 0) return bad("misaligned input");
  if (c->rows > 1 && !c->x_exponents && c->x_stride < c->dim) return bad("rows of the input overlap");
  const bool modulated = c->scale || c->shift;
  if (modulated != (c->samples != 0)) return bad("samples go with a scale or a shift");
  if (c->samples >= (1u << 16)) return bad("too many samples (2^16 or more)");
  if (c->cu ? !modulated || c->cu % 8 != 0 : modulated && c->rows % c->samples != 0)
    return bad("samples' rows must be given, or the same number for each");
  for (uint64_t p : {c->weight, c->bias, c->weight_grad, c->bias_grad})
    if (p % kTypeBytes[c->weight_dtype]) return bad("misaligned weight");
  for (uint64_t p : {c->scale, c->shift, c->scale_grad, c->shift_grad})
    if (p % kTypeBytes[c->scale_dtype]) return bad("misaligned modulation");
  if (c->stats % 8) return bad("misaligned statistics");  // read in pairs
  if (!backward) {
    if ((c->kept != 0) != (c->kept_exponents != 0) || c->kept % 8) return bad("both the 8-bit values and their exponents");
    return 0;
  }
  if (!c->grad || c->grad % size || !c->stats) return bad("the gradient and the forward pass's statistics are needed");
  if (c->rows > 1 && c->grad_stride < c->dim) return bad("rows of the gradient overlap");
  if ((c->weight_grad && !c->weight) || (c->bias_grad && !c->bias) || (c->scale_grad && !c->scale) ||
      (c->shift_grad && !c->shift))
    return bad("a gradient of what is not there");
  return 0;
}

int run(const mo_norm_call* c, bool backward, uint64_t workspace, uint64_t bytes, uint64_t stream) {
  if (int rc = check(c, backward)) return rc;
  const Plan p = plan_of(*c, backward);
  const uint64_t needed = backward ? workspace_bytes(*c, p) : 0;
  if (needed && (!workspace || workspace % 256 || bytes < needed))
    return mo::set_error(MO_E_INVALID, "workspace missing, misaligned or smaller than mo_norm_workspace_bytes");
  NormArgs a = {};
  a.x = (const void*)c->x, a.x_exponents = (const uint8_t*)c->x_exponents, a.grad = (const void*)c->grad;
  a.out = (void*)c->out, a.stats = (float*)c->stats;
  a.weight = (const void*)c->weight, a.bias = (const void*)c->bias;
  a.scale = (const void*)c->scale, a.shift = (const void*)c->shift;
  a.cu = (const int64_t*)c->cu;
  if (!backward) a.kept = (int8_t*)c->kept, a.kept_exponents = (uint8_t*)c->kept_exponents;
  a.x_stride = c->rows > 1 ? c->x_stride : c->dim, a.grad_stride = c->rows > 1 ? c->grad_stride : c->dim;
  a.scale_stride = c->scale_stride, a.shift_stride = c->shift_stride;
  a.rows = (uint32_t)c->rows, a.dim = c->dim, a.samples = c->samples;
  a.groups = (c->dim + 31) / 32, a.pitch = pitch_of(*c);
  a.lanes = p.lanes, a.per = p.per, a.chunk = p.chunk;
  a.weight_kind = c->weight_dtype, a.scale_kind = c->scale_dtype, a.layer = c->layer, a.eps = c->eps;
  const uint32_t share = c->samples && !c->cu ? (uint32_t)(c->rows / c->samples) : 1;
  const mo::FastDiv f = mo::make_fastdiv(share);
  a.by_share = {f.d, f.m, f.s};
  if (backward) {
    a.weight_grad = (void*)c->weight_grad, a.bias_grad = (void*)c->bias_grad;
    a.scale_grad = (void*)c->scale_grad, a.shift_grad = (void*)c->shift_grad;
    if (wants_sums(*c)) a.partial = (float*)workspace;
    if (wants_sample_sums(*c)) a.sample_sums = (float*)workspace + p.slots * 2 * a.pitch;
  }
  const bool eights = backward ? a.x_exponents != nullptr : a.kept != nullptr, singly = odd(*c);
  auto name = [&]() {
    return std::string("mo_norm_") + (backward ? "backward_" : "forward_") + (!eights ? "" : backward ? "kept_" : "keep_") +
           kTypeNames[c->dtype] + "_" + std::to_string(p.iter) + (singly ? "_odd" : "");
  };
  const int id = ((backward * 2 + eights) * 3 + (int)c->dtype) * 6 + p.iter / 2 * 2 + singly;
  hipFunction_t kernel = nullptr;
  if (int rc = kernels().get(id, name, &kernel)) return rc;
  void* params[] = {&a};
  if (int rc = mo::launch(kernel, (uint32_t)div_up(p.groups, p.per), 1, 1, p.lanes * p.per, stream, params, "norm launch"))
    return rc;
  if (!a.partial) return 0;
  if (int rc = kernels().get(72, [] { return "mo_norm_sums"; }, &kernel)) return rc;
  if (int rc = mo::launch(kernel, (c->dim + 15) / 16, c->samples ? c->samples : 1, 1, 1024, stream, params, "norm sums launch"))
    return rc;
  if (!a.sample_sums) return 0;
  if (int rc = kernels().get(73, [] { return "mo_norm_sample_sums"; }, &kernel)) return rc;
  return mo::launch(kernel, (c->dim + 255) / 256, 1, 1, 256, stream, params, "norm sums launch");
}

}  // namespace

extern "C" {

uint64_t mo_norm_workspace_bytes(const mo_norm_call* call) {
  uint64_t bytes = 0;
  const int rc = mo::guarded([&]() -> int {
    if (int bad = check(call, true)) return bad;
    bytes = workspace_bytes(*call, plan_of(*call, true));
    return 0;
  });
  return rc ? 0 : bytes;
}

int mo_norm_forward(const mo_norm_call* call, uint64_t stream) {
  return mo::guarded([&]() -> int { return run(call, false, 0, 0, stream); });
}

int mo_norm_backward(const mo_norm_call* call, uint64_t workspace, uint64_t workspace_bytes, uint64_t stream) {
  return mo::guarded([&]() -> int { return run(call, true, workspace, workspace_bytes, stream); });
}

}  // extern "C"
