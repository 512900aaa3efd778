// Host side of the low-rank adapters (csrc/mo_adapters.hip): argument checks, workspaces, launches. C ABI: mo_adapters_*.
#include "mo_adapters.h"

#include "mo_layout.h"
#include "mo_module.h"

extern "C" const unsigned char mo_adapters_code[];

namespace {

using mo_adapters::Args;

const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

mo::Kernels& kernels() {
  static mo::Kernels k(mo_adapters_code);
  return k;
}

int check(const mo_adapters_call* c, bool backward) {
  auto bad = [](const char* what) { return mo::set_error(MO_E_INVALID, what); };
  if (!c) return bad("null call");
  if (c->dtype > MO_DTYPE_F32) return bad("unknown element type");
  const uint32_t size = kTypeBytes[c->dtype];
  if (c->rows == 0 || c->rows >= (1ull << 31) - 65536) return bad("no rows, or too many");
  if (c->in_features == 0 || c->in_features > (1u << 20) || c->out_features == 0 || c->out_features > (1u << 20))
    return bad("features must be 1 to 2^20");
  if (c->rank == 0 || c->rank > mo_adapters::kMaxRank) return bad("rank must be 1 to 128");
  if (c->requests == 0 || c->requests >= (1u << 16) || c->adapters == 0 || c->adapters >= (1u << 16))
    return bad("requests and adapters must be 1 to 2^16 - 1");
  if (!c->index && c->adapters != 1 && c->adapters != c->requests) return bad("an index is needed: requests are not adapters");
  if (!c->cu && c->rows % c->requests) return bad("requests' rows must be given, or the same number for each");
  if (c->cu % 8 || c->index % 8 || c->scale % 4 || c->hidden % 4) return bad("misaligned pointer");
  if ((!c->x && (!backward || c->da)) || !c->a || !c->b || c->a % size || c->b % size || !c->hidden) return bad("null or misaligned operands");
  if (c->x_exponents ? !backward || c->x % 8 != 0 : c->x % size != 0) return bad("misaligned input");
  const bool many = c->rows > 1;
  if (many && c->x && !c->x_exponents && c->x_stride < c->in_features) return bad("rows of the input overlap");
  if (!backward) {
    if (!c->result || !c->y || c->result % size || c->y % size) return bad("null or misaligned result");
    if (many && c->result_stride < c->out_features) return bad("rows of the result overlap");
    return 0;
  }
  if (!c->grad || c->grad % size || c->add % size || c->dx % size || c->da % size || c->db % size)
    return bad("null or misaligned gradients");
  if (!c->dx && !c->da && !c->db) return bad("no gradient is asked for");
  if (many && (c->grad_stride < c->out_features || (c->add && c->add_stride < c->in_features))) return bad("rows of a gradient overlap");
  return 0;
}

uint64_t workspace_bytes(const mo_adapters_call& c, bool backward) {
  return backward ? (c.rows * c.rank * 4 + 255) & ~uint64_t(255) : 0;
}

int launch(const mo_adapters_call* c, Args& a, const char* what, uint64_t items, uint32_t per, uint64_t stream) {
  const uint64_t blocks = (items + per - 1) / per;
  if (blocks >= (1ull << 31)) return mo::set_error(MO_E_INVALID, "too many values");
  hipFunction_t kernel;
  if (int rc = kernels().get(std::string("mo_adapters_") + what + "_" + kTypeNames[c->dtype], &kernel)) return rc;
  void* params[] = {&a};
  return mo::launch(kernel, (uint32_t)blocks, 1, 1, 256, stream, params, "adapters launch");
}

int run(const mo_adapters_call* c, bool backward, uint64_t workspace, uint64_t bytes, uint64_t stream) {
  if (int rc = check(c, backward)) return rc;
  const uint64_t needed = workspace_bytes(*c, backward);
  if (needed && (!workspace || workspace % 256 || bytes < needed))
    return mo::set_error(MO_E_INVALID, "workspace missing, misaligned or smaller than mo_adapters_workspace_bytes");
  Args a = {};
  a.x = (const void*)c->x, a.x_exponents = (const uint8_t*)c->x_exponents;
  a.result = (const void*)c->result, a.y = (void*)c->y, a.a = (const void*)c->a, a.b = (const void*)c->b;
  a.scale = (const float*)c->scale, a.cu = (const int64_t*)c->cu, a.index = (const int64_t*)c->index;
  a.hidden = (float*)c->hidden, a.grad = (const void*)c->grad, a.add = (const void*)c->add;
  a.dx = (void*)c->dx, a.da = (void*)c->da, a.db = (void*)c->db, a.back = (float*)workspace;
  a.x_stride = c->x_stride, a.result_stride = c->result_stride, a.grad_stride = c->grad_stride, a.add_stride = c->add_stride;
  a.rows = (uint32_t)c->rows, a.requests = c->requests, a.adapters = c->adapters, a.rank = c->rank;
  a.in = c->in_features, a.out = c->out_features, a.groups = (c->in_features + 31) / 32;
  a.factor = c->factor;
  const mo::FastDiv f = mo::make_fastdiv(c->cu ? 1 : (uint32_t)(c->rows / c->requests));
  a.by_share = {f.d, f.m, f.s};
  const uint64_t values = c->rows * c->rank;
  if (!backward) {
    if (int rc = launch(c, a, "hidden", values, 4, stream)) return rc;
    return launch(c, a, "y", c->rows * c->out_features, 256, stream);
  }
  if (c->dx || c->da)
    if (int rc = launch(c, a, "back", values, 4, stream)) return rc;
  const uint64_t weights = (uint64_t)c->adapters * c->rank;
  if (c->dx)
    if (int rc = launch(c, a, "dx", c->rows * c->in_features, 256, stream)) return rc;
  if (c->da)
    if (int rc = launch(c, a, "da", weights * c->in_features, 256, stream)) return rc;
  if (c->db)
    if (int rc = launch(c, a, "db", weights * c->out_features, 256, stream)) return rc;
  return 0;
}

}  // namespace

extern "C" {

uint64_t mo_adapters_workspace_bytes(const mo_adapters_call* call, uint32_t backward) {
  uint64_t bytes = 0;
  const int rc = mo::guarded([&]() -> int {
    if (int bad = check(call, backward != 0)) return bad;
    bytes = workspace_bytes(*call, backward != 0);
    return 0;
  });
  return rc ? 0 : bytes;
}

int mo_adapters_forward(const mo_adapters_call* call, uint64_t workspace, uint64_t workspace_bytes, uint64_t stream) {
  return mo::guarded([&]() -> int { return run(call, false, workspace, workspace_bytes, stream); });
}

int mo_adapters_backward(const mo_adapters_call* call, uint64_t workspace, uint64_t workspace_bytes, uint64_t stream) {
  return mo::guarded([&]() -> int { return run(call, true, workspace, workspace_bytes, stream); });
}

}  // extern "C"
