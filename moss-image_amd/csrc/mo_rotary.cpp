// Host side of the rotary positions (csrc/mo_rotary.hip): argument checks, the choice of lanes and
// pairs a lane, launches. C ABI: mo_rotary_*.
#include "mo_rotary.h"

#include <hip/hip_runtime_api.h>

#include <map>
#include <mutex>
#include <string>

#include "../../include/moss_offload.h"
#include "mo_layout.h"

extern "C" const unsigned char mo_rotary_code[];

namespace mo {
int set_error(int code, const std::string& msg);
int set_hip_error(int e, const char* what);
}  // namespace mo

namespace {

using mo_rotary::Args;
using mo_rotary::kMaxBlocks;
using mo_rotary::kMaxHead;
using mo_rotary::Side;

const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};
const uint32_t kVecs[4] = {1, 2, 4, 8};

struct Module {
  hipModule_t module = nullptr;
  hipFunction_t turn[2][3][4] = {};  // [backward][type][kVecs index]; eight fp32 pairs have no kernel
  hipFunction_t weight_sum = nullptr, table = nullptr;
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
    if ((e = hipModuleLoadData(&m.module, mo_rotary_code)) != hipSuccess)
      return mo::set_hip_error((int)e, "hipModuleLoadData (rotary code object)");
    bool ok = (e = hipModuleGetFunction(&m.weight_sum, m.module, "mo_rotary_weight_sum")) == hipSuccess &&
              (e = hipModuleGetFunction(&m.table, m.module, "mo_rotary_table_kernel")) == hipSuccess;
    for (int back = 0; back < 2; ++back)
      for (int t = 0; t < 3; ++t)
        for (int v = 0; v < (t == MO_DTYPE_F32 ? 3 : 4); ++v) {
          const std::string name = std::string("mo_rotary_") + (back ? "backward_" : "forward_") + kTypeNames[t] + "_" +
                                   std::to_string(kVecs[v]);
          ok = ok && (e = hipModuleGetFunction(&m.turn[back][t][v], m.module, name.c_str())) == hipSuccess;
        }
    if (!ok) return mo::set_hip_error((int)e, "hipModuleGetFunction (rotary)");
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

bool fits(uint64_t pointer, uint32_t bytes) { return pointer % (bytes > 16 ? 16 : bytes) == 0; }

// Pairs a lane: the most that 16 bytes hold, halved until the rotary part and the rest of a head are
// whole numbers of them and every row that the lanes read or write by them is aligned to them.
uint32_t pick_vec(const mo_rotary_call& c) {
  const uint32_t size = kTypeBytes[c.dtype], table = kTypeBytes[c.table_dtype], weight = kTypeBytes[c.weight_dtype];
  uint32_t v = 16 / size;
  for (; v > 1; v /= 2) {
    bool ok = c.rotary_dim / 2 % v == 0 && (c.head_dim - c.rotary_dim) / 2 % v == 0 && fits(c.table, v * table) &&
              c.table_batch % v == 0;
    for (const mo_rotary_side& s : c.side) {
      if (!s.heads) continue;
      for (int64_t stride : {s.x_batch, s.x_token, s.x_head}) ok = ok && (!s.x || stride % v == 0);
      for (int64_t stride : {s.grad_batch, s.grad_token, s.grad_head}) ok = ok && (!s.grad || stride % v == 0);
      ok = ok && fits(s.x, v * size) && fits(s.grad, v * size) && fits(s.out, v * size) && fits(s.weight, v * weight);
    }
    if (ok) break;
  }
  return v;
}

mo_rotary::Divisor divisor(uint32_t d) {
  const mo::FastDiv f = mo::make_fastdiv(d);
  return {f.d, f.m, f.s};
}

struct Plan {
  uint32_t vec, lanes, blocks[2];
};

Plan plan_of(const mo_rotary_call& c, bool backward) {
  Plan p = {};
  p.vec = pick_vec(c);
  const uint32_t held = c.head_dim / 2 / p.vec + (c.head_dim / 2 % p.vec != 0);
  p.lanes = 1;
  while (p.lanes < held && p.lanes < 64) p.lanes *= 2;
  for (int i = 0; i < 2; ++i) {
    const uint64_t rows = (uint64_t)c.batch * c.tokens * c.side[i].heads;
    uint64_t blocks = div_up(rows * p.lanes, 256);
    if (backward && c.side[i].weight && blocks > kMaxBlocks) blocks = kMaxBlocks;
    p.blocks[i] = (uint32_t)blocks;
  }
  return p;
}

int check(const mo_rotary_call* c, bool backward) {
  if (!c) return mo::set_error(MO_E_INVALID, "null call");
  if (c->dtype > MO_DTYPE_F32 || c->table_dtype > MO_DTYPE_F32 || c->weight_dtype > MO_DTYPE_F32)
    return mo::set_error(MO_E_INVALID, "unknown element type");
  if (c->batch == 0 || c->tokens == 0) return mo::set_error(MO_E_INVALID, "no tokens");
  if (c->head_dim == 0 || c->head_dim % 2 || c->head_dim > kMaxHead)
    return mo::set_error(MO_E_INVALID, "head_dim must be even, 2 to 512");
  if (c->rotary_dim == 0 || c->rotary_dim % 2 || c->rotary_dim > c->head_dim)
    return mo::set_error(MO_E_INVALID, "rotary_dim must be even, 2 to head_dim");
  if (!c->table || c->table % kTypeBytes[c->table_dtype]) return mo::set_error(MO_E_INVALID, "null or misaligned table");
  if (!c->side[0].heads && !c->side[1].heads) return mo::set_error(MO_E_INVALID, "no heads");
  for (const mo_rotary_side& s : c->side) {
    if (!s.heads) continue;
    const uint32_t size = kTypeBytes[c->dtype];
    if (!s.out || s.out % size || s.x % size || s.grad % size) return mo::set_error(MO_E_INVALID, "null or misaligned heads");
    if (!backward && !s.x) return mo::set_error(MO_E_INVALID, "null input");
    if (backward && !s.grad) return mo::set_error(MO_E_INVALID, "null gradient");
    if (backward && s.weight && !s.x) return mo::set_error(MO_E_INVALID, "the norm's gradient needs the input");
    if (backward && s.weight && !s.weight_grad) return mo::set_error(MO_E_INVALID, "null weight gradient");
    if (s.weight % kTypeBytes[c->weight_dtype] || s.weight_grad % kTypeBytes[c->weight_dtype])
      return mo::set_error(MO_E_INVALID, "misaligned weight");
    if ((uint64_t)c->batch * c->tokens >= (1ull << 31) || (uint64_t)c->batch * c->tokens * s.heads >= (1ull << 31))
      return mo::set_error(MO_E_INVALID, "too many heads (2^31 or more)");
  }
  return 0;
}

uint64_t partial_bytes(const mo_rotary_call& c, const Plan& p) {
  uint64_t n = 0;
  for (int i = 0; i < 2; ++i)
    if (c.side[i].heads && c.side[i].weight) n += (uint64_t)p.blocks[i] * c.head_dim * 4;
  return (n + 255) & ~uint64_t(255);
}

int run(const mo_rotary_call* c, bool backward, uint64_t workspace, uint64_t workspace_bytes, uint64_t stream) {
  if (int rc = check(c, backward)) return rc;
  Module m;
  if (int rc = load_module(&m)) return rc;
  const Plan p = plan_of(*c, backward);
  const uint64_t needed = backward ? partial_bytes(*c, p) : 0;
  if (needed && (!workspace || workspace % 256 || workspace_bytes < needed))
    return mo::set_error(MO_E_INVALID, "workspace missing, misaligned or smaller than mo_rotary_workspace_bytes");
  Args a = {};
  uint64_t at = workspace;
  uint32_t most = 0;
  for (int i = 0; i < 2; ++i) {
    const mo_rotary_side& s = c->side[i];
    if (!s.heads) continue;
    Side& d = a.side[i];
    d.x = (const void*)s.x, d.grad = (const void*)s.grad, d.out = (void*)s.out, d.weight = (const void*)s.weight;
    d.x_batch = s.x_batch, d.x_token = s.x_token, d.x_head = s.x_head;
    d.g_batch = s.grad_batch, d.g_token = s.grad_token, d.g_head = s.grad_head;
    d.heads = s.heads, d.blocks = p.blocks[i], d.by_heads = divisor(s.heads);
    if (backward && s.weight) {
      d.partial = (float*)at, d.weight_grad = (void*)s.weight_grad;
      at += (uint64_t)d.blocks * c->head_dim * 4;
    }
    if (d.blocks > most) most = d.blocks;
  }
  a.table = (const void*)c->table, a.table_batch = c->table_batch;
  a.batch = c->batch, a.tokens = c->tokens, a.head_dim = c->head_dim, a.rotary_dim = c->rotary_dim;
  a.table_kind = c->table_dtype, a.weight_kind = c->weight_dtype, a.interleaved = c->interleaved, a.eps = c->eps;
  a.by_tokens = divisor(c->tokens);
  uint32_t lanes = p.lanes, vec = 0;
  while (kVecs[vec] != p.vec) ++vec;
  void* params[] = {&a, &lanes};
  hipError_t e = hipModuleLaunchKernel(m.turn[backward][c->dtype][vec], most, 2, 1, 256, 1, 1, 0, (hipStream_t)stream,
                                       params, nullptr);
  if (e != hipSuccess) return mo::set_hip_error((int)e, "rotary launch");
  if (needed) {
    void* sums[] = {&a};
    e = hipModuleLaunchKernel(m.weight_sum, (c->head_dim + 15) / 16, 2, 1, 1024, 1, 1, 0, (hipStream_t)stream, sums,
                              nullptr);
    if (e != hipSuccess) return mo::set_hip_error((int)e, "rotary weight sum launch");
  }
  return 0;
}

}  // namespace

extern "C" {

uint64_t mo_rotary_workspace_bytes(const mo_rotary_call* call) {
  uint64_t bytes = 0;
  const int rc = guarded([&]() -> int {
    if (int bad = check(call, true)) return bad;
    bytes = partial_bytes(*call, plan_of(*call, true));
    return 0;
  });
  return rc ? 0 : bytes;
}

int mo_rotary_forward(const mo_rotary_call* call, uint64_t stream) {
  return guarded([&]() -> int { return run(call, false, 0, 0, stream); });
}

int mo_rotary_backward(const mo_rotary_call* call, uint64_t workspace, uint64_t workspace_bytes, uint64_t stream) {
  return guarded([&]() -> int { return run(call, true, workspace, workspace_bytes, stream); });
}

int mo_rotary_table(uint64_t coordinates, uint64_t bands, uint64_t out, uint32_t dtype, uint64_t rows, uint32_t axes,
                    uint32_t n_bands, float amplitude, uint64_t stream) {
  return guarded([&]() -> int {
    if (!coordinates || !bands || !out) return mo::set_error(MO_E_INVALID, "null pointer");
    if (dtype > MO_DTYPE_F32) return mo::set_error(MO_E_INVALID, "unknown element type");
    if (rows == 0 || axes == 0 || n_bands == 0) return mo::set_error(MO_E_INVALID, "empty table");
    if (coordinates % 4 || bands % 4 || out % kTypeBytes[dtype]) return mo::set_error(MO_E_INVALID, "misaligned pointer");
    if (axes > (1u << 15) || n_bands > (1u << 15) || rows >= (1ull << 31))
      return mo::set_error(MO_E_INVALID, "table too large");
    const uint64_t blocks = div_up(rows * axes * n_bands, 256);
    if (blocks >= (1ull << 31)) return mo::set_error(MO_E_INVALID, "table too large");
    Module m;
    if (int rc = load_module(&m)) return rc;
    const void *C = (const void*)coordinates, *B = (const void*)bands;
    void* O = (void*)out;
    void* params[] = {&C, &B, &O, &rows, &axes, &n_bands, &amplitude, &dtype};
    const hipError_t e =
        hipModuleLaunchKernel(m.table, (uint32_t)blocks, 1, 1, 256, 1, 1, 0, (hipStream_t)stream, params, nullptr);
    return e == hipSuccess ? 0 : mo::set_hip_error((int)e, "rotary table launch");
  });
}

}  // extern "C"
