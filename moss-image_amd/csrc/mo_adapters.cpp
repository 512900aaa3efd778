// Host side of the low-rank adapters (csrc/mo_adapters.hip): argument checks, workspaces, launches. C ABI: mo_adapters_*.
#include "mo_adapters.h"

#include "mo_layout.h"
#include "mo_module.h"

extern "C" const unsigned char mo_adapters_code[];

namespace {

using mo_adapters::Requests;

const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

// Workgroups that a launch aims at: four, four and three for each of 256 CUs.
constexpr uint64_t kShrinkGroups = 1024, kExpandGroups = 1024, kOuterGroups = 768;

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
  if (c->requests == 0 || c->requests >= (1u << 16) || c->adapters == 0 || c->adapters >= (1u << 15))
    return bad("requests must be 1 to 2^16 - 1 and adapters 1 to 2^15 - 1");
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

uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t round_up(uint64_t a, uint64_t b) { return div_up(a, b) * b; }
template <class N>
N between(N low, N value, N high) { return value < low ? low : value > high ? high : value; }

// Rows a tile and splits of the features of a shrink. Short requests take tiles of 16 rows, whose other rows would be
// empty; the features are shared out until there are some workgroups for every CU, 256 features each at least.
struct ShrinkPlan {
  uint32_t ranks, tiles, splits, span;
  uint64_t slots;
};
ShrinkPlan shrink_plan(const mo_adapters_call& c, uint32_t features) {
  ShrinkPlan p = {};
  p.ranks = c.rank <= 16 ? 1 : c.rank <= 32 ? 2 : c.rank <= 64 ? 4 : 8;
  p.tiles = p.ranks < 8 && c.rows >= 32ull * c.requests ? 2 : 1;
  const uint64_t tiles = div_up(c.rows, p.tiles * 16);
  const uint64_t splits = between<uint64_t>(1, div_up(kShrinkGroups, tiles), 8);
  p.span = (uint32_t)round_up(div_up(features, splits), 256);
  p.splits = (uint32_t)div_up(features, p.span);
  p.slots = tiles + c.requests + 1;
  return p;
}

// Rows a tile and columns a wave of an expand: as many as leave some workgroups for every CU.
struct ExpandPlan {
  uint32_t rank, tiles, cols;
  uint64_t slots;
};
ExpandPlan expand_plan(const mo_adapters_call& c, uint32_t features) {
  ExpandPlan p = {};
  p.rank = c.rank <= 16 ? 16 : c.rank <= 32 ? 32 : c.rank <= 64 ? 64 : 128;
  p.tiles = p.rank < 128 && c.rows >= 64ull * c.requests ? 4 : 1;
  const uint64_t tiles = div_up(c.rows, p.tiles * 16);
  p.cols = (uint32_t)round_up(between<uint64_t>(1, tiles * features / (4 * kExpandGroups), 512), 32);
  p.slots = tiles + c.requests + 1;
  return p;
}

// Splits of the rows of a weight's gradient: some workgroups for every CU again, 128 rows each at least.
void share_rows(const mo_adapters_call& c, mo_adapters::Side* side, uint32_t cols) {
  side->cols = cols;
  side->tiles = (uint32_t)div_up(cols, mo_adapters::kOuterCols);
  const uint64_t used = c.adapters < c.requests ? c.adapters : c.requests;
  uint64_t splits = div_up(kOuterGroups, side->tiles * used);
  splits = between<uint64_t>(1, splits, div_up(c.rows, 128));
  if (splits > mo_adapters::kMaxSplits) splits = mo_adapters::kMaxSplits;
  side->span = (uint32_t)round_up(div_up(c.rows, splits), 32);
  side->splits = (uint32_t)div_up(c.rows, side->span);
}

// Where what a call needs for itself lies in its workspace.
struct Room {
  uint64_t back, planes, turned_a, turned_b, da, db, bytes;  // offsets
};
Room room_of(const mo_adapters_call& c, bool backward) {
  Room r = {};
  auto take = [&](uint64_t bytes) {
    const uint64_t at = r.bytes;
    r.bytes += round_up(bytes, 256);
    return at;
  };
  const uint64_t between_bytes = c.rows * c.rank * 4, size = kTypeBytes[c.dtype];
  if (!backward) {
    const ShrinkPlan p = shrink_plan(c, c.in_features);
    if (p.splits > 1) r.planes = take(p.splits * between_bytes);
    return r;
  }
  if (c.dx || c.da) {
    const ShrinkPlan p = shrink_plan(c, c.out_features);
    r.back = take(between_bytes);
    if (p.splits > 1) r.planes = take(p.splits * between_bytes);
    r.turned_b = take((uint64_t)c.adapters * c.rank * c.out_features * size);
  }
  if (c.dx) r.turned_a = take((uint64_t)c.adapters * c.rank * c.in_features * size);
  mo_adapters::Side side = {};
  if (c.da) {
    share_rows(c, &side, c.in_features);
    if (side.splits > 1) r.da = take(4ull * side.splits * c.adapters * c.rank * c.in_features);
  }
  if (c.db) {
    share_rows(c, &side, c.out_features);
    if (side.splits > 1) r.db = take(4ull * side.splits * c.adapters * c.rank * c.out_features);
  }
  return r;
}

int start(const std::string& name, uint64_t gx, uint64_t gy, uint64_t gz, void* args, uint64_t stream) {
  if (gx >= (1ull << 31) || gy >= (1u << 16) || gz > (1u << 16)) return mo::set_error(MO_E_INVALID, "too many values");
  hipFunction_t kernel;
  if (int rc = kernels().get("mo_adapters_" + name, &kernel)) return rc;
  void* params[] = {args};
  return mo::launch(kernel, (uint32_t)gx, (uint32_t)gy, (uint32_t)gz, 256, stream, params, "adapters launch");
}

int shrink(const mo_adapters_call& c, const Requests& by, uint64_t x, uint64_t stride, uint64_t w, uint32_t features, uint64_t to,
           uint64_t planes, bool scaled, uint64_t stream) {
  const ShrinkPlan p = shrink_plan(c, features);
  mo_adapters::Shrink a = {};
  a.by = by, a.x = (const void*)x, a.w = (const void*)w, a.to = (float*)(p.splits > 1 ? planes : to);
  a.x_stride = stride, a.features = features, a.span = p.span, a.scaled = scaled;
  return start(std::string("shrink_") + kTypeNames[c.dtype] + "_" + std::to_string(p.ranks) + "_" + std::to_string(p.tiles),
               p.slots, p.splits, 1, &a, stream);
}

// `splits` > 1: h's, with their sum left at `h`.
int expand(const mo_adapters_call& c, const Requests& by, uint64_t h, uint64_t planes, uint32_t splits, uint64_t v, uint64_t base,
           uint64_t stride, uint64_t to, uint32_t features, bool scaled, uint64_t stream) {
  const ExpandPlan p = expand_plan(c, features);
  mo_adapters::Expand a = {};
  a.by = by, a.h = (const float*)(splits > 1 ? planes : h), a.h_sum = splits > 1 ? (float*)h : nullptr;
  a.v = (const void*)v, a.base = (const void*)base, a.to = (void*)to, a.base_stride = stride;
  a.features = features, a.splits = splits, a.cols = p.cols, a.scaled = scaled;
  return start(std::string("expand_") + kTypeNames[c.dtype] + "_" + std::to_string(p.rank) + "_" + std::to_string(p.tiles),
               p.slots, div_up(features, 4 * p.cols), 1, &a, stream);
}

int run(const mo_adapters_call* call, bool backward, uint64_t workspace, uint64_t bytes, uint64_t stream) {
  if (int rc = check(call, backward)) return rc;
  const mo_adapters_call& c = *call;
  const Room room = room_of(c, backward);
  if (room.bytes && (!workspace || workspace % 256 || bytes < room.bytes))
    return mo::set_error(MO_E_INVALID, "workspace missing, misaligned or smaller than mo_adapters_workspace_bytes");
  Requests by = {};
  by.cu = (const int64_t*)c.cu, by.index = (const int64_t*)c.index, by.scale = (const float*)c.scale, by.factor = c.factor;
  by.rows = (uint32_t)c.rows, by.requests = c.requests, by.adapters = c.adapters, by.rank = c.rank;
  by.share = c.cu ? 0 : (uint32_t)(c.rows / c.requests);
  const uint64_t planes = workspace + room.planes;
  if (!backward) {
    if (int rc = shrink(c, by, c.x, c.x_stride, c.a, c.in_features, c.hidden, planes, false, stream)) return rc;
    return expand(c, by, c.hidden, planes, shrink_plan(c, c.in_features).splits, c.b, c.result, c.result_stride, c.y,
                  c.out_features, true, stream);
  }
  const uint64_t back = workspace + room.back;
  const char* type = kTypeNames[c.dtype];
  if (c.dx || c.da) {
    mo_adapters::Turn t = {};
    auto side = [&](int i, uint64_t from, uint64_t to, uint32_t rows, uint32_t cols) {
      t.from[i] = (const void*)from, t.to[i] = (void*)to, t.rows[i] = rows, t.cols[i] = cols;
      t.tiles[i] = (uint32_t)(div_up(rows, 32) * div_up(cols, 32));
    };
    side(0, c.b, workspace + room.turned_b, c.out_features, c.rank);
    if (c.dx) side(1, c.a, workspace + room.turned_a, c.rank, c.in_features);
    if (int rc = start(std::string("turn_") + type, (uint64_t)t.tiles[0] + t.tiles[1], c.adapters, 1, &t, stream)) return rc;
    const uint32_t splits = shrink_plan(c, c.out_features).splits;
    if (int rc = shrink(c, by, c.grad, c.grad_stride, workspace + room.turned_b, c.out_features, back, planes, true, stream))
      return rc;
    if (c.dx) {
      if (int rc = expand(c, by, back, planes, splits, workspace + room.turned_a, c.add, c.add_stride, c.dx, c.in_features, false,
                          stream))
        return rc;
    } else if (splits > 1) {
      hipFunction_t kernel;
      if (int rc = kernels().get("mo_adapters_sum", &kernel)) return rc;
      const float* from = (const float*)planes;
      float* to = (float*)back;
      uint64_t count = c.rows * c.rank;
      uint32_t parts = splits;
      void* params[] = {&from, &to, &count, &parts};
      if (int rc = mo::launch(kernel, (uint32_t)div_up(count, 256), 1, 1, 256, stream, params, "adapters launch")) return rc;
    }
  }
  if (!c.da && !c.db) return 0;
  mo_adapters::Outer o = {};
  o.by = by;
  if (c.da) {
    mo_adapters::Side& s = o.side[0];
    share_rows(c, &s, c.in_features);
    s.wide = (const void*)c.x, s.exponents = (const uint8_t*)c.x_exponents, s.narrow = (const float*)back;
    s.planes = (float*)(workspace + room.da), s.to = (void*)c.da, s.stride = c.x_stride, s.groups = (c.in_features + 31) / 32;
  }
  if (c.db) {
    mo_adapters::Side& s = o.side[1];
    share_rows(c, &s, c.out_features);
    s.wide = (const void*)c.grad, s.narrow = (const float*)c.hidden, s.planes = (float*)(workspace + room.db), s.to = (void*)c.db;
    s.stride = c.grad_stride, s.turned = 1, s.scaled = 1;
  }
  const uint32_t ranks = c.rank <= 16 ? 1 : c.rank <= 32 ? 2 : 4;
  const uint32_t most = o.side[0].splits > o.side[1].splits ? o.side[0].splits : o.side[1].splits;
  if (int rc = start(std::string("outer_") + type + "_" + std::to_string(ranks), (uint64_t)o.side[0].tiles + o.side[1].tiles, most,
                     (uint64_t)c.adapters * div_up(c.rank, ranks * 16), &o, stream))
    return rc;
  if (most <= 1) return 0;
  const uint64_t size = (uint64_t)c.rank * (c.in_features > c.out_features ? c.in_features : c.out_features);
  return start(std::string("join_") + type, div_up(size, 1024), c.adapters, 2, &o, stream);
}

}  // namespace

extern "C" {

uint64_t mo_adapters_workspace_bytes(const mo_adapters_call* call, uint32_t backward) {
  uint64_t bytes = 0;
  const int rc = mo::guarded([&]() -> int {
    if (int bad = check(call, backward != 0)) return bad;
    bytes = room_of(*call, backward != 0).bytes;
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
