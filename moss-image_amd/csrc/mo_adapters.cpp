// Host side of the low-rank adapters (csrc/mo_adapters.hip): argument checks, workspaces, launches. C ABI: mo_adapters_*.
#include "mo_adapters.h"

#include "mo_layout.h"
#include "mo_module.h"

extern "C" const unsigned char mo_adapters_code[];

namespace {

using mo_adapters::Requests;

const char* const kTypeNames[3] = {"f16", "bf16", "f32"};  // by MO_DTYPE_*
constexpr uint32_t kTypeBytes[3] = {2, 2, 4};

// Workgroups that a launch aims at: an expand has three on a CU at a time, and many rounds leave no CU waiting long (half or twice
// as many: the same within 2 %).
constexpr uint64_t kExpandGroups = 4096, kOuterGroups = 384;

mo::Kernels& kernels() {
  static mo::Kernels k(mo_adapters_code);
  return k;
}

int check(const mo_adapters_call* c, bool backward) {
  auto bad = [](const char* what) { return mo::set_error(MO_E_INVALID, what); };
  if (!c) return bad("null call");
  if (c->dtype > MO_DTYPE_F32) return bad("unknown element type");
  const uint32_t size = kTypeBytes[c->dtype];
  // a lane's offsets from its wave's address have 31 bits: 31 rows of the tokens, and a whole matrix of an adapter
  if (c->rows == 0 || c->rows >= mo_adapters::kMaxRows) return bad("rows must be 1 to 2^26 - 1");
  if (c->rows > 1 && (c->x_stride > mo_adapters::kMaxStride || c->result_stride > mo_adapters::kMaxStride ||
                      c->grad_stride > mo_adapters::kMaxStride || c->add_stride > mo_adapters::kMaxStride))
    return bad("rows are more than 2^22 elements apart");
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

// The distance between rows; of one row, its length.
uint64_t stride_of(const mo_adapters_call& c, uint64_t stride, uint32_t features) { return c.rows > 1 ? stride : features; }

uint64_t div_up(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t round_up(uint64_t a, uint64_t b) { return div_up(a, b) * b; }
template <class N>
N between(N low, N value, N high) { return value < low ? low : value > high ? high : value; }

// Whether every eight neighbouring values lie in a row and on the 4-byte grid: features and rank are multiples of eight, and so on.
// Other calls have kernels in which each lane reads its eight at an address of its own, and the last of a row value by value (bfloat16, 4608
// rows of 3072 to 8192 both ways: ranks 4 and 12 196 and 205 us, 8 and 16 114 and 118; 16 ranks of 3071 features 200).
bool odd(const mo_adapters_call& c) {
  const uint64_t size = kTypeBytes[c.dtype];
  uint64_t off = (c.in_features | c.out_features | c.rank) % 8;
  for (uint64_t p : {c.x_exponents ? 0 : c.x, c.result, c.y, c.a, c.b, c.grad, c.add, c.dx, c.da, c.db}) off |= p % 4;
  if (c.rows > 1)
    for (uint64_t s : {c.x_exponents ? 0 : c.x_stride, c.result_stride, c.grad_stride, c.add_stride}) off |= s * size % 4;
  return off != 0;
}

// Rows a tile and splits of the features of a shrink. Tiles of 128 rows, which share the weight, where they and the splits
// make a workgroup for every CU (tiles of 16 and of 128 in a call, us: 4608 rows of 16384, 16 ranks 60.4 and 47.6; 17792 rows of 8192,
// 64 ranks 222 and 146; 1333 rows of 3072, 16 ranks 14.8 and 16.6; 1333 of 8192, 64 ranks 36.3 and 46.1); not for short requests,
// whose other rows would be empty. Splits as long as all workgroups are on the GPU at once (past that, a few that
// come late cost as much as all others: twice as many for 16 ranks, 4608 rows of 16384, 47.3 us for 42.5), 512 features each at
// least for tiles of 128, 1024 for those of 16, and up to 16.
struct ShrinkPlan {
  uint32_t ranks, rows, splits, span;
  uint64_t slots;
};
ShrinkPlan shrink_plan(const mo_adapters_call& c, uint32_t features) {
  ShrinkPlan p = {};
  p.ranks = c.rank <= 16 ? 1 : c.rank <= 32 ? 2 : c.rank <= 64 ? 4 : 8;
  const bool fits = c.dtype != MO_DTYPE_F32 || p.ranks < 8;  // in LDS, with two buffers of the weight
  const uint64_t tall = div_up(c.rows, 128), most = div_up(features, 512);
  p.rows = !odd(c) && fits && c.rows >= 128ull * c.requests && tall * (most < 16 ? most : 16) >= 256 ? 128 : 16;
  const uint64_t tiles = div_up(c.rows, p.rows), least = p.rows == 128 ? 512 : 1024;
  const uint64_t splits = between<uint64_t>(1, (p.rows == 128 ? 512 : 1024) / tiles, div_up(features, least));
  p.span = (uint32_t)round_up(div_up(features, splits > 16 ? 16 : splits), p.rows == 128 ? 128 : 1024);  // whole steps
  p.splits = (uint32_t)div_up(features, p.span);
  p.slots = tiles + c.requests + 1;
  return p;
}

// Rows a tile and columns a workgroup of an expand. Tiles of 128 rows share v, but each of their workgroups adds up h's planes, one for
// each split of the shrink, for the columns that it has. They are taken with more than 16 ranks and 2048 rows or more: in float32
// where a workgroup has 20 columns for every plane, in bfloat16 where its columns times its ranks are 4096 for every plane, in float16
// so with more than 64 ranks; not for short requests, whose other rows would be empty. The expand alone in tiles of 16 and of 128, us:
//   bfloat16  32 ranks, one plane: 1333 rows of 8192 12.1 and 11.7, 4608 of 8192 29.5 and 26.3; two: 17792 of 8192 126 and 134; 64 ranks, one
//     plane: 4608 of 3072 21.1 and 18.2; two: 17792 of 8192 186 and 134; three: 4608 of 3072 (2730 a plane) 24.3 and 26.2, of 8192
//     (8192) 49.5 and 42.2; eight: 8192 of 3072 (2048) 43.3 and 53.7, of 8192 (4096) 95.3 and 84.1; 128 ranks, one plane: 1333 of 3072 16.2 and
//     16.7, 4608 of 8192 114 and 63
//   float32   32 ranks, one plane: 4608 of 3072 33.3 and 27.3; 13: 4608 of 3072 (10 columns a plane) 45.9 and 50.3, of 8192 (30) 91.5 and 85.8; 64
//     ranks, two: 17792 of 8192 390 and 274; eight: 8192 of 1024 (16) 36.1 and 35.7, of 3072 (32) 87.3 and 76.5; 16: 2048 of 8192 (8) 67 and 109
//   float16   32 ranks: 17792 of 8192 147 and 175; 64: 4608 of 3072 30.2 and 31.9; 128: 4608 of 3072 85.1 and 54.0
// Columns so that there are some rounds of workgroups.
struct ExpandPlan {
  uint32_t rank, rows, cols;
  uint64_t slots;
};
ExpandPlan expand_plan(const mo_adapters_call& c, uint32_t features, uint32_t planes) {
  ExpandPlan p = {};
  p.rank = c.rank <= 16 ? 16 : c.rank <= 32 ? 32 : c.rank <= 64 ? 64 : 128;
  auto cols = [&](uint64_t rows) {
    return (uint32_t)round_up(between<uint64_t>(1, div_up(c.rows, rows) * features / (rows == 128 ? 1024 : kExpandGroups), 4096),
                              rows == 128 ? 128 : 512);
  };
  const bool worth = c.dtype == MO_DTYPE_F32 ? cols(128) >= 20 * planes
                                             : cols(128) * p.rank >= 4096 * planes && (c.dtype == MO_DTYPE_BF16 || p.rank > 64);
  p.rows = !odd(c) && p.rank > 16 && c.rows >= 2048 && c.rows >= 128ull * c.requests && worth ? 128 : 16;
  p.cols = cols(p.rows);
  p.slots = div_up(c.rows, p.rows) + c.requests + 1;
  return p;
}

// Splits of the rows of the weights' gradients, the same for both: a workgroup or two for every CU (twice as many, which leave
// twice the planes: 4608 rows of 3072, 64 ranks, a backward pass 93.9 us for 80.1; fewer: 17792 of 8192 320 for 288), 128 rows
// each at least, and no more planes than 256 MB hold.
void share_rows(const mo_adapters_call& c, mo_adapters::Side* a, mo_adapters::Side* b) {
  a->cols = c.da ? c.in_features : 0, b->cols = c.db ? c.out_features : 0;
  a->tiles = (uint32_t)div_up(a->cols, mo_adapters::kOuterCols), b->tiles = (uint32_t)div_up(b->cols, mo_adapters::kOuterCols);
  const uint64_t plane = 4ull * c.adapters * c.rank * (a->cols + b->cols);
  uint64_t splits = between<uint64_t>(1, div_up(kOuterGroups, a->tiles + b->tiles), div_up(c.rows, 128));
  const uint64_t held = (256u << 20) / plane;
  splits = between<uint64_t>(1, splits, held ? held : 1);
  if (splits > mo_adapters::kMaxSplits) splits = mo_adapters::kMaxSplits;
  a->span = b->span = (uint32_t)round_up(div_up(c.rows, splits), 32);
  a->splits = b->splits = (uint32_t)div_up(c.rows, a->span);
}

// Whether a forward pass runs in one launch, where every workgroup reads the adapter's whole a: up to 128 KB of it and
// with no more workgroups than CUs. bfloat16, one launch and two in us: 16 rows with an adapter each, 16 ranks, 1024 x 1024
// 9.7 and 11.7, 3072 x 3072 (98 KB) 11.9 and 12.4; 32 ranks of 3072 (196 KB) 15.1 and 13.3; 64 of 1024 (128 KB) 16.0 and 16.4;
// 1333 rows, 16 ranks, 3072 x 3072 (252 workgroups) 14.9 and 16.2, 3072 x 8192 (672) 30.8 and 20.8. float32 of more than
// 32 ranks has not the registers: 64 of 512 25.8 and 20.9. The host's time for a launch, some 5 us, is saved besides.
bool is_few(const mo_adapters_call& c) {
  const uint64_t tiles = div_up(c.rows, 16) + c.requests - 1, weight = (uint64_t)c.rank * c.in_features * kTypeBytes[c.dtype];
  return !odd(c) && c.rank <= (c.dtype == MO_DTYPE_F32 ? 32 : 64) && weight <= (128u << 10) &&
         tiles * div_up(c.out_features, 1024) <= 256;
}

// The turned copies of the weights are the adapters', or, where the requests are fewer, the requests': of a large pool of
// adapters only those are read and have room that some request has (333 rows with one of 16 adapters, 64 ranks, 3072 and 8192
// features: the copies 5.1 us, those of all 19.5).
bool by_request(const mo_adapters_call& c) { return c.requests < c.adapters; }
uint64_t places(const mo_adapters_call& c) { return by_request(c) ? c.requests : c.adapters; }

// Where what a call needs for itself lies in its workspace.
struct Room {
  uint64_t back, planes, turned_a, turned_b, turned_hidden, turned_back, da, db, bytes;  // offsets
};
Room room_of(const mo_adapters_call& c, bool backward) {
  Room r = {};
  auto take = [&](uint64_t bytes) {
    const uint64_t at = r.bytes;
    r.bytes += round_up(bytes, 256);
    return at;
  };
  const uint64_t between_bytes = c.rows * c.rank * 4, size = kTypeBytes[c.dtype];
  const uint64_t turned = round_up(c.rows, 32) * c.rank * 4;  // in whole steps of 32 rows
  if (!backward) {
    if (is_few(c)) return r;
    const ShrinkPlan p = shrink_plan(c, c.in_features);
    if (p.splits > 1) r.planes = take(p.splits * between_bytes);
    return r;
  }
  if (c.dx || c.da) {
    const ShrinkPlan p = shrink_plan(c, c.out_features);
    r.planes = take(p.splits * between_bytes);
    r.turned_b = take(places(c) * c.rank * c.out_features * size);
  }
  if (c.dx) r.turned_a = take(places(c) * c.rank * c.in_features * size);
  if (c.da) r.turned_back = take(turned);
  if (c.db) r.turned_hidden = take(turned);
  if (c.da || c.db) {
    mo_adapters::Side a = {}, b = {};
    share_rows(c, &a, &b);
    if (c.da && a.splits > 1) r.da = take(4ull * a.splits * c.adapters * c.rank * c.in_features);
    if (c.db && b.splits > 1) r.db = take(4ull * b.splits * c.adapters * c.rank * c.out_features);
  }
  return r;
}

// The kernels of one type: each with a size and a form, which make its name and its number.
enum Kind { kShrink, kExpand, kOuter, kJoin, kTurn, kFew };
int start(const mo_adapters_call& c, Kind kind, uint32_t size, const char* form, uint64_t gx, uint64_t gy, uint64_t gz, void* args,
          uint64_t stream, uint32_t threads = 256) {
  if (gx >= (1ull << 31) || gy >= (1u << 16) || gz >= (1u << 16)) return mo::set_error(MO_E_INVALID, "too many values");
  static const char* const names[] = {"shrink_", "expand_", "outer_", "join_", "turn_", "few_"};
  auto name = [&]() {
    std::string n = std::string("mo_adapters_") + names[kind] + kTypeNames[c.dtype];
    if (size) n += "_" + std::to_string(size);
    if (*form) n += std::string("_") + form;
    return n;
  };
  const int step = size >= 128 ? 7 : size >= 64 ? 6 : size >= 32 ? 5 : size >= 16 ? 4 : size >= 8 ? 3 : size >= 4 ? 2 : size >= 2 ? 1 : 0;
  // sizes: up to 8 of a shrink and an outer, 16 to 128 of an expand; forms: "", "odd", "tall"
  const int place = *form == 't' ? 1 : *form == 'o' ? 2 : 0;
  const int id = kind == kShrink ? step * 3 + place : kind == kExpand ? 12 + (step - 4) * 3 + place
                 : kind == kOuter ? 24 + step * 3 + place
                 : kind == kFew   ? 33 + step
                 : kind == kJoin  ? 36
                                  : 37;
  hipFunction_t kernel = nullptr;
  if (int rc = kernels().get((int)c.dtype * 40 + id, name, &kernel)) return rc;
  void* params[] = {args};
  return mo::launch(kernel, (uint32_t)gx, (uint32_t)gy, (uint32_t)gz, threads, stream, params, "adapters launch");
}

int shrink(const mo_adapters_call& c, const Requests& by, uint64_t x, uint64_t stride, uint64_t w, uint32_t features, uint64_t to,
           bool backward, uint64_t stream) {
  const ShrinkPlan p = shrink_plan(c, features);
  mo_adapters::Shrink a = {};
  a.by = by, a.x = (const void*)x, a.w = (const void*)w, a.to = (float*)to;
  a.x_stride = stride, a.features = features, a.span = p.span, a.scaled = backward, a.by_request = backward && by_request(c);
  return start(c, kShrink, p.ranks, odd(c) ? "odd" : p.rows == 128 ? "tall" : "", p.slots, p.splits, 1, &a, stream, 512);
}

int expand(const mo_adapters_call& c, mo_adapters::Expand& a, uint64_t stream) {
  const ExpandPlan p = expand_plan(c, a.features, a.splits);
  a.cols = p.cols;
  return start(c, kExpand, p.rank, odd(c) ? "odd" : p.rows == 128 ? "tall" : "", p.slots, div_up(a.features, p.cols), 1, &a, stream);
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
  mo_adapters::Expand e = {};
  e.by = by;
  if (!backward && is_few(c)) {
    mo_adapters::Few f = {};
    f.in.by = by, f.in.x = (const void*)c.x, f.in.w = (const void*)c.a, f.in.to = (float*)c.hidden;
    f.in.x_stride = stride_of(c, c.x_stride, c.in_features), f.in.features = c.in_features;
    f.out.v = (const void*)c.b, f.out.base = (const void*)c.result, f.out.to = (void*)c.y;
    f.out.base_stride = stride_of(c, c.result_stride, c.out_features), f.out.features = c.out_features;
    return start(c, kFew, c.rank <= 16 ? 1 : c.rank <= 32 ? 2 : 4, "", div_up(c.rows, 16) + c.requests + 1,
                 div_up(c.out_features, 1024), 1, &f, stream, 512);
  }
  if (!backward) {
    e.splits = shrink_plan(c, c.in_features).splits;
    const uint64_t to = e.splits > 1 ? planes : c.hidden;
    if (int rc = shrink(c, by, c.x, stride_of(c, c.x_stride, c.in_features), c.a, c.in_features, to, false, stream)) return rc;
    e.h = (const float*)to, e.h_sum = e.splits > 1 ? (float*)c.hidden : nullptr;
    e.v = (const void*)c.b, e.base = (const void*)c.result, e.base_stride = stride_of(c, c.result_stride, c.out_features), e.to = (void*)c.y;
    e.features = c.out_features, e.scaled = 1;
    return expand(c, e, stream);
  }
  mo_adapters::Turn t = {};
  t.by = by, t.places = (uint32_t)places(c), t.by_request = by_request(c), t.count = by.rows, t.rank = c.rank;
  auto turned = [&](int i, uint64_t from, uint64_t to, uint32_t rows, uint32_t cols) {
    t.from[i] = (const void*)from, t.to[i] = (void*)to, t.rows[i] = rows, t.cols[i] = cols;
    t.tiles[i] = (uint32_t)(div_up(rows, 32) * div_up(cols, 32));
  };
  if (c.dx || c.da) turned(0, c.b, workspace + room.turned_b, c.out_features, c.rank);
  if (c.dx) turned(1, c.a, workspace + room.turned_a, c.rank, c.in_features);
  const uint64_t narrow = div_up(c.rows, 32) * div_up(c.rank, 32);
  if (c.db) t.narrow = (const float*)c.hidden, t.turned = (float*)(workspace + room.turned_hidden), t.splits = 1;
  const uint64_t weights = (uint64_t)t.tiles[0] + t.tiles[1];
  if (int rc = start(c, kTurn, 0, "", weights + (c.db ? narrow : 0), weights ? places(c) : 1, 1, &t, stream)) return rc;
  if (c.dx || c.da) {
    if (int rc = shrink(c, by, c.grad, stride_of(c, c.grad_stride, c.out_features), workspace + room.turned_b, c.out_features, planes, true, stream)) return rc;
    const uint32_t splits = shrink_plan(c, c.out_features).splits;
    if (c.dx) {
      e.splits = splits, e.h = (const float*)planes, e.turned = c.da ? (float*)(workspace + room.turned_back) : nullptr;
      e.v = (const void*)(workspace + room.turned_a), e.base = (const void*)c.add, e.base_stride = stride_of(c, c.add_stride, c.in_features);
      e.to = (void*)c.dx, e.features = c.in_features, e.by_request = by_request(c);
      if (int rc = expand(c, e, stream)) return rc;
    } else {
      t.tiles[0] = t.tiles[1] = 0;
      t.narrow = (const float*)planes, t.turned = (float*)(workspace + room.turned_back), t.splits = splits;
      if (int rc = start(c, kTurn, 0, "", narrow, 1, 1, &t, stream)) return rc;
    }
  }
  if (!c.da && !c.db) return 0;
  mo_adapters::Outer o = {};
  o.by = by;
  mo_adapters::Side &a = o.side[0], &b = o.side[1];
  share_rows(c, &a, &b);
  a.wide = (const void*)c.x, a.exponents = (const uint8_t*)c.x_exponents, a.narrow = (const float*)(workspace + room.turned_back);
  a.planes = (float*)(workspace + room.da), a.to = (void*)c.da, a.stride = stride_of(c, c.x_stride, c.in_features), a.groups = (c.in_features + 31) / 32;
  b.wide = (const void*)c.grad, b.narrow = (const float*)(workspace + room.turned_hidden);
  b.planes = (float*)(workspace + room.db), b.to = (void*)c.db, b.stride = stride_of(c, c.grad_stride, c.out_features);
  b.turned = 1, b.scaled = 1;
  // up to 64 ranks a workgroup (by 32, which read the rows again: 17792 rows of 8192 and 3072, 64 ranks, 200 us for 138)
  const uint32_t ranks = c.rank <= 16 ? 1 : c.rank <= 32 ? 2 : 4;
  if (int rc = start(c, kOuter, ranks, odd(c) ? "odd" : "", (uint64_t)a.tiles + b.tiles, a.splits,
                     (uint64_t)c.adapters * div_up(c.rank, ranks * 16), &o, stream))
    return rc;
  if (a.splits == 1) return 0;
  const uint64_t size = (uint64_t)c.rank * (a.cols > b.cols ? a.cols : b.cols);
  return start(c, kJoin, 0, "", div_up(size, 1024), c.adapters, 2, &o, stream);
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
