// C entry points of the record cache's operators: every size, alignment and
// device range is checked here, before anything is enqueued.
#include <math.h>

#include <algorithm>
#include <numeric>

#include "../../include/seoulkv4_hip.h"
#include "skv_cache.h"
#include "skv_dense.h"

namespace skv {

namespace {

constexpr int GROUPS = SKV_GROUPS, QHEADS = SKV_GROUPS * SKV_HEADS;

// Collects the checks of one call: the first failure's code stays.
struct Check {
  int code = SKV_OK;

  explicit Check(const char* what) : what_(what) {}
  bool ok() const { return code == SKV_OK; }
  template <typename... A>
  bool require(bool cond, const char* fmt, A... args) {
    if (ok() && !cond) code = note_call_error(SKV_EINVAL, fmt, args...);
    return ok();
  }
  // device memory of the current device that holds `bytes` from ptr on
  void memory(const char* name, const void* ptr, uint64_t bytes, unsigned align) {
    if (!require(ptr != nullptr, "%s: NULL %s", what_, name)) return;
    if (!require((uintptr_t)ptr % align == 0, "%s: %s must be %u-byte aligned", what_, name, align)) return;
    if (device_ < 0) {
      const hipError_t e = hipGetDevice(&device_);
      if (e != hipSuccess) {
        code = note_call_error(SKV_EHIP, "%s: no current device: %s", what_, hipGetErrorString(e));
        return;
      }
    }
    if (const char* why = device_range_error(ptr, bytes, device_))
      code = note_call_error(SKV_EINVAL, "%s: %s (%llu bytes) %s", what_, name,
                             (unsigned long long)bytes, why);
  }

 private:
  const char* what_;
  int device_ = -1;
};

// Whether `count` steps of a stride reach at most 2^40 elements, which keeps
// every sum and product below in 64 bits.
bool steps_fit(int64_t stride, int count) {
  return stride >= 0 && stride <= ((int64_t)1 << 40) / (count > 1 ? count - 1 : 1);
}

// Elements from a row tensor's first to one past its last.
uint64_t extent(const Rows& r, int batch, int n, int heads, int dim) {
  return (uint64_t)(batch - 1) * r.sb + (uint64_t)(n - 1) * r.st + (uint64_t)(heads - 1) * r.sh + dim;
}

// Whether no two rows of an output share an element, by strides alone: in
// ascending order each is at least what the dimensions below it span.
bool rows_apart(const Rows& r, int batch, int n, int heads, int dim) {
  struct { int64_t stride; int count; } d[3] = {{r.sb, batch}, {r.st, n}, {r.sh, heads}};
  std::sort(d, d + 3, [](const auto& a, const auto& b) { return a.stride < b.stride; });
  uint64_t span = dim;
  for (const auto& x : d) {
    if (x.count == 1) continue;
    if ((uint64_t)x.stride < span) return false;
    span += (uint64_t)(x.count - 1) * x.stride;
  }
  return true;
}

bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x < y + nb && y < x + na;
}

// Whether two row tensors of `batch` x n tokens share no byte, by strides alone:
// for some of the dimensions, both step along these in multiples of a period,
// and what y spans along the others lies between what x does and its copy a
// period on (heads of one fused row: the token's stride).  No such dimensions:
// may overlap.
bool apart(const Rows& x, int x_heads, const Rows& y, int y_heads, int batch, int n, int dim, unsigned size) {
  const int64_t x_stride[3] = {x.sb, x.st, x.sh}, y_stride[3] = {y.sb, y.st, y.sh};
  const int x_count[3] = {batch, n, x_heads}, y_count[3] = {batch, n, y_heads};
  for (int steps = 0; steps < 8; ++steps) {
    uint64_t period = 0, x_span = dim, y_span = dim;
    auto add = [&](int d, int count, int64_t stride, uint64_t& span) {
      if (count == 1) return;
      if (steps >> d & 1) period = std::gcd(period, (uint64_t)stride);
      else span += (uint64_t)(count - 1) * stride;
    };
    for (int d = 0; d < 3; ++d) {
      add(d, x_count[d], x_stride[d], x_span);
      add(d, y_count[d], y_stride[d], y_span);
    }
    x_span *= size;
    y_span *= size;
    if (period == 0) {
      if (!overlap(x.data, x_span, y.data, y_span)) return true;
      continue;
    }
    period *= size;
    const int64_t off = (int64_t)((uintptr_t)y.data - (uintptr_t)x.data) % (int64_t)period;
    const uint64_t from = off < 0 ? off + period : off;
    if (x_span <= from && from + y_span <= period) return true;
  }
  return false;
}

Rows rows_of(Check& c, const char* name, const skv_rows* r, int batch, int n, int heads, int dim,
             unsigned size, bool output) {
  Rows out{};
  if (!c.ok()) return out;
  if (!c.require(r != nullptr, "NULL %s rows", name)) return out;
  out = Rows{r->data, r->batch_stride, r->token_stride, r->head_stride};
  if (!c.require(steps_fit(out.sb, batch) && steps_fit(out.st, n) && steps_fit(out.sh, heads),
                 "%s: strides must lie in [0, 2^40], their steps in all too", name))
    return out;
  if (output && !c.require(rows_apart(out, batch, n, heads, dim), "%s: output rows overlap", name))
    return out;
  c.memory(name, out.data, extent(out, batch, n, heads, dim) * size, size);
  return out;
}

// The same elements, or none in common.
void in_place_or_apart(Check& c, const char* name, const Rows& x, const Rows& y, int batch, int n,
                       int heads, int dim, unsigned size) {
  const bool same = x.data == y.data && (batch == 1 || x.sb == y.sb) && (n == 1 || x.st == y.st) &&
                    (heads == 1 || x.sh == y.sh);
  c.require(same || apart(x, heads, y, heads, batch, n, dim, size),
            "%s overlaps its input in another layout", name);
}

bool four_bits(const skv_record_cache& c) { return c.record_bytes == RECORD_FOUR; }

uint64_t record_bytes(const skv_record_cache& c) {
  const uint64_t rows = c.page_tokens ? (uint64_t)c.n_pages * c.page_tokens
                                      : (uint64_t)c.batch * c.capacity;
  return rows * GROUPS * (four_bits(c) ? RECORD_FOUR : RECORD_EIGHT);
}

CacheView view_of(Check& k, const skv_record_cache* c) {
  CacheView v{};
  if (!k.require(c != nullptr, "NULL cache") ||
      !k.require(c->batch >= 1 && c->batch <= CACHE_MAX_BATCH, "batch %d outside [1, %d]", c->batch,
                 CACHE_MAX_BATCH) ||
      !k.require(c->capacity >= 1 && c->capacity <= CACHE_MAX_SLOTS, "capacity %d outside [1, 2^20]",
                 c->capacity) ||
      !k.require(c->record_bytes == 0 || c->record_bytes == RECORD_EIGHT || four_bits(*c),
                 "records of %d bytes: 512 (8 bits a value) or 272 (4 bits)", c->record_bytes))
    return v;
  const int pt = c->page_tokens;
  if (pt == 0) {
    k.require(c->n_pages == 0 && c->table_len == 0 && !c->page_table,
              "a contiguous cache (page_tokens 0) has no pages and no table");
  } else if (k.require(pt >= 16 && pt <= 65536 && !(pt & (pt - 1)),
                       "page_tokens %d is no power of two in [16, 65536]", pt)) {
    k.require(c->n_pages >= 1 && c->n_pages < (int64_t)1 << 31 &&
                  c->n_pages * GROUPS * pt <= (int64_t)1 << 31, "a pool holds 1 page to 2^31 records, not %lld pages",
              (long long)c->n_pages);
    k.require(c->table_len >= 1 && (int64_t)c->table_len * pt == c->capacity,
              "capacity %d is not table_len %d x page_tokens %d", c->capacity, c->table_len, pt);
  }
  if (!k.ok()) return v;
  k.memory("records", c->records, record_bytes(*c), 16);
  if (pt) k.memory("page table", c->page_table, (uint64_t)c->batch * c->table_len * 4, 4);
  k.memory("lengths", c->lengths, (uint64_t)c->batch * 4, 4);
  const uint64_t slots = (uint64_t)c->batch * GROUPS * c->capacity;
  if (k.ok() && c->positions) k.memory("slot positions", c->positions, slots * 4, 4);
  if (k.ok() && c->weights) k.memory("weights", c->weights, slots * 4, 4);
  if (k.ok() && c->status) k.memory("status", c->status, 4, 4);
  v.records = static_cast<uint8_t*>(c->records);
  v.table = pt ? c->page_table : nullptr;
  v.lengths = c->lengths;
  v.n_pages = (uint32_t)c->n_pages;
  v.table_len = c->table_len;
  v.shift = pt ? __builtin_ctz((unsigned)pt) : 0;
  v.batch = c->batch;
  v.capacity = c->capacity;
  v.four = four_bits(*c);
  return v;
}

RotaryArgs rotary_of(Check& k, const skv_rotary_table* t, const void* positions, int64_t sb,
                     int positions64, int batch, int n, int dim) {
  RotaryArgs r{};
  if (t) {
    if (!k.require(t->pairs >= 1 && 2 * (int64_t)t->pairs <= dim, "%d pairs do not fit a head of %d",
                   t->pairs, dim) ||
        !k.require(isfinite(t->scale), "the rotary scale is not finite"))
      return r;
    k.memory("turns", t->turns, (uint64_t)t->pairs * 8, 8);
    r.turns = t->turns;
    r.pairs = t->pairs;
    r.scale = t->scale;
  }
  if (positions && k.require((sb == 0 || sb >= n) && steps_fit(sb, batch),
                             "position rows of %d at stride %lld", n, (long long)sb)) {
    const unsigned size = positions64 ? 8 : 4;
    k.memory("positions", positions, ((uint64_t)(batch - 1) * sb + n) * size, size);
  }
  r.positions = positions;
  r.position_sb = sb;
  r.positions64 = positions64 != 0;
  return r;
}

NormArgs norm_of(Check& k, const skv_head_norm* n, int rows_dtype, int heads, int dim) {
  NormArgs w{};
  if (!k.require(n != nullptr, "NULL norm") ||
      !k.require(n->dtype == rows_dtype || n->dtype == SKV_FP32, "a weight of dtype %d for rows of dtype %d", n->dtype,
                 rows_dtype) ||
      !k.require(isfinite(n->eps) && n->eps > 0.f, "eps must be positive and finite"))
    return w;
  const unsigned size = n->dtype == SKV_FP32 ? 4 : 2;
  k.memory("norm weight", n->weight, (uint64_t)(n->per_head ? heads : 1) * dim * size, size);
  w.weight = n->weight;
  w.sh = n->per_head ? dim : 0;
  w.eps = n->eps;
  w.wide = n->dtype == SKV_FP32;
  return w;
}

// The window's sizes; needed: a call that has one.
Window window_of(Check& c, int window, int sink, bool needed) {
  c.require(sink >= 0 && window >= (needed ? 1 : 0) && (window > 0 || sink == 0),
            "window %d must be positive and sink %d not negative", window, sink);
  return Window{window, sink};
}

void workspace_of(Check& c, const void* workspace, int64_t bytes, int64_t need) {
  c.require(bytes >= need, "a workspace of %lld bytes, %lld needed", (long long)bytes, (long long)need);
  if (c.ok() && need) c.memory("workspace", workspace, need, 16);
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return note_call_error(SKV_EHIP, "%s launch failed: %s", what, hipGetErrorString(e));
  return SKV_OK;
}

}  // namespace

}  // namespace skv

using namespace skv;

extern "C" {

// What the turns of rows have in common.
static int rotary_operands(Check& k, const skv_rotary_table* table, int dtype, int batch, int n, int heads, int dim,
                           const void* positions, int64_t position_batch_stride, int positions64, RotaryArgs& r) {
  k.require(table != nullptr, "NULL rotary table");
  k.require(dtype == SKV_BF16 || dtype == SKV_FP16 || dtype == SKV_FP32, "unknown dtype %d", dtype);
  k.require(dim >= 2 && dim <= 1024, "head dimension %d outside [2, 1024]", dim);
  // a grid holds fewer than 2^32 threads
  k.require(batch >= 1 && n >= 1 && heads >= 1 && heads <= 65535 &&
                (int64_t)batch * n <= ((int64_t)1 << 31) / dim,
            "%d x %d tokens of %d heads x %d: at most 65535 heads and 2^31 / dim tokens a call", batch, n,
            heads, dim);
  k.require(positions != nullptr, "NULL positions");
  if (k.ok()) r = rotary_of(k, table, positions, position_batch_stride, positions64, batch, n, dim);
  return k.code;
}

// What the normed ones have beside that.
static int norm_operands(Check& k, const skv_rotary_table* table, const skv_head_norm* norm, const skv_rows* x, int dtype,
                         int batch, int n, int heads, int dim, const void* positions, int64_t position_batch_stride,
                         int positions64, NormRows& a) {
  if (rotary_operands(k, table, dtype, batch, n, heads, dim, positions, position_batch_stride, positions64, a.r) != SKV_OK)
    return k.code;
  // (64 lanes a token)
  k.require((int64_t)batch * n <= (int64_t)1 << 25, "%d x %d tokens: at most 2^25 a call", batch, n);
  if (k.ok()) a.w = norm_of(k, norm, dtype, heads, dim);
  a.x = rows_of(k, "x", x, batch, n, heads, dim, dtype == SKV_FP32 ? 4 : 2, false);
  a.interleaved = table->interleaved != 0;
  a.batch = batch;
  a.n = n;
  a.heads = heads;
  a.dim = dim;
  return k.code;
}

int skv_rotary(const skv_rotary_table* table, const skv_rows* x, const skv_rows* y, int dtype,
               int batch, int n, int heads, int dim, const void* positions,
               int64_t position_batch_stride, int positions64, int transpose, void* stream) {
  Check k("rotary");
  RotaryArgs r;
  if (rotary_operands(k, table, dtype, batch, n, heads, dim, positions, position_batch_stride, positions64, r) != SKV_OK)
    return k.code;
  const unsigned size = dtype == SKV_FP32 ? 4 : 2;
  const Rows in = rows_of(k, "x", x, batch, n, heads, dim, size, false);
  if (!k.ok()) return k.code;
  const Rows out = rows_of(k, "y", y, batch, n, heads, dim, size, true);
  if (k.ok()) in_place_or_apart(k, "y", in, out, batch, n, heads, dim, size);
  if (!k.ok()) return k.code;
  (void)hipGetLastError();  // a launch error below is this call's, not an earlier one's
  launch_rotary(r, table->interleaved != 0, transpose != 0, in, out, dtype, batch, n, heads, dim,
                static_cast<hipStream_t>(stream));
  return launched("rotary");
}

int skv_norm_rotary(const skv_rotary_table* table, const skv_head_norm* norm, const skv_rows* x, const skv_rows* y,
                    int dtype, int batch, int n, int heads, int dim, const void* positions,
                    int64_t position_batch_stride, int positions64, void* stream) {
  Check k("norm rotary");
  NormRows a{};
  if (norm_operands(k, table, norm, x, dtype, batch, n, heads, dim, positions, position_batch_stride, positions64, a) !=
      SKV_OK)
    return k.code;
  const unsigned size = dtype == SKV_FP32 ? 4 : 2;
  const Rows out = rows_of(k, "y", y, batch, n, heads, dim, size, true);
  if (k.ok()) in_place_or_apart(k, "y", a.x, out, batch, n, heads, dim, size);
  if (!k.ok()) return k.code;
  (void)hipGetLastError();
  launch_norm_rotary(a, out, dtype, static_cast<hipStream_t>(stream));
  return launched("norm rotary");
}

int64_t skv_norm_grad_workspace(int64_t tokens, int heads, int dim, int per_head) {
  if (tokens < 1 || tokens > (int64_t)1 << 25 || heads < 1 || heads > 65535 || dim < 2 || dim > 1024) return 0;
  return (int64_t)norm_grad_workspace(tokens, heads, dim, per_head != 0);
}

int skv_norm_rotary_grad(const skv_rotary_table* table, const skv_head_norm* norm, const skv_rows* g, const skv_rows* x,
                         const skv_rows* dx, int dtype, int batch, int n, int heads, int dim, const void* positions,
                         int64_t position_batch_stride, int positions64, void* dweight, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  Check k("norm rotary gradient");
  NormRows a{};
  if (norm_operands(k, table, norm, x, dtype, batch, n, heads, dim, positions, position_batch_stride, positions64, a) !=
      SKV_OK)
    return k.code;
  const unsigned size = dtype == SKV_FP32 ? 4 : 2;
  const Rows in = rows_of(k, "g", g, batch, n, heads, dim, size, false);
  const Rows out = rows_of(k, "dx", dx, batch, n, heads, dim, size, true);
  if (k.ok()) in_place_or_apart(k, "dx", a.x, out, batch, n, heads, dim, size);
  if (k.ok()) in_place_or_apart(k, "dx", in, out, batch, n, heads, dim, size);
  if (k.ok()) {
    const unsigned weight_size = a.w.wide ? 4 : 2;
    k.memory("dweight", dweight, (uint64_t)(norm->per_head ? heads : 1) * dim * weight_size, weight_size);
  }
  if (k.ok())
    workspace_of(k, workspace, workspace_bytes,
                 skv_norm_grad_workspace((int64_t)batch * n, heads, dim, norm->per_head));
  if (!k.ok()) return k.code;
  (void)hipGetLastError();
  launch_norm_grad(a, in, out, dtype, dweight, norm->dtype, static_cast<float*>(workspace),
                   static_cast<hipStream_t>(stream));
  return launched("norm rotary gradient");
}

int skv_cache_write(const skv_record_cache* cache, const skv_rotary_table* table, const skv_rows* k,
                    const skv_rows* v, const skv_rows* q, const skv_rows* q_out, int n,
                    const void* positions, int positions64, const int32_t* counts, void* stream) {
  return skv_cache_write_normed(cache, table, nullptr, nullptr, k, v, q, q_out, n, positions, positions64, counts,
                                stream);
}

int skv_cache_write_normed(const skv_record_cache* cache, const skv_rotary_table* table, const skv_head_norm* q_norm,
                           const skv_head_norm* k_norm, const skv_rows* k, const skv_rows* v, const skv_rows* q,
                           const skv_rows* q_out, int n, const void* positions, int positions64, const int32_t* counts,
                           void* stream) {
  Check c("cache write");
  WriteArgs a{};
  a.c = view_of(c, cache);
  if (!c.ok()) return c.code;
  const int batch = cache->batch;
  c.require(n >= 1 && n <= cache->capacity, "%d tokens for a capacity of %d", n, cache->capacity);
  c.require((int64_t)batch * n <= ((int64_t)1 << 31) / SKV_DIM, "%d x %d tokens: at most 2^23 a call", batch, n);
  c.require((q == nullptr) == (q_out == nullptr), "q and q_out go together");
  c.require(!q_norm || q, "a norm of q without q");
  NormArgs qw{}, kw{};
  if (c.ok() && q_norm) qw = norm_of(c, q_norm, SKV_BF16, QHEADS, SKV_DIM);
  if (c.ok() && k_norm) kw = norm_of(c, k_norm, SKV_BF16, GROUPS, SKV_DIM);
  if (!c.ok()) return c.code;
  a.r = rotary_of(c, table, positions, n, positions64, batch, n, SKV_DIM);
  if (c.ok())
    c.require(!overlap(positions, (uint64_t)batch * n * (positions64 ? 8 : 4), cache->positions,
                       (uint64_t)batch * GROUPS * cache->capacity * 4),
              "the positions lie in the cache's own, which the write changes");
  a.interleaved = table ? table->interleaved != 0 : 0;
  if (c.ok()) a.k = rows_of(c, "k", k, batch, n, GROUPS, SKV_DIM, 2, false);
  if (c.ok()) a.v = rows_of(c, "v", v, batch, n, GROUPS, SKV_DIM, 2, false);
  if (c.ok() && q) {
    a.q = rows_of(c, "q", q, batch, n, QHEADS, SKV_DIM, 2, false);
    if (c.ok()) a.q_out = rows_of(c, "q_out", q_out, batch, n, QHEADS, SKV_DIM, 2, true);
    if (c.ok()) in_place_or_apart(c, "q_out", a.q, a.q_out, batch, n, QHEADS, SKV_DIM, 2);
    // k and v are read while q_out is written
    if (c.ok())
      c.require(apart(a.q_out, QHEADS, a.k, GROUPS, batch, n, SKV_DIM, 2) &&
                    apart(a.q_out, QHEADS, a.v, GROUPS, batch, n, SKV_DIM, 2),
                "q_out overlaps k or v");
  }
  if (c.ok() && counts) c.memory("counts", counts, (uint64_t)batch * 4, 4);
  if (!c.ok()) return c.code;
  a.n = n;
  a.counts = counts;
  a.positions = cache->positions;
  a.weights = cache->weights;
  a.status = cache->status;
  (void)hipGetLastError();
  if (q_norm || k_norm || a.c.four) launch_cache_write_normed(a, qw, kw, static_cast<hipStream_t>(stream));
  else launch_cache_write(a, static_cast<hipStream_t>(stream));
  return launched("cache write");
}

int64_t skv_tree_workspace(int batch, int n) {
  if (batch < 1 || batch > CACHE_MAX_BATCH || n < 1 || n > TREE_MAX_DRAFTS) return 0;
  return (int64_t)tree_workspace(batch, n);
}

// What the attention operators have in common; most: drafts of a sequence.
static int tree_operands(Check& c, const skv_record_cache* cache, const skv_rows* q, int n, int most,
                         const int64_t* tree, const int32_t* counts, float cap, CacheView& view,
                         Rows& rows) {
  view = view_of(c, cache);
  if (!c.ok()) return c.code;
  c.require(n >= 1 && n <= most, "%d drafts outside [1, %d]", n, most);
  c.require(cap == 0.f || (cap >= 0x1p-100f && cap <= 0x1p100f), "cap must be 0 or lie in [2^-100, 2^100]");
  if (!c.ok()) return c.code;
  rows = rows_of(c, "q", q, cache->batch, n, QHEADS, SKV_DIM, 2, false);
  if (c.ok())
    c.require(((uintptr_t)rows.data & 15) == 0 && rows.sb % 8 == 0 && rows.st % 8 == 0 && rows.sh % 8 == 0,
              "q rows must be 16-byte aligned");
  const uint64_t tokens = (uint64_t)cache->batch * n;
  if (c.ok() && tree) c.memory("tree", tree, tokens * 8, 8);
  if (c.ok() && counts) c.memory("counts", counts, (uint64_t)cache->batch * 4, 4);
  return c.code;
}

static int tree_decode(const skv_record_cache* cache, const skv_rows* q, int n, const int64_t* tree,
                       const int32_t* counts, float cap, int window, int sink, bool windowed, void* out, float* lse,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  Check c("tree decode");
  TreeArgs a{};
  a.window = window_of(c, window, sink, windowed);
  if (tree_operands(c, cache, q, n, TREE_MAX_DRAFTS, tree, counts, cap, a.c, a.q) != SKV_OK) return c.code;
  const uint64_t rows = (uint64_t)cache->batch * n * QHEADS;
  c.memory("out", out, rows * SKV_DIM * 2, 16);
  if (c.ok()) c.memory("lse", lse, rows * 4, 4);
  const int64_t need = skv_tree_workspace(cache->batch, n);
  c.require(workspace_bytes >= need, "a workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
            (long long)need);
  if (c.ok()) c.memory("workspace", workspace, need, 16);
  if (!c.ok()) return c.code;
  a.n = n;
  a.tree = tree;
  a.counts = counts;
  a.cap = cap;
  a.part = static_cast<float*>(workspace);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  (void)hipGetLastError();
  launch_tree(a, static_cast<hipStream_t>(stream));
  return launched("tree decode");
}

int skv_tree_decode(const skv_record_cache* cache, const skv_rows* q, int n, const int64_t* tree,
                    const int32_t* counts, float cap, void* out, float* lse, void* workspace,
                    int64_t workspace_bytes, void* stream) {
  return tree_decode(cache, q, n, tree, counts, cap, 0, 0, false, out, lse, workspace, workspace_bytes, stream);
}

int skv_tree_decode_window(const skv_record_cache* cache, const skv_rows* q, int n, const int64_t* tree,
                           const int32_t* counts, float cap, int window, int sink, void* out, float* lse,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  return tree_decode(cache, q, n, tree, counts, cap, window, sink, true, out, lse, workspace, workspace_bytes, stream);
}

int64_t skv_attend_workspace(int batch, int n) {
  if (batch < 1 || batch > CACHE_MAX_BATCH || n < 1 || n > ATTEND_MAX_TOKENS / batch) return 0;
  return (int64_t)attend_workspace(batch, n);
}

int skv_attend(const skv_record_cache* cache, const skv_rows* q, int n, const int32_t* counts, float cap, int window,
               int sink, void* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  Check c("attend");
  AttendArgs a{};
  a.window = window_of(c, window, sink, false);
  const int batch = cache && cache->batch > 0 ? cache->batch : 1;
  if (tree_operands(c, cache, q, n, ATTEND_MAX_TOKENS / batch, nullptr, counts, cap, a.c, a.q) != SKV_OK) return c.code;
  const uint64_t rows = (uint64_t)cache->batch * n * QHEADS;
  c.memory("out", out, rows * SKV_DIM * 2, 16);
  if (c.ok()) c.memory("lse", lse, rows * 4, 4);
  if (c.ok() && n > TREE_MAX_DRAFTS) {
    // some blocks write results while others read queries (fewer tokens are read by
    // one kernel and written by the next)
    const int64_t st = QHEADS * SKV_DIM;
    in_place_or_apart(c, "out", a.q, Rows{out, n * st, st, SKV_DIM}, batch, n, QHEADS, SKV_DIM, 2);
    c.require(!overlap(lse, rows * 4, a.q.data, 2 * extent(a.q, batch, n, QHEADS, SKV_DIM)), "lse overlaps q");
  }
  if (c.ok()) workspace_of(c, workspace, workspace_bytes, skv_attend_workspace(batch, n));
  if (!c.ok()) return c.code;
  a.n = n;
  a.counts = counts;
  a.cap = cap;
  a.work = workspace;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  (void)hipGetLastError();
  launch_attend(a, static_cast<hipStream_t>(stream));
  return launched("attend");
}

static int key_weights(const skv_record_cache* cache, const skv_rows* q, int n, const float* lse, const int64_t* tree,
                       const int32_t* counts, float cap, int window, int sink, bool windowed, int accumulate,
                       void* stream) {
  Check c("key weights");
  WeightArgs a{};
  a.window = window_of(c, window, sink, windowed);
  if (tree_operands(c, cache, q, n, TREE_MAX_DRAFTS, tree, counts, cap, a.c, a.q) != SKV_OK) return c.code;
  c.require(cache->weights != nullptr, "the cache has no weights");
  if (c.ok()) c.memory("lse", lse, (uint64_t)cache->batch * n * QHEADS * 4, 4);
  if (!c.ok()) return c.code;
  a.n = n;
  a.tree = tree;
  a.counts = counts;
  a.cap = cap;
  a.lse = lse;
  a.weights = cache->weights;
  a.accumulate = accumulate != 0;
  (void)hipGetLastError();
  launch_key_weights(a, static_cast<hipStream_t>(stream));
  return launched("key weights");
}

int skv_key_weights(const skv_record_cache* cache, const skv_rows* q, int n, const float* lse,
                    const int64_t* tree, const int32_t* counts, float cap, int accumulate,
                    void* stream) {
  return key_weights(cache, q, n, lse, tree, counts, cap, 0, 0, false, accumulate, stream);
}

int skv_key_weights_window(const skv_record_cache* cache, const skv_rows* q, int n, const float* lse,
                           const int64_t* tree, const int32_t* counts, float cap, int window, int sink,
                           int accumulate, void* stream) {
  return key_weights(cache, q, n, lse, tree, counts, cap, window, sink, true, accumulate, stream);
}

int64_t skv_evict_workspace(int batch, int capacity, int keep) {
  if (batch < 1 || batch > CACHE_MAX_BATCH || capacity < 1 || capacity > CACHE_MAX_SLOTS || keep < 1)
    return 0;
  return (int64_t)evict_workspace(batch, capacity, keep);
}

int skv_evict(const skv_record_cache* cache, const skv_record_cache* to, int keep, int sink,
              int local, void* workspace, int64_t workspace_bytes, void* stream) {
  Check c("evict");
  EvictArgs a{};
  a.from = view_of(c, cache);
  if (c.ok()) a.to = view_of(c, to);
  if (!c.ok()) return c.code;
  c.require(cache->weights != nullptr, "the cache has no weights");
  c.require(to->batch == cache->batch, "caches of %d and %d sequences", cache->batch, to->batch);
  c.require(four_bits(*to) == four_bits(*cache), "caches of records of 8 and of 4 bits");
  c.require(sink >= 0 && local >= 0 && keep >= 1 && (int64_t)sink + local <= keep,
            "keep %d must be positive and hold sink %d + local %d", keep, sink, local);
  c.require(keep <= to->capacity, "keep %d above the capacity %d of the cache it goes to", keep, to->capacity);
  if (!c.ok()) return c.code;
  const uint64_t from_slots = (uint64_t)cache->batch * GROUPS * cache->capacity * 4;
  const uint64_t to_slots = (uint64_t)to->batch * GROUPS * to->capacity * 4;
  const bool one_pool = cache->page_tokens && to->page_tokens == cache->page_tokens &&
                        cache->records == to->records && cache->n_pages == to->n_pages;
  c.require(one_pool || !overlap(cache->records, record_bytes(*cache), to->records, record_bytes(*to)),
            "the two caches share records");
  c.require(!overlap(cache->weights, from_slots, to->weights, to_slots) &&
                !overlap(cache->positions, from_slots, to->positions, to_slots) &&
                !overlap(cache->lengths, (uint64_t)cache->batch * 4, to->lengths, (uint64_t)to->batch * 4),
            "the two caches share weights, positions or lengths");
  const int64_t need = skv_evict_workspace(cache->batch, cache->capacity, keep);
  c.require(workspace_bytes >= need, "a workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
            (long long)need);
  if (c.ok()) c.memory("workspace", workspace, need, 16);
  if (!c.ok()) return c.code;
  a.positions = cache->positions;
  a.weights = cache->weights;
  a.to_positions = cache->positions ? to->positions : nullptr;
  a.to_weights = to->weights;
  a.to_lengths = to->lengths;
  a.to_status = to->status;
  a.keep = keep;
  a.sink = sink;
  a.local = local;
  a.workspace = workspace;
  (void)hipGetLastError();
  launch_evict(a, static_cast<hipStream_t>(stream));
  return launched("evict");
}

}  // extern "C"
