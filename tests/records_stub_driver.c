/* Drives the argument checks of the record cache's entry points without a
 * GPU: this program defines the HIP runtime calls that they make, device
 * memory is one counted host block and a launch runs nothing.  Every refusal
 * has to name its reason and launch nothing; every accepted call has to launch.
 * tests/test_records_host.py builds and runs it. */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <hip/hip_runtime_api.h>

#include "seoulkv4_hip.h"

static char *arena;
static const size_t ARENA = (size_t)64 << 20;
static int launches, checks;

hipError_t hipGetDevice(int *d) { *d = 0; return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
const char *hipGetErrorString(hipError_t e) { (void)e; return "stub"; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *p) {
  memset(a, 0, sizeof *a);
  if ((const char *)p < arena || (const char *)p >= arena + ARENA) return hipErrorInvalidValue;
  a->type = hipMemoryTypeDevice;
  return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t *base, size_t *size, hipDeviceptr_t p) {
  (void)p;
  *base = arena;
  *size = ARENA;
  return hipSuccess;
}
static dim3 grid, block;
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t shared, hipStream_t st) {
  (void)shared; (void)st;
  grid = g;
  block = b;
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *shared, hipStream_t *st) {
  *g = grid;
  *b = block;
  *shared = 0;
  *st = NULL;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t shared, hipStream_t st) {
  (void)f; (void)args; (void)shared; (void)st;
  if (!g.x || !g.y || (uint64_t)g.x * b.x >= (1ull << 32)) {
    fprintf(stderr, "FAILED grid %u x %u of %u threads\n", g.x, g.y, b.x);
    exit(2);
  }
  ++launches;
  return hipSuccess;
}

static void accept(const char *what, int code) {
  if (code != SKV_OK || !launches) {
    fprintf(stderr, "FAILED %s: code %d (%s), %d launches\n", what, code, skv_last_error(NULL), launches);
    exit(2);
  }
  launches = 0;
  ++checks;
}
static void refuse(const char *what, int code, const char *text) {
  if (code != SKV_EINVAL || launches || !strstr(skv_last_error(NULL), text)) {
    fprintf(stderr, "FAILED %s: code %d (%s), wanted \"%s\", %d launches\n", what, code,
            skv_last_error(NULL), text, launches);
    exit(2);
  }
  ++checks;
}

static skv_record_cache cache(void) { /* 2 sequences of 64 slots */
  skv_record_cache c = {0};
  c.records = arena;
  c.batch = 2;
  c.capacity = 64;
  c.lengths = (int32_t *)(arena + (1 << 20));
  c.positions = (int32_t *)(arena + (2 << 20));
  c.weights = (float *)(arena + (3 << 20));
  c.status = (int32_t *)(arena + (4 << 20));
  return c;
}
static skv_record_cache paged(void) { /* the same in 8 pages of 16 */
  skv_record_cache c = cache();
  c.n_pages = 8;
  c.page_tokens = 16;
  c.table_len = 4;
  c.page_table = (int32_t *)(arena + (5 << 20));
  return c;
}
static skv_rows rows(size_t at, int heads, int n) {
  skv_rows r = {arena + at, (int64_t)n * heads * 256, heads * 256, 256};
  return r;
}

#define WITH(type, make, change, call, what, text) \
  do {                                             \
    type x = make;                                 \
    change;                                        \
    refuse(what, call, text);                      \
  } while (0)

int main(void) {
  arena = aligned_alloc(4096, ARENA);
  if (!arena) return 3;
  void *far = arena + ARENA - 64, *host = malloc(256);
  const skv_rows q = rows((size_t)8 << 20, 16, 3), k = rows((size_t)12 << 20, 4, 3), v = rows((size_t)13 << 20, 4, 3);
  const skv_rows qo = rows((size_t)16 << 20, 16, 3);
  const skv_rotary_table t = {(const uint64_t *)(arena + (20 << 20)), 128, 0, 1.0f};
  int64_t *tree = (int64_t *)(arena + (21 << 20));
  int32_t *counts = (int32_t *)(arena + (22 << 20));
  void *out = arena + (24 << 20), *work = arena + (28 << 20);
  float *lse = (float *)(arena + (25 << 20));
  const int64_t size = skv_tree_workspace(2, 3);
  skv_record_cache c = cache(), p = paged();

  /* tree decode */
#define TREE(C, Q, N, CAP, OUT, LSE, W, S) skv_tree_decode(C, Q, N, tree, counts, CAP, OUT, LSE, W, S, NULL)
  accept("tree", TREE(&c, &q, 3, 0.f, out, lse, work, size));
  accept("tree paged, capped", TREE(&p, &q, 3, 30.f, out, lse, work, size));
  accept("a chain without counts", skv_tree_decode(&c, &q, 3, NULL, NULL, 0.f, out, lse, work, size, NULL));
  refuse("no cache", TREE(NULL, &q, 3, 0.f, out, lse, work, size), "NULL cache");
  WITH(skv_record_cache, c, x.batch = 0, TREE(&x, &q, 3, 0.f, out, lse, work, size), "batch 0", "batch");
  WITH(skv_record_cache, c, x.batch = 1025, TREE(&x, &q, 3, 0.f, out, lse, work, size), "batch", "batch");
  WITH(skv_record_cache, c, x.capacity = 0, TREE(&x, &q, 3, 0.f, out, lse, work, size), "capacity 0", "capacity");
  WITH(skv_record_cache, c, x.capacity = (1 << 20) + 1, TREE(&x, &q, 3, 0.f, out, lse, work, size), "capacity", "capacity");
  WITH(skv_record_cache, c, x.capacity = 1 << 20, TREE(&x, &q, 3, 0.f, out, lse, work, size), "records too short", "extends past");
  WITH(skv_record_cache, c, x.records = NULL, TREE(&x, &q, 3, 0.f, out, lse, work, size), "no records", "NULL records");
  WITH(skv_record_cache, c, x.records = arena + 8, TREE(&x, &q, 3, 0.f, out, lse, work, size), "records by 8", "aligned");
  WITH(skv_record_cache, c, x.records = host, TREE(&x, &q, 3, 0.f, out, lse, work, size), "host records", "not device memory");
  WITH(skv_record_cache, c, x.lengths = NULL, TREE(&x, &q, 3, 0.f, out, lse, work, size), "no lengths", "NULL lengths");
  WITH(skv_record_cache, c, x.n_pages = 3, TREE(&x, &q, 3, 0.f, out, lse, work, size), "pages of none", "contiguous");
  WITH(skv_record_cache, c, x.weights = far, TREE(&x, &q, 3, 0.f, out, lse, work, size), "short weights", "extends past");
  WITH(skv_record_cache, p, x.page_tokens = 24, TREE(&x, &q, 3, 0.f, out, lse, work, size), "pages of 24", "power of two");
  WITH(skv_record_cache, p, x.page_tokens = 8, TREE(&x, &q, 3, 0.f, out, lse, work, size), "pages of 8", "power of two");
  WITH(skv_record_cache, p, x.n_pages = 0, TREE(&x, &q, 3, 0.f, out, lse, work, size), "no pages", "pages");
  WITH(skv_record_cache, p, x.n_pages = (int64_t)1 << 60, TREE(&x, &q, 3, 0.f, out, lse, work, size), "2^60 pages", "pages");
  WITH(skv_record_cache, p, x.table_len = 3, TREE(&x, &q, 3, 0.f, out, lse, work, size), "short table", "table_len");
  WITH(skv_record_cache, p, x.page_table = NULL, TREE(&x, &q, 3, 0.f, out, lse, work, size), "no table", "page table");
  refuse("no drafts", TREE(&c, &q, 0, 0.f, out, lse, work, size), "drafts");
  refuse("65 drafts", TREE(&c, &q, 65, 0.f, out, lse, work, size), "drafts");
  refuse("cap NaN", TREE(&c, &q, 3, NAN, out, lse, work, size), "cap");
  refuse("cap < 0", TREE(&c, &q, 3, -1.f, out, lse, work, size), "cap");
  refuse("cap inf", TREE(&c, &q, 3, INFINITY, out, lse, work, size), "cap");
  refuse("tiny cap", TREE(&c, &q, 3, 1e-38f, out, lse, work, size), "cap");
  refuse("huge cap", TREE(&c, &q, 3, 1e38f, out, lse, work, size), "cap");
  refuse("no q", TREE(&c, NULL, 3, 0.f, out, lse, work, size), "NULL q");
  WITH(skv_rows, q, x.data = (char *)x.data + 2, TREE(&c, &x, 3, 0.f, out, lse, work, size), "q by 2", "16-byte");
  WITH(skv_rows, q, x.token_stride = 4097, TREE(&c, &x, 3, 0.f, out, lse, work, size), "odd strides", "16-byte");
  WITH(skv_rows, q, x.batch_stride = -8, TREE(&c, &x, 3, 0.f, out, lse, work, size), "negative stride", "strides");
  WITH(skv_rows, q, x.batch_stride = (int64_t)1 << 41, TREE(&c, &x, 3, 0.f, out, lse, work, size), "huge stride", "strides");
  WITH(skv_rows, q, x.batch_stride = (int64_t)1 << 40, TREE(&c, &x, 3, 0.f, out, lse, work, size), "far rows", "extends past");
  refuse("no out", TREE(&c, &q, 3, 0.f, NULL, lse, work, size), "NULL out");
  refuse("short out", TREE(&c, &q, 3, 0.f, far, lse, work, size), "extends past");
  refuse("no lse", TREE(&c, &q, 3, 0.f, out, NULL, work, size), "NULL lse");
  refuse("small workspace", TREE(&c, &q, 3, 0.f, out, lse, work, size - 1), "workspace");
  refuse("no workspace", TREE(&c, &q, 3, 0.f, out, lse, NULL, size), "NULL workspace");
  refuse("short workspace", TREE(&c, &q, 3, 0.f, out, lse, far, size), "extends past");

  /* key weights */
#define WEIGH(C, LSE) skv_key_weights(C, &q, 3, LSE, tree, counts, 0.f, 1, NULL)
  accept("weights", WEIGH(&p, lse));
  WITH(skv_record_cache, c, x.weights = NULL, WEIGH(&x, lse), "no weights", "no weights");
  refuse("weights without lse", WEIGH(&c, NULL), "NULL lse");

  /* write */
#define WRITE(C, T, K, V, Q, O, N) skv_cache_write(C, T, K, V, Q, O, N, NULL, 0, counts, NULL)
  accept("write", WRITE(&c, &t, &k, &v, &q, &qo, 3));
  accept("write in place, unturned", WRITE(&p, NULL, &k, &v, &q, &q, 3));
  accept("write without q", WRITE(&p, &t, &k, &v, NULL, NULL, 3));
  refuse("q without q_out", WRITE(&c, &t, &k, &v, &q, NULL, 3), "go together");
  refuse("no tokens", WRITE(&c, &t, &k, &v, NULL, NULL, 0), "tokens");
  refuse("too many tokens", WRITE(&c, &t, &k, &v, NULL, NULL, 65), "capacity");
  refuse("no v", WRITE(&c, &t, &k, NULL, NULL, NULL, 3), "NULL v");
  WITH(skv_rotary_table, t, x.pairs = 129, WRITE(&c, &x, &k, &v, NULL, NULL, 3), "129 pairs", "pairs");
  WITH(skv_rotary_table, t, x.pairs = 0, WRITE(&c, &x, &k, &v, NULL, NULL, 3), "0 pairs", "pairs");
  WITH(skv_rotary_table, t, x.scale = NAN, WRITE(&c, &x, &k, &v, NULL, NULL, 3), "scale", "scale");
  WITH(skv_rotary_table, t, x.turns = NULL, WRITE(&c, &x, &k, &v, NULL, NULL, 3), "no turns", "turns");
  WITH(skv_rows, q, x.data = (char *)x.data + 512, WRITE(&c, &t, &k, &v, &q, &x, 3), "q_out beside q", "overlaps");
  WITH(skv_rows, qo, x.head_stride = 0, WRITE(&c, &t, &k, &v, &q, &x, 3), "q_out on itself", "overlap");
  WITH(skv_rows, qo, x.data = k.data, WRITE(&c, &t, &k, &v, &q, &x, 3), "q_out on k", "overlaps k or v");

  /* rotary */
  const skv_rows in = {arena + (8 << 20), 0, 512, 128}, other = {arena + (9 << 20), 0, 512, 128};
  const skv_rotary_table small = {t.turns, 32, 1, 1.0f};
  int64_t *at = (int64_t *)(arena + (23 << 20));
#define TURN(T, X, Y, TYPE, B, N, H, DIM, P, SB) skv_rotary(T, X, Y, TYPE, B, N, H, DIM, P, SB, 1, 0, NULL)
  accept("rotary", TURN(&small, &in, &other, SKV_FP16, 1, 5, 4, 128, at, 0));
  accept("rotary in place", TURN(&small, &in, &in, SKV_FP32, 1, 5, 4, 128, at, 0));
  refuse("no table", TURN(NULL, &in, &other, SKV_BF16, 1, 5, 4, 128, at, 0), "NULL rotary table");
  refuse("type", TURN(&small, &in, &other, 3, 1, 5, 4, 128, at, 0), "dtype");
  refuse("no tokens", TURN(&small, &in, &other, SKV_BF16, 1, 0, 4, 128, at, 0), "tokens");
  refuse("too many tokens", TURN(&small, &in, &other, SKV_BF16, 4, 1 << 30, 4, 128, at, 0), "tokens");
  refuse("too many heads", TURN(&small, &in, &other, SKV_BF16, 1, 5, 65536, 128, at, 0), "heads");
  refuse("dim", TURN(&small, &in, &other, SKV_BF16, 1, 5, 4, 1025, at, 0), "dimension");
  refuse("pairs past the head", TURN(&small, &in, &other, SKV_BF16, 1, 5, 4, 62, at, 0), "pairs");
  refuse("no positions", TURN(&small, &in, &other, SKV_BF16, 1, 5, 4, 128, NULL, 0), "NULL positions");
  refuse("overlapping positions", TURN(&small, &in, &other, SKV_BF16, 2, 5, 4, 128, at, 4), "position rows");
  refuse("short positions", TURN(&small, &in, &other, SKV_BF16, 1, 50, 4, 128, far, 0), "extends past");
  WITH(skv_rows, in, x.data = (char *)x.data + 256, TURN(&small, &in, &x, SKV_BF16, 1, 5, 4, 128, at, 0), "y beside x", "overlaps");
  WITH(skv_rows, other, x.token_stride = 128, TURN(&small, &in, &x, SKV_BF16, 1, 5, 4, 128, at, 0), "y on itself", "overlap");
  WITH(skv_rows, in, x.data = (char *)x.data + 2, TURN(&small, &x, &other, SKV_FP32, 1, 5, 4, 128, at, 0), "x by 2", "aligned");

  /* evict */
  skv_record_cache to = cache();
  to.records = arena + ((size_t)32 << 20);
  to.lengths = (int32_t *)(arena + (33 << 20));
  to.positions = (int32_t *)(arena + (34 << 20));
  to.weights = (float *)(arena + (35 << 20));
  const int64_t need = skv_evict_workspace(2, 64, 20);
#define EVICT(C, T, KEEP, SINK, LOCAL, S) skv_evict(C, T, KEEP, SINK, LOCAL, work, S, NULL)
  accept("evict", EVICT(&c, &to, 20, 4, 16, need));
  WITH(skv_record_cache, to, (x.positions = NULL, x.weights = NULL), (accept("records alone", EVICT(&p, &x, 20, 4, 16, need)), EVICT(&p, NULL, 20, 4, 16, need)), "no target", "NULL cache");
  refuse("sink + local past keep", EVICT(&c, &to, 20, 5, 16, need), "keep");
  refuse("sink < 0", EVICT(&c, &to, 20, -1, 16, need), "keep");
  refuse("sums past 32 bits", EVICT(&c, &to, 20, 2147483647, 2147483647, need), "keep");
  refuse("keep 0", EVICT(&c, &to, 0, 0, 0, need), "keep");
  refuse("keep past the capacity", EVICT(&c, &to, 65, 0, 0, need * 9), "capacity");
  refuse("small workspace", EVICT(&c, &to, 20, 4, 16, need - 1), "workspace");
  refuse("onto itself", EVICT(&c, &c, 20, 4, 16, need), "share records");
  WITH(skv_record_cache, to, x.records = (char *)c.records + 512, EVICT(&c, &x, 20, 4, 16, need), "shifted", "share records");
  WITH(skv_record_cache, to, x.weights = c.weights, EVICT(&c, &x, 20, 4, 16, need), "one weights", "share weights");
  WITH(skv_record_cache, to, x.lengths = c.lengths, EVICT(&c, &x, 20, 4, 16, need), "one lengths", "share weights");
  WITH(skv_record_cache, to, x.batch = 1, EVICT(&c, &x, 20, 4, 16, need), "batches", "sequences");
  WITH(skv_record_cache, c, x.weights = NULL, EVICT(&x, &to, 20, 4, 16, need), "no weights", "no weights");

  if (skv_tree_workspace(0, 3) || skv_tree_workspace(2, 65) || skv_evict_workspace(2, 64, 0) ||
      skv_evict_workspace(2, 0, 4) || skv_tree_workspace(1024, 64) <= 0)
    return 4;
  printf("records stub driver ok: %d checks\n", checks);
  return 0;
}
