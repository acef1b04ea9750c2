/* Drives the checks of a chain's attention on how its results lie to its
 * queries, over the stub of records_stub_driver.c.
 * tests/test_attend_rows.py builds and runs it. */
int stub_main(void);
#define main stub_main
#include "records_stub_driver.c"
#undef main

static skv_rows at(size_t base, int64_t sb, int64_t st, int64_t sh) {
  skv_rows r = {arena + base, sb, st, sh};
  return r;
}

int main(void) {
  arena = aligned_alloc(4096, ARENA);
  if (!arena) return 3;
  skv_record_cache c = cache();
  c.batch = 1;
  c.capacity = 4096; /* 8 MB of records */
  c.lengths = (int32_t *)(arena + (9 << 20));
  c.positions = NULL;
  c.weights = NULL;
  c.status = NULL;
  const size_t M = 16 << 20;
  enum { N = 1536 };
  const int64_t st = 16 * 256;
  const size_t rows = (size_t)N * st * 2;
  const skv_rows q = at(M, 0, st, 256);
  float *lse = (float *)(arena + (10 << 20));
#define ATTEND(Q, COUNT, OUT, LSE) skv_attend(&c, Q, COUNT, NULL, 0.f, 0, 0, OUT, LSE, arena, 0, NULL)
  /* (its workspace is larger than the stub's memory: refused last) */
#define APART "a workspace of 0 bytes"
  refuse("results beside the queries", ATTEND(&q, N, arena + M + rows, lse), APART);
  refuse("in place", ATTEND(&q, N, arena + M, lse), APART);
  refuse("a token on", ATTEND(&q, N, arena + M + 2 * st, lse), "out overlaps its input");
  refuse("a token back", ATTEND(&q, N, arena + M - 2 * st, lse), "out overlaps its input");
  refuse("a head on", ATTEND(&q, N, arena + M + 512, lse), "out overlaps its input");
  refuse("the last row", ATTEND(&q, N, arena + M + rows - 16, lse), "out overlaps its input");

  /* queries that are heads of fused rows, results over their storage */
  const skv_rows fused = at(M, 0, 24 * 256, 256);
  refuse("over the fused rows", ATTEND(&fused, N, arena + M, lse), "out overlaps its input");
  refuse("behind the fused rows", ATTEND(&fused, N, arena + M + (size_t)N * 24 * 512, lse), APART);

  /* lse in the queries */
  refuse("lse in q", ATTEND(&q, N, arena + M + rows, (float *)(arena + M + 4096)), "lse overlaps q");
  refuse("lse before q", ATTEND(&q, N, arena + M + rows, (float *)(arena + M - (size_t)N * 64)), APART);
  refuse("lse into q", ATTEND(&q, N, arena + M + rows, (float *)(arena + M - (size_t)N * 64 + 4)), "lse overlaps q");

  /* few tokens are read by one kernel and written by the next */
  void *work = arena + (40 << 20);
  const int64_t size = skv_tree_workspace(1, 8);
#define FEW(Q, OUT) skv_attend(&c, Q, 8, NULL, 0.f, 0, 0, OUT, lse, work, size, NULL)
  accept("8 tokens, a token on", FEW(&q, arena + M + 2 * st));
  accept("8 fused tokens", FEW(&fused, arena + M));
  printf("attend rows driver ok: %d checks\n", checks);
  return 0;
}
