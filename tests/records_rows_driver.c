/* Drives the checks of the record cache's entry points on how row tensors lie
 * to each other, over the stub of records_stub_driver.c.
 * tests/test_records_rows.py builds and runs it. */
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
  const skv_rotary_table t = {(const uint64_t *)(arena + (20 << 20)), 128, 0, 1.0f};
  const size_t M = 8 << 20;
#define PUT(K, V, Q, O, N) skv_cache_write(&c, &t, &K, &V, &Q, &O, N, NULL, 0, NULL, NULL)

  /* 3 tokens of 2 sequences, 24 heads a token (16 of q, 4 of k, 4 of v) */
  const int64_t st = 24 * 256, sb = 3 * st;
  const skv_rows q = at(M, sb, st, 256), k = at(M + 16 * 512, sb, st, 256), v = at(M + 20 * 512, sb, st, 256);
  const skv_rows last_of_q = at(M + 12 * 512, sb, st, 256), one_over = at(M + 15 * 512, sb, st, 256);
  const skv_rows before = at(M + 3 * 512, sb, st, 256), later = at(M + 4 * 2 * st, sb, st, 256);
  accept("fused rows in place", PUT(k, v, q, q, 3));
  accept("one token", PUT(k, v, q, q, 1));
  refuse("k in q", PUT(last_of_q, v, q, q, 3), "overlaps k or v");
  refuse("v in q", PUT(k, before, q, q, 3), "overlaps k or v");
  refuse("one head of k in q", PUT(one_over, v, q, q, 3), "overlaps k or v");
  refuse("k is q", PUT(q, v, q, q, 3), "overlaps k or v");
  refuse("k in another token's q", PUT(later, v, q, q, 3), "overlaps k or v");
  refuse("k in q, one token", PUT(one_over, v, q, q, 1), "overlaps k or v");

  /* heads before tokens */
  const int64_t hs = 3 * 256, hb = 24 * hs;
  const skv_rows hq = at(M, hb, 256, hs), hk = at(M + 16 * 2 * hs, hb, 256, hs), hv = at(M + 20 * 2 * hs, hb, 256, hs);
  const skv_rows hin = at(M + 15 * 2 * hs, hb, 256, hs);
  accept("heads first in place", PUT(hk, hv, hq, hq, 3));
  refuse("heads first, k in q", PUT(hin, hv, hq, hq, 3), "overlaps k or v");

  /* broadcast k and v, every other head of a row */
  const skv_rows bk = at(2 * M, 0, 0, 256), bv = at(2 * M + 2048, 0, 0, 0);
  accept("broadcast k and v", PUT(bk, bv, q, q, 3));
  const skv_rows even = at(M, 2 * 3 * 32 * 256, 32 * 256, 512), odd = at(M + 512, 2 * 3 * 32 * 256, 32 * 256, 512);
  accept("k between the heads of q", PUT(odd, bv, even, even, 3));
  const skv_rows part = at(M + 2, 2 * 3 * 32 * 256, 32 * 256, 512);
  refuse("k one element into q", PUT(part, bv, even, even, 3), "overlaps k or v");

  /* turned into another place of the fused rows */
  const skv_rows from = at(3 * M, 3 * 16 * 256, 16 * 256, 256);
  accept("q turned into the rows beside k and v", PUT(k, v, from, q, 3));
  refuse("q turned over k", PUT(one_over, v, from, q, 3), "overlaps k or v");

  /* rotary: heads beside heads, token rows beside token rows */
  const skv_rotary_table small = {t.turns, 32, 1, 1.0f};
#undef TURN
#define TURN(X, Y, B, N, H) skv_rotary(&small, &X, &Y, SKV_BF16, B, N, H, 256, positions, 0, 1, 0, NULL)
  int64_t *positions = (int64_t *)(arena + (23 << 20));
  const skv_rows heads = at(M, sb, st, 256), beside = at(M + 4 * 512, sb, st, 256), over = at(M + 3 * 512, sb, st, 256);
  accept("heads beside heads", TURN(heads, beside, 2, 3, 4));
  accept("one token's heads beside its heads", TURN(heads, beside, 1, 1, 4));
  refuse("heads over heads", TURN(heads, over, 2, 3, 4), "overlaps its input");
  const skv_rows first = at(M, 0, 2 * 1024, 256), second = at(M + 2048, 0, 2 * 1024, 256);
  accept("every other token", TURN(first, second, 1, 5, 4));
  refuse("every other token, 5 heads", TURN(first, second, 1, 5, 5), "overlaps its input");
  const skv_rows wide = at(M, sb, st, 256), narrow = at(M, sb, st, 512);
  refuse("the same start in another layout", TURN(wide, narrow, 2, 3, 4), "overlaps its input");

  /* strides whose reach wraps round 64 bits */
  const skv_rotary_table one = {t.turns, 1, 0, 1.0f};
  const int many = (1 << 25) + 1; /* times 2^39 elements */
  const skv_rows far_in = at(M, (int64_t)1 << 39, 2, 2), flat = at(3 * M, 2, 2, 2), all_one = at(3 * M, 0, 2, 2);
#define FAR(X, Y, B, N, P, SB) skv_rotary(&one, &X, &Y, SKV_BF16, B, N, 1, 2, P, SB, 1, 0, NULL)
  refuse("x and y wrap round", FAR(far_in, far_in, many, 1, positions, 0), "strides");
  refuse("y wraps round", FAR(all_one, far_in, many, 1, positions, 0), "strides");
  const skv_rows far_tokens = at(M, 0, (int64_t)1 << 39, 2);
  refuse("tokens wrap round", FAR(far_tokens, flat, 1, many, positions, 0), "");
  refuse("positions wrap round", FAR(flat, flat, 5, 1, positions, (int64_t)1 << 62), "position rows");
  refuse("positions wrap round in bytes", FAR(flat, flat, 5, 1, positions, (int64_t)1 << 59), "position rows");
  refuse("positions before their start", FAR(flat, flat, 5, 1, positions, -8), "position rows");

  /* positions that the write itself changes */
#define AT(C, P, WIDE) skv_cache_write(&C, &t, &k, &v, NULL, NULL, 3, P, WIDE, NULL, NULL)
  accept("positions of their own", AT(c, positions, 1));
  refuse("the cache's positions", AT(c, c.positions + 64, 0), "cache's own");
  refuse("into the cache's positions", AT(c, c.positions - 5, 0), "cache's own");
  refuse("64-bit ones there", AT(c, c.positions + 2 * 4 * 64 - 2, 1), "cache's own");
  accept("behind them", AT(c, c.positions + 2 * 4 * 64, 0));
  skv_record_cache plain = c;
  plain.positions = NULL;
  accept("a cache without", AT(plain, c.positions + 64, 0));

  printf("records rows driver ok: %d checks\n", checks);
  return 0;
}
