/* The launches of the norm gradient over the stub of records_stub_driver.c:
 * their grids against the workspace and the heads.
 * tests/test_norm_grid.py builds and runs it. */
int stub_main(void);
#define main stub_main
#define hipLaunchKernel stub_launch
#include "records_stub_driver.c"
#undef main
#undef hipLaunchKernel

static dim3 grids[2];
static int per, shares;

/* k_norm_grad(r, w, g, x, y, tokens, units, n, heads, dim, per, ..), then
 * k_norm_weight(partial, shares, ..) */
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t shared, hipStream_t st) {
  if (launches < 2) grids[launches] = g;
  if (launches == 0) per = *(int *)args[10];
  if (launches == 1) shares = *(int *)args[1];
  return stub_launch(f, g, b, args, shared, st);
}

static void fail(const char *what, int tokens, int heads, int dim, int each) {
  fprintf(stderr, "FAILED %s: %d tokens, %d heads, dim %d, per_head %d: grid %u x %u of %d heads, %d shares\n", what,
          tokens, heads, dim, each, grids[0].x, grids[0].y, per, shares);
  exit(2);
}

int main(void) {
  arena = aligned_alloc(4096, ARENA);
  if (!arena) return 3;
  const int tokens[] = {1, 2, 3, 7, 16, 100, 1000, 8192}, heads[] = {1, 2, 3, 5, 20, 300, 1023, 1025, 4097, 65535};
  /* 4 and 2 heads in flight, of rows in 16-byte pieces and not */
  const struct { int dim, step, batch; } forms[] = {{16, 16, 4}, {128, 128, 4}, {256, 256, 4}, {520, 520, 2},
                                                    {16, 17, 4}, {30, 30, 4},   {250, 251, 4}, {300, 301, 2}};
  for (unsigned f = 0; f < sizeof forms / sizeof *forms; ++f)
    for (int i = 0; i < 8; ++i)
      for (int j = 0; j < 10; ++j)
        for (int each = 0; each < 2; ++each) {
          const int dim = forms[f].dim, n = tokens[i], h = heads[j];
          const int64_t row = (int64_t)h * forms[f].step, bytes = n * row * 2;
          const int64_t size = skv_norm_grad_workspace(n, h, dim, each);
          if (bytes > (4 << 20) || size > (16 << 20) || (each ? h : 1) * dim * 4 > (8 << 20)) continue;
          const skv_rows x = {arena, 0, row, forms[f].step}, g = {arena + (8 << 20), 0, row, forms[f].step},
                         y = {arena + (16 << 20), 0, row, forms[f].step};
          const skv_rotary_table t = {(const uint64_t *)(arena + (24 << 20)), dim >= 16 && dim % 16 == 0 ? 8 : 1, 0, 1.0f};
          const skv_head_norm w = {arena + (26 << 20), SKV_FP32, each, 1e-6f};
          const int code = skv_norm_rotary_grad(&t, &w, &g, &x, &y, SKV_BF16, 1, n, h, dim, arena + (25 << 20), 0, 0,
                                                arena + (40 << 20), arena + (48 << 20), size, NULL);
          if (launches != 2) fail(skv_last_error(NULL), n, h, dim, each);
          accept("gradient", code);
          const int64_t rows = (int64_t)grids[0].x * grids[0].y;
          if (rows * dim * 4 > size) fail("partial sums past the workspace", n, h, dim, each);
          if (rows != (int64_t)shares * (each ? h : 1)) fail("shares", n, h, dim, each);
          if ((int64_t)per * grids[0].y < h) fail("heads left out", n, h, dim, each);
          if ((int64_t)per * (grids[0].y - 1) >= h) fail("a block without heads", n, h, dim, each);
          if (per % (each ? 1 : forms[f].batch)) fail("heads in flight are no whole number", n, h, dim, each);
        }
  if (checks < 500) return 4;
  printf("norm grid driver ok: %d checks\n", checks);
  return 0;
}
