// Rotary positions, alone and on the way into a record cache.
//
// A pair (a, b) of a head at position p becomes s (a cos t - b sin t, b cos t +
// a sin t) with t = p inv_i.  inv_i is held in 2^-64 turns, so p inv_i modulo
// a turn is one wrapping 64-bit product, exact for any position where an FP32
// angle would be off by p 2^-24 radians; its top 32 bits are the angle.
//
// Both kernels are bound by memory.  A thread owns 8 pairs (two 16-byte loads
// in BF16) of one token and keeps their sines and cosines in registers while
// it walks the heads, so they are formed once per token and not once per
// head; few tokens are spread over the chip by splitting the heads.  4 heads
// are in flight at once.  32768 tokens x 20 heads x 256 in BF16: 139 us, 4.8
// TB/s (torch's copy of as many bytes: 160 us); 32768 tokens into a cache with
// their queries: 175 us, 4.2 TB/s (188 with one row in flight); a single
// token of 8 sequences 4.4 us, the launch.
//
// Where the turned part is no multiple of 16 elements, or rows or strides are
// not 16-byte aligned, every access is one element (N = 1): 34 of 256 elements
// of those 32768 x 20 heads 340 us (32 of 256: 226, mostly the copy of what is
// not turned; in place 34 against 22), written with their queries 404 (32: 181).
#include "skv_cache.h"
#include "skv_device.h"

namespace skv {

namespace {

constexpr double PI = 3.14159265358979323846;
constexpr int RO_BLOCK = 256;
constexpr int RO_TARGET_BLOCKS = 2048;  // 8 blocks of 4 waves on each of 256 CUs

__device__ __forceinline__ int64_t position_of(const RotaryArgs& r, int b, int i) {
  const int64_t at = (int64_t)b * r.position_sb + i;
  return r.positions64 ? static_cast<const int64_t*>(r.positions)[at]
                       : static_cast<const int32_t*>(r.positions)[at];
}

// scale (cos, sin) of `turns` 2^-64 turns per position at position p.  The
// angle is brought within an eighth of a turn of a quarter's multiple before it
// becomes FP32 (off by pi 2^-27 then, a whole half turn by pi 2^-25), where the
// series of sin pi r and cos pi r end after r^9 and r^10, within 2e-9 and 2e-10;
// pi is two words, so a rounding of the sine is one of its last sum.  Off by at
// most 7.3e-8 in all (4e6 angles), and fewer instructions than a function that
// reduces its argument once more (5003 x 7 rows of 48 FP32 elements: 8.8 us, 9.4
// with one).
__device__ __forceinline__ float2 turn(uint64_t turns, int64_t p, float scale) {
  const uint32_t hi = (uint32_t)((turns * (uint64_t)p) >> 32);  // 2^-32 turns
  const uint32_t quarters = (hi + (1u << 29)) >> 30;
  const float r = (float)(int)(hi << 2) * 0x1p-33f;  // (the low 30 bits, signed)
  const float t = r * r;
  constexpr double PI2 = PI * PI;
  constexpr float PI_HI = (float)PI, PI_LO = (float)(PI - PI_HI);
  constexpr float S3 = (float)(-PI * PI2 / 6), S5 = (float)(PI * PI2 * PI2 / 120),
                  S7 = (float)(-PI * PI2 * PI2 * PI2 / 5040), S9 = (float)(PI * PI2 * PI2 * PI2 * PI2 / 362880);
  constexpr float C2 = (float)(-PI2 / 2), C4 = (float)(PI2 * PI2 / 24), C6 = (float)(-PI2 * PI2 * PI2 / 720),
                  C8 = (float)(PI2 * PI2 * PI2 * PI2 / 40320),
                  C10 = (float)(-PI2 * PI2 * PI2 * PI2 * PI2 / 3628800);
  const float s = fmaf(r, PI_HI, r * fmaf(t, fmaf(t, fmaf(t, fmaf(t, S9, S7), S5), S3), PI_LO));
  const float c = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, C10, C8), C6), C4), C2), 1.f);
  const float a = quarters & 1 ? s : c, b = quarters & 1 ? c : s;
  const float cosine = __uint_as_float(__float_as_uint(a) ^ ((quarters + 1) & 2) << 30);
  const float sine = __uint_as_float(__float_as_uint(b) ^ (quarters & 2) << 30);
  return make_float2(cosine * scale, sine * scale);
}

struct BF16 { uint16_t u; };
struct FP16 { _Float16 h; };

__device__ __forceinline__ float load1(const BF16* p) { return bf16_f32(p->u); }
__device__ __forceinline__ float load1(const FP16* p) { return (float)p->h; }
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ void store1(BF16* p, float f) { p->u = (uint16_t)bf16_rne(f); }
__device__ __forceinline__ void store1(FP16* p, float f) { p->h = (_Float16)f; }
__device__ __forceinline__ void store1(float* p, float f) { *p = f; }

// Eight 16-byte aligned elements.
__device__ __forceinline__ void load8(const BF16* p, float f[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16_f32(u[i] & 0xffffu);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const FP16* p, float f[8]) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  const h8 v = *reinterpret_cast<const h8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
}
__device__ __forceinline__ void load8(const float* p, float f[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void store8(BF16* p, const float f[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = bf16_rne(f[2 * i]) | bf16_rne(f[2 * i + 1]) << 16;
  *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(FP16* p, const float f[8]) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  h8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (_Float16)f[i];
  *reinterpret_cast<h8*>(p) = v;
}
__device__ __forceinline__ void store8(float* p, const float f[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// Unit u of a head: N pairs (u < pairs / N), or N elements past the turned
// ones.  N = 8 where rows and pairs are multiples of 8 elements, else 1.  A
// unit's first elements lie at lo, its pairs' second at hi (half layout);
// interleaved pairs fill [lo, lo + 2 N).
template <int N, bool INTER>
struct Unit {
  int lo, hi, pair;
  bool turned;
  __device__ Unit(int u, int pairs) {
    const int first = pairs / N;
    turned = u < first;
    pair = u * N;
    lo = turned ? (INTER ? 2 * pair : pair) : 2 * pairs + (u - first) * N;
    hi = INTER ? lo + N : pairs + pair;
  }
};

template <int N, typename T>
__device__ __forceinline__ void loadn(const T* p, float f[N]) {
  if constexpr (N == 8) load8(p, f);
  else f[0] = load1(p);
}
template <int N, typename T>
__device__ __forceinline__ void storen(T* p, const float f[N]) {
  if constexpr (N == 8) store8(p, f);
  else store1(p, f[0]);
}

// The 2 N elements of a unit (x: at lo, y: at hi) turned in place.
template <int N, bool INTER>
__device__ __forceinline__ void turn_unit(float x[N], float y[N], const float2 cs[N]) {
  if constexpr (!INTER || N == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float a = x[i], b = y[i];
      x[i] = fmaf(a, cs[i].x, -(b * cs[i].y));
      y[i] = fmaf(b, cs[i].x, a * cs[i].y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = fmaf(a, cs[i].x, -(b * cs[i].y));
      x[2 * i + 1] = fmaf(b, cs[i].x, a * cs[i].y);
      a = y[2 * i];
      b = y[2 * i + 1];
      y[2 * i] = fmaf(a, cs[N / 2 + i].x, -(b * cs[N / 2 + i].y));
      y[2 * i + 1] = fmaf(b, cs[N / 2 + i].x, a * cs[N / 2 + i].y);
    }
  }
}

template <int N>
__device__ __forceinline__ void unit_turns(const RotaryArgs& r, int pair, int64_t p, float sign,
                                           float2 cs[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    cs[i] = turn(r.turns[pair + i], p, r.scale);
    cs[i].y *= sign;
  }
}

// Thread: unit of a token (grid x), heads h0 .. h0 + per - 1 (grid y).
template <typename T, int N, bool INTER>
__global__ __launch_bounds__(RO_BLOCK) void k_rotary(RotaryArgs r, Rows x, Rows y, int64_t items,
                                                     int units, int n, int heads, int per,
                                                     float sign) {
  const int64_t item = (int64_t)blockIdx.x * RO_BLOCK + threadIdx.x;
  if (item >= items) return;
  const int64_t token = item / units;
  const int b = (int)(token / n), i = (int)(token % n);
  const Unit<N, INTER> u((int)(item % units), r.pairs);
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
  const T* in = static_cast<const T*>(x.data) + b * x.sb + i * x.st + h0 * x.sh;
  T* out = const_cast<T*>(static_cast<const T*>(y.data)) + b * y.sb + i * y.st + h0 * y.sh;
  if (!u.turned) {
    for (int h = h0; h < h1; ++h, in += x.sh, out += y.sh) {
      float f[N];
      loadn<N>(in + u.lo, f);
      storen<N>(out + u.lo, f);
    }
    return;
  }
  float2 cs[N];
  unit_turns<N>(r, u.pair, position_of(r, b, i), sign, cs);
#pragma unroll 4
  for (int h = h0; h < h1; ++h, in += x.sh, out += y.sh) {
    float f[N], g[N];
    loadn<N>(in + u.lo, f);
    loadn<N>(in + u.hi, g);
    turn_unit<N, INTER>(f, g, cs);
    storen<N>(out + u.lo, f);
    storen<N>(out + u.hi, g);
  }
}

// FP8 bytes of N values at p.
template <int N>
__device__ __forceinline__ void store_fp8(uint8_t* p, const float f[N]) {
  if constexpr (N == 8) {
    int w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], w[i], true);
    }
    *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)w[0], (uint32_t)w[1]);
  } else {
    p[0] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[0], 0.f, 0, false);
  }
}

// The rows of a token in the order that the threads walk them: query heads, K
// heads, V heads.
constexpr int WR_Q = G * H, WR_K = WR_Q + G, WR_ROWS = WR_K + G;

// Thread: unit of a token (grid x), rows r0 .. r0 + per - 1 of the token (grid
// y; without queries they start at the K heads).
template <int N, bool INTER>
__global__ __launch_bounds__(RO_BLOCK) void k_cache_write(WriteArgs a, int64_t items, int units,
                                                          int first, int per) {
  const int64_t item = (int64_t)blockIdx.x * RO_BLOCK + threadIdx.x;
  if (item >= items) return;
  const int64_t token = item / units;
  const int b = (int)(token / a.n), i = (int)(token % a.n), unit = (int)(item % units);
  const Unit<N, INTER> u(unit, a.r.pairs);
  const int r0 = first + blockIdx.y * per, r1 = min(r0 + per, WR_ROWS);
  const int slot = a.c.length(b) + i;
  const bool wanted = !a.counts || i < a.counts[b];
  const bool fits = wanted && slot < a.c.capacity;
  uint32_t page = 0;
  bool held = fits;
  if (fits && a.c.table) {
    page = a.c.page(b, slot);
    held = page < a.c.n_pages;
  }
  const int64_t p = a.r.positions ? position_of(a.r, b, i) : slot;
  float2 cs[N];
  if (u.turned) unit_turns<N>(a.r, u.pair, p, 1.f, cs);
  auto source = [&](const Rows& r, int h) {
    return static_cast<const BF16*>(r.data) + b * r.sb + i * r.st + h * r.sh;
  };
  auto record = [&](int g) {
    return a.c.records + (a.c.table ? a.c.row_in(page, g, slot) : a.c.row(b, g, slot)) * 512;
  };
#pragma unroll 4
  for (int row = r0; row < min(r1, WR_Q); ++row) {
    const BF16* in = source(a.q, row);
    BF16* out = const_cast<BF16*>(source(a.q_out, row));
    float f[N], g[N];
    loadn<N>(in + u.lo, f);
    if (u.turned) {
      loadn<N>(in + u.hi, g);
      turn_unit<N, INTER>(f, g, cs);
      storen<N>(out + u.hi, g);
    }
    storen<N>(out + u.lo, f);
  }
  if (held) {
#pragma unroll 4
    for (int row = max(r0, WR_Q); row < min(r1, WR_K); ++row) {
      const BF16* in = source(a.k, row - WR_Q);
      uint8_t* out = record(row - WR_Q) + 256;
      float f[N], g[N];
      loadn<N>(in + u.lo, f);
      if (u.turned) {
        loadn<N>(in + u.hi, g);
        turn_unit<N, INTER>(f, g, cs);
        store_fp8<N>(out + u.hi, g);
      }
      store_fp8<N>(out + u.lo, f);
    }
#pragma unroll 4
    for (int row = max(r0, WR_K); row < r1; ++row) {
      const BF16* in = source(a.v, row - WR_K);
      uint8_t* out = record(row - WR_K);
      for (int e = N * unit; e < D; e += N * units) {
        float f[N];
        loadn<N>(in + e, f);
        store_fp8<N>(out + e, f);
      }
    }
  }
  if (unit == 0 && blockIdx.y == 0) {
    if (held) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const size_t at = a.c.row(b, g, slot);
        if (a.positions) a.positions[at] = (int)p;
        if (a.weights) a.weights[at] = 0.f;
      }
    } else if (wanted && a.status) {
      atomicOr(a.status, fits ? STATUS_PAGE : STATUS_CAPACITY);
    }
  }
}

bool rows_by_8(const Rows& r, int size) {
  return ((uintptr_t)r.data & 15) == 0 && r.sb * size % 16 == 0 && r.st * size % 16 == 0 &&
         r.sh * size % 16 == 0;
}

// Splits of `rows` rows per token over grid y, for `blocks` blocks in x.
int split_rows(int64_t blocks, int rows, int& per) {
  int64_t splits = (RO_TARGET_BLOCKS + blocks - 1) / blocks;
  if (splits > rows) splits = rows;
  per = (rows + (int)splits - 1) / (int)splits;
  return (rows + per - 1) / per;
}

template <typename T, int N, bool INTER>
void rotary_rows(const RotaryArgs& a, bool transpose, const Rows& x, const Rows& y, int batch, int n,
                 int heads, int dim, hipStream_t st) {
  // in place the elements past the turned ones stay as they are
  const int units = a.pairs / N + (x.data == y.data ? 0 : (dim - 2 * a.pairs) / N);
  const int64_t items = (int64_t)batch * n * units;
  const int64_t blocks = (items + RO_BLOCK - 1) / RO_BLOCK;
  int per;
  const int splits = split_rows(blocks, heads, per);
  hipLaunchKernelGGL((k_rotary<T, N, INTER>), dim3((unsigned)blocks, splits), dim3(RO_BLOCK), 0, st,
                     a, x, y, items, units, n, heads, per, transpose ? -1.f : 1.f);
}

template <typename T>
void rotary_typed(const RotaryArgs& a, bool interleaved, bool transpose, const Rows& x,
                  const Rows& y, int batch, int n, int heads, int dim, hipStream_t st) {
  const bool by8 = a.pairs % 8 == 0 && dim % 8 == 0 && rows_by_8(x, sizeof(T)) && rows_by_8(y, sizeof(T));
  auto run = by8 ? (interleaved ? rotary_rows<T, 8, true> : rotary_rows<T, 8, false>)
                 : (interleaved ? rotary_rows<T, 1, true> : rotary_rows<T, 1, false>);
  run(a, transpose, x, y, batch, n, heads, dim, st);
}

}  // namespace

void launch_rotary(const RotaryArgs& a, bool interleaved, bool transpose, const Rows& x,
                   const Rows& y, int dtype, int batch, int n, int heads, int dim, hipStream_t st) {
  auto run = dtype == 0 ? rotary_typed<BF16> : dtype == 1 ? rotary_typed<FP16> : rotary_typed<float>;
  run(a, interleaved, transpose, x, y, batch, n, heads, dim, st);
}

void launch_cache_write(const WriteArgs& a, hipStream_t st) {
  const bool by8 = a.r.pairs % 8 == 0 && rows_by_8(a.k, 2) && rows_by_8(a.v, 2) &&
                   (!a.q.data || (rows_by_8(a.q, 2) && rows_by_8(a.q_out, 2)));
  const int step = by8 ? 8 : 1;
  const int units = a.r.pairs / step + (D - 2 * a.r.pairs) / step;
  const int64_t items = (int64_t)a.c.batch * a.n * units;
  const int64_t blocks = (items + RO_BLOCK - 1) / RO_BLOCK;
  const int first = a.q.data ? 0 : WR_Q;
  int per;
  const int splits = split_rows(blocks, WR_ROWS - first, per);
  auto kernel = by8 ? (a.interleaved ? k_cache_write<8, true> : k_cache_write<8, false>)
                    : (a.interleaved ? k_cache_write<1, true> : k_cache_write<1, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, splits), dim3(RO_BLOCK), 0, st, a, items, units,
                     first, per);
}

}  // namespace skv
