// Attention of drafted tokens over a record cache, and the attention weight
// of its keys (interfaces in skv_cache.h).
//
// Rows: the 4 query heads of KV head g for each of n drafts, row 4 i + h.  A
// wave holds 16 RT of them as matrix-core columns and walks pairs of 16-key
// tiles.  Scores: K is widened from FP8 to BF16 (exact) and multiplied by the
// BF16 queries as they are.  (FP8 products of 128 dims at a time would take K
// as stored, but that instruction drops bits of small products: sums of 256
// were off by up to 9e-6 of the sum of magnitudes, BF16 ones by none.)
// Sums: the lane that holds a score also needs it as column operand of
// softmax x V, so nothing moves between lanes; V is widened to FP16 (exact)
// and a probability is rounded once to FP16, by at most 2^-11 of itself (the
// running maximum sits at 2^7 .. 2^15, so terms down to 2^-31 of it count;
// BF16 would be off by 2^-8, as much as the result's own rounding).  Sums,
// maxima and row totals are FP32.
//
// The sequences' pairs lie in one row, cut into equal shares, one per block:
// a batch of ragged sequences loads every CU alike.  A share that spans
// sequences leaves one partial in each; k_tree_merge joins a sequence's.
//
// Bounds (131072 keys, contiguous, whole calls on one cache over and over): one
// to 4 drafts 49 us (51 where several caches take turns), of which the kernel
// 44, 6.0 TB/s, the record stream; 8 drafts 54, 16 66 (73 in turns): the wait for
// records, since 256 registers a wave leave 8 waves a CU and one pair ahead; 32
// drafts 93, 64 drafts 154, with a cap 174: multiplying and weighing, which two
// waves a SIMD overlap little (loads two or three steps ahead changed nothing
// there).  One draft of many ragged paged sequences: 64 of up to 8192 keys
// (279530 in all) 113 us, 5.1 TB/s, 256 of up to 4096 (504279) 195 us, 5.3 TB/s:
// a share holds pieces of several sequences, each with queries to stage and a
// partial to store.  Loads pay where no wait stands between their issue and
// their use: see the loops' notes on branches and spills (7 to 9 registers of
// the two-tile instances are spilled, outside those loops).
#include <type_traits>

#include "skv_cache.h"
#include "skv_device.h"
#include "skv_tile.h"

namespace skv {

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

constexpr int TR_PAIR = 32;      // keys per step of a wave
constexpr int TR_BLOCKS = 64;    // shares per KV head: one block per CU
constexpr float TR_LN2 = 0.6931471805599453f;
// Scaled probabilities are 2^(z - m), z in log2 units, and m is moved to 7
// below a row's largest score when one exceeds m by more than 15.
constexpr float TR_BASE = 7.f, TR_MOST = 15.f;

// What a sequence has: rows of drafts, slots that some row may see.
struct Sequence {
  int len, drafts, keys, rows;
  __device__ Sequence(const CacheView& c, const int* counts, int n, int b) {
    len = c.length(b);
    const int k = counts ? min(max(counts[b], 0), n) : n;
    rows = H * k;
    drafts = min(k, c.capacity - len);
    keys = len + drafts;
  }
  // The drafts that are there, as a mask.
  __device__ __forceinline__ uint64_t there() const { return drafts < 64 ? (1ull << max(drafts, 0)) - 1ull : ~0ull; }
  // The same in scalar registers, for a sequence that the whole wave is at.
  __device__ Sequence uniform() const {
    Sequence s = *this;
    s.len = __builtin_amdgcn_readfirstlane(len);
    s.drafts = __builtin_amdgcn_readfirstlane(drafts);
    s.keys = __builtin_amdgcn_readfirstlane(keys);
    s.rows = __builtin_amdgcn_readfirstlane(rows);
    return s;
  }
};

// Pairs of a sequence; with WHOLE one without rows counts too.
template <bool WHOLE>
__device__ __forceinline__ int sequence_pairs(const Sequence& s) {
  return WHOLE || s.rows ? (s.keys + TR_PAIR - 1) / TR_PAIR : 0;
}

// s_start[b]: pairs of the sequences before b; s_start[batch]: all.
template <bool WHOLE>
__device__ __forceinline__ int sequence_starts(const CacheView& c, const int* counts, int n, int* s_start) {
  if (threadIdx.x < WAVE) {
    int carry = 0;
    for (int b0 = 0; b0 < c.batch; b0 += WAVE) {
      const int b = b0 + threadIdx.x;
      const int pairs = b < c.batch ? sequence_pairs<WHOLE>(Sequence(c, counts, n, b)) : 0;
      const int inc = wave_incl_scan(pairs);
      if (b < c.batch) s_start[b] = carry + inc - pairs;
      carry += __builtin_amdgcn_readlane(inc, WAVE - 1);
    }
    if (threadIdx.x == 0) s_start[c.batch] = carry;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(s_start[c.batch]);
}

// Block k's share of `total` pairs begins here (k of `blocks`, blocks <= total).
__host__ __device__ __forceinline__ int share_start(int total, int blocks, int k) {
  return (int)((int64_t)total * k / blocks);
}
// The share that holds pair p.
__device__ __forceinline__ int share_of(int total, int blocks, int p) {
  return (int)((((int64_t)p + 1) * blocks - 1) / total);
}

// The sequence that holds pair p: the last one that starts at or before it.
__device__ __forceinline__ int sequence_of(const int* s_start, int batch, int p) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_start[mid] <= p) lo = mid;
    else hi = mid;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The 16 keys from slot t on (t a multiple of 16): where they lie, the last of
// them in reach, and whether their page is none: they are invisible then, the
// pool's first 16 records are read in their place.
struct Tile {
  const uint8_t* at;
  int last;
  bool bad;
};
template <bool PAGED>
__device__ __forceinline__ Tile tile_at(const CacheView& c, int b, int g, int t, int keys) {
  const int ta = min(t, (keys - 1) & ~15);  // a second tile past the end is the last again, masked
  Tile x;
  x.last = min(15, keys - 1 - ta);
  x.bad = false;
  if constexpr (PAGED) {
    // a scalar load: a vector load's wait would be one for the records in
    // flight too
    typedef const __attribute__((address_space(4))) uint32_t* scalar;
    const uint32_t page = reinterpret_cast<scalar>(reinterpret_cast<uintptr_t>(
        c.table + (size_t)b * c.table_len))[ta >> c.shift];
    x.bad = page >= c.n_pages;
    x.at = c.records + (x.bad ? 0 : c.row_in(page, g, ta) * 512);
  } else {
    x.at = c.records + c.row(b, g, ta) * 512;
  }
  return x;
}

// WHOLE: all 16 keys are in reach.
template <bool WHOLE>
__device__ __forceinline__ void load_k(uint4 (&k)[4], const Tile& x, int lane) {
  const uint32_t at = (WHOLE ? lane & 15 : min(lane & 15, x.last)) * 512 + (lane >> 4) * 16;
#pragma unroll
  for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const uint4*>(x.at + 256 + 64 * j + at);
}
// ONCE: no other wave reads the tile.  Where two row waves do, streaming loads
// brought a fifth of the records from memory twice (12 drafts of 24 ragged
// sequences: 557 MB and 124 us, 455 MB and 118 us with plain ones).
template <bool WHOLE, bool ONCE>
__device__ __forceinline__ void load_v(uint4 (&v)[4], const Tile& x, int lane) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 4 * (lane >> 4) + r;
    const uint8_t* at = x.at + (uint32_t)((WHOLE ? row : min(row, x.last)) * 512 + 16 * (lane & 15));
    v[r] = ONCE ? load_stream(at) : *reinterpret_cast<const uint4*>(at);
  }
}

// ---------------------------------------------------------------- queries
// The score step's column operands of 16 rows: [step][lane] 16 bytes, the dims
// step_dim(step, kb) .. +7 of row col for lane 16 kb + col.
constexpr int STEPS = D / 32;
constexpr int IMG_TILE = STEPS * WAVE;  // uint4 per 16 rows

// Step 2 j + half takes the dims that half `half` of a lane's K word j holds.
__device__ __forceinline__ int step_dim(int step, int kb) {
  return 64 * (step >> 1) + 16 * kb + 8 * (step & 1);
}

// Copies the rows of a sequence into the image of `tiles` tiles; rows past
// `rows` are 0.
template <int THREADS>
__device__ __forceinline__ void stage_queries(const Rows& q, int b, int g, int tiles, int rows, uint4* img) {
  for (int at = threadIdx.x; at < tiles * IMG_TILE; at += THREADS) {
    const int lane = at & 63, step = (at >> 6) & (STEPS - 1), row = (at / IMG_TILE) * 16 + (lane & 15);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (row < rows)
      w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q.data) + b * q.sb +
                                          (row / H) * q.st + (g * H + row % H) * q.sh +
                                          step_dim(step, lane >> 4));
    img[at] = w;
  }
}

template <bool HI>
__device__ __forceinline__ v2bf fp8_bf16x2(uint32_t w) {
  return __builtin_bit_cast(v2bf, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, HI));
}

// The row operand of a step from its 8 FP8 bytes.
__device__ __forceinline__ v8bf k_operand(uint32_t lo, uint32_t hi) {
  const v2bf p[4] = {fp8_bf16x2<false>(lo), fp8_bf16x2<true>(lo), fp8_bf16x2<false>(hi), fp8_bf16x2<true>(hi)};
  return v8bf{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
}

// q . k of two tiles of 16 keys (lane: keys 4 kb + r) for RT tiles of 16 rows
// (lane: row col).
template <int RT>
__device__ __forceinline__ void scores(const uint4 (&k)[2][4], const uint4* img, int lane, v4f (&acc)[RT][2]) {
  // the image is read from LDS for every pair: held in registers it would
  // leave too few for the records in flight
  asm volatile("" : "+v"(lane));
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt][0] = acc[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int step = 0; step < STEPS; ++step) {
    v8bf a[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint4 w = k[x][step >> 1];
      a[x] = (step & 1) ? k_operand(w.z, w.w) : k_operand(w.x, w.y);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const v8bf q = __builtin_bit_cast(v8bf, img[rt * IMG_TILE + step * WAVE + lane]);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        acc[rt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[x], q, acc[rt][x], 0, 0, 0);
    }
    if (step & 1) __builtin_amdgcn_sched_barrier(0);  // two steps' operands live at a time
  }
}

// Scores in log2 units are s unit; s is q . k, or with a cap q . k put through
// cap tanh(x / cap) in units of q . k, x = q . k / 16.
struct ScoreScale {
  float unit;
  float in, out;  // x / cap = in q . k; cap in units of q . k
  __device__ explicit ScoreScale(float cap) {
    unit = 0.0625f * DN_LOG2E;
    in = cap > 0.f ? 0.0625f / cap : 0.f;
    out = 16.f * cap;
  }
  // Caps the scores of two tiles of 16 keys.  Up to half the cap 7 terms of the
  // series are exact to 9e-8; where all of a wave's scores are, as is usual,
  // the exponential and the reciprocal are not needed.
  __device__ __forceinline__ void squash(v4f (&s)[2]) const {
    // tanh x = x (1 + T[0] x^2 + T[1] x^4 + ..)
    constexpr float T[6] = {-1.f / 3.f, 2.f / 15.f, -17.f / 315.f, 62.f / 2835.f, -1382.f / 155925.f,
                            21844.f / 6081075.f};
    float most = 0.f, x[8], t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s[e >> 2][e & 3] * in;
      most = fmaxf(most, fabsf(x[e]));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = x[e] * x[e];
      t[e] = x[e] * fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, T[5], T[4]), T[3]), T[2]), T[1]), T[0]), 1.f);
    }
    if (__ballot(!(most < 0.5f))) {  // (fmaxf drops NaN, which the series passes on)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ax = fabsf(x[e]);
        const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(ax * (2.f * DN_LOG2E)) + 1.f), 1.f);
        t[e] = ax >= 0.5f ? copysignf(far, x[e]) : t[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] = out * t[e];
  }
};

// Drafts that row 4 i + h of a sequence sees, one bit each.
__device__ __forceinline__ uint64_t row_mask(const int64_t* tree, int n, int b, int i) {
  if (tree) return (uint64_t)tree[(size_t)b * n + i];
  return ((2ull << i) - 1ull);
}

// Whether the key in slot t is visible to a row with mask `bits`.
__device__ __forceinline__ bool sees(const Sequence& s, uint64_t bits, int t) {
  const int j = t - s.len;
  return j < 0 || (j < s.drafts && ((bits >> j) & 1ull));
}

// 0x80 in every byte of w that is an FP8 NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

template <bool HI>
__device__ __forceinline__ v2h fp8_f16x2(uint32_t w) {
  return __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, HI));
}

// Of a tile's V (lane 16 kb + c: dims 16 c .. +15 of keys 4 kb + r), dims 16 c +
// 4 w + i of the 4 keys, transposed and widened: half i's 4 values.
__device__ __forceinline__ void v_halves(const uint4 (&v)[4], int w, uint2 (&half)[4]) {
  const uint32_t y[4] = {(&v[0].x)[w], (&v[1].x)[w], (&v[2].x)[w], (&v[3].x)[w]};
  const uint32_t lo01 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u);
  const uint32_t hi01 = __builtin_amdgcn_perm(y[1], y[0], 0x07030602u);
  const uint32_t lo23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
  const uint32_t hi23 = __builtin_amdgcn_perm(y[3], y[2], 0x07030602u);
  const uint32_t d[4] = {__builtin_amdgcn_perm(lo23, lo01, 0x05040100u), __builtin_amdgcn_perm(lo23, lo01, 0x07060302u),
                         __builtin_amdgcn_perm(hi23, hi01, 0x05040100u), __builtin_amdgcn_perm(hi23, hi01, 0x07060302u)};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    half[i] = make_uint2(__builtin_bit_cast(uint32_t, fp8_f16x2<false>(d[i])),
                         __builtin_bit_cast(uint32_t, fp8_f16x2<true>(d[i])));
}

// Row operands of softmax x V: element 4 x + r is key 4 kb + r of tile x.
__device__ __forceinline__ void v_operands(const uint4 (&v)[2][4], int w, v8h (&va)[4]) {
  uint2 half[2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) v_halves(v[x], w, half[x]);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    va[i] = __builtin_bit_cast(v8h, make_uint4(half[0][i].x, half[0][i].y, half[1][i].x, half[1][i].y));
}

// The partials: share k of sequence b has index k + b (each next one moves
// either k or b on by one).  [G][blocks + batch][tiles] of 16 rows as the waves
// hold them, [16 i][lane] four sums (RowSums) and [16] (m, total) pairs: whole
// lines both ways.  Then [G][blocks + batch] flags (see k_tree_merge), then the
// sequences' starts.
struct Partials {
  float4* o;
  float2* stats;
  int* nan;
  int* starts;
  size_t shares;  // per group
  int tiles;
  __host__ __device__ Partials(void* part, int batch, int n) {
    shares = TR_BLOCKS + batch;
    tiles = (n * H + 15) / 16;
    o = static_cast<float4*>(part);
    stats = reinterpret_cast<float2*>(o + shares * G * tiles * 16 * WAVE);
    nan = reinterpret_cast<int*>(stats + shares * G * tiles * 16);
    starts = nan + shares * G;
  }
  // Tile 0 of share k of sequence b.
  __device__ __forceinline__ size_t tile(int g, int k, int b) const { return (g * shares + k + b) * tiles; }
};

// ------------------------------------------------------------- attention
// What a wave holds of RT tiles of 16 rows: lane (kb, col) sums of row col
// (o[i][r]: dim 16 (4 kb + r) + i), the base of its exponents and its total.
template <int RT>
struct RowSums {
  v4f o[RT][16];
  float m[RT], l[RT];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) o[rt][i] = v4f{0.f, 0.f, 0.f, 0.f};
      m[rt] = -INFINITY;
      l[rt] = 0.f;
    }
  }

  // Probabilities of 8 keys from their scores s (-inf: invisible; s unit: in
  // log2 units) as column operand.
  __device__ __forceinline__ v8h weigh(int rt, const v4f (&s)[2], float unit) {
    float tm = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * unit;
    if (__ballot(tm > m[rt] + TR_MOST)) {
      tm = fmaxf(tm, __shfl_xor(tm, 16));
      tm = fmaxf(tm, __shfl_xor(tm, 32));
      const bool grow = tm > m[rt] + TR_MOST;
      const float mn = grow ? tm - TR_BASE : m[rt];
      const float al = grow ? __builtin_amdgcn_exp2f(m[rt] - mn) : 1.f;
      l[rt] *= al;
      m[rt] = mn;
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[rt][i][r] *= al;
    }
    // while a row has seen nothing its m is -inf: 0 stands in, so that
    // invisible keys give 2^-inf and not NaN
    const float base = m[rt] == -INFINITY ? 0.f : m[rt];
    float p[8];
    v8h pb;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], unit, -base));
      pb[e] = (_Float16)p[e];
    }
    l[rt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    return pb;
  }

  // Totals over the lanes of a row.
  __device__ __forceinline__ void total() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += __shfl_xor(l[rt], 16);
      l[rt] += __shfl_xor(l[rt], 32);
    }
  }

  // Joins the sums of the first `live` key waves of each row wave into kw 0,
  // halving their number in every step; `rows`: the real ones (the others'
  // lanes move nothing).  buf: (live / 2) RW RT 16 WAVE uint4.
  template <int RW>
  __device__ __forceinline__ void join(int live, int rw, int kw, int rows, int lane, uint4* buf, float2* ml) {
    const int row = rw * RT * 16 + (lane & 15);
#pragma nounroll
    for (; live > 1; live = (live + 1) / 2) {
      const int half = (live + 1) / 2;
      __syncthreads();
      if (kw >= half && kw < live) {
        const int slot = (kw - half) * RW + rw;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if (row + rt * 16 >= rows) continue;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            buf[((slot * RT + rt) * 16 + i) * WAVE + lane] = __builtin_bit_cast(uint4, o[rt][i]);
          ml[(slot * RT + rt) * WAVE + lane] = make_float2(m[rt], l[rt]);
        }
      }
      __syncthreads();
      if (kw < live - half) {
        const int slot = kw * RW + rw;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if (row + rt * 16 >= rows) continue;
          const float2 x = ml[(slot * RT + rt) * WAVE + lane];
          const float mn = fmaxf(m[rt], x.x);
          // (an empty side counts 0: its m is -inf; a NaN total stays NaN)
          const float f0 = l[rt] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[rt] - mn);
          const float f1 = x.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x.x - mn);
          m[rt] = mn;
          l[rt] = fmaf(l[rt], f0, x.y * f1);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const v4f other = __builtin_bit_cast(v4f, buf[((slot * RT + rt) * 16 + i) * WAVE + lane]);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[rt][i][r] = fmaf(o[rt][i][r], f0, other[r] * f1);
            if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // 4 loads in flight, not 16
          }
        }
      }
    }
  }

  // Writes the partial of tiles tile0 .., of which rows below `rows` are real.
  __device__ __forceinline__ void store(const Partials& part, size_t tile, int tile0, int rows, int lane) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if ((tile0 + rt) * 16 + (lane & 15) >= rows) continue;
      const size_t at = tile + tile0 + rt;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        part.o[(at * 16 + i) * WAVE + lane] = make_float4(o[rt][i][0], o[rt][i][1], o[rt][i][2], o[rt][i][3]);
      if (lane < 16) part.stats[at * 16 + lane] = make_float2(m[rt], l[rt]);
    }
  }
};

// Which of slots len + j .. +3 a row sees (bits 0 .. 3; j > -64) whose mask of
// the drafts that are there is `bits`.
__device__ __forceinline__ uint32_t seen4(uint64_t bits, int j) {
  if (j < 0) bits = (bits << -j) | ((1ull << -j) - 1ull);
  else bits = j < 64 ? bits >> j : 0ull;
  return (uint32_t)bits;
}

// The scores of invisible keys of a pair become -inf: of tiles without a page,
// and with EDGE of drafts that the row does not see (`bits`: those it does) and
// keys past the end.  j: the lane's first key, from the first draft on.
template <bool EDGE>
__device__ __forceinline__ void hide(v4f (&s)[2], uint64_t bits, int j, bool bad0, bool bad1) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t seen = (x ? bad1 : bad0) ? 0u : EDGE ? seen4(bits, j + 16 * x) : ~0u;
#pragma unroll
    for (int r = 0; r < 4; ++r) s[x][r] = (seen >> r) & 1u ? s[x][r] : -INFINITY;
  }
}

// Takes NaN in 4 words as 0 (see k_tree_merge); whether there was one.
__device__ __forceinline__ uint32_t drop_nan(uint4& v) {
  uint32_t any = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t& u = (&v.x)[w];
    const uint32_t flag = nan_bytes(u) >> 7;
    u &= ~(flag * 0xffu);
    any |= flag;
  }
  return any;
}

// A block's share of the pairs of KV head g: the piece of one sequence after
// the other, `piece` called for each.  A single sequence (the latency of short
// contexts) needs no starts.
template <typename F>
__device__ __forceinline__ void each_piece(const TreeArgs& a, int* s_start, F piece) {
  const int g = blockIdx.y, k = blockIdx.x;
  int total;
  if (a.c.batch == 1) {
    total = sequence_pairs<false>(Sequence(a.c, a.counts, a.n, 0).uniform());
  } else {
    total = sequence_starts<false>(a.c, a.counts, a.n, s_start);
    if (k == 0 && g == 0) {
      int* starts = Partials(a.part, a.c.batch, a.n).starts;
      for (int b = threadIdx.x; b <= a.c.batch; b += blockDim.x) starts[b] = s_start[b];
    }
  }
  const int blocks = min((int)gridDim.x, total);
  if (k >= blocks) return;
  const int end = share_start(total, blocks, k + 1);
  for (int p0 = share_start(total, blocks, k); p0 < end;) {
    int b = 0, first = 0, p1 = end;
    if (a.c.batch > 1) {
      b = sequence_of(s_start, a.c.batch, p0);
      first = __builtin_amdgcn_readfirstlane(s_start[b]);
      p1 = min(end, __builtin_amdgcn_readfirstlane(s_start[b + 1]));
    }
    piece(b, first, p0, p1);
    p0 = p1;
  }
}

// A block: KW waves along the keys x RW along the rows, RT tiles of 16 rows a
// wave; every wave loads its pairs of tiles itself, one pair in registers
// whose K half is loaded anew after the scores and whose V half after the
// sums.  Registers: 64 RT sums, 32 of K, 32 of V a lane.
template <int RT, int RW, int KW, bool PAGED>
__global__ __launch_bounds__(RW * KW * 64) void k_tree(TreeArgs a) {
  constexpr int WAVES = RW * KW, TILES = RT * RW;
  constexpr int JOIN = (KW / 2) * RW * RT * 16 * WAVE;
  constexpr int IMG = TILES * IMG_TILE;
  __shared__ uint4 s_buf[IMG > JOIN ? IMG : JOIN];  // the queries' image, then the sums in transit
  __shared__ float2 s_ml[(KW / 2) * RW * RT * WAVE];
  __shared__ uint64_t s_bits[TILES * 16];
  __shared__ int s_start[CACHE_MAX_BATCH + 1];
  __shared__ int s_nan;
  const int g = blockIdx.y, k = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, kw = wave / RW, col = lane & 15, kb = lane >> 4;
  // (formed where it is used: its addresses do not stay in registers)
  auto partials = [&] {
    float* at = a.part;
    asm volatile("" : "+s"(at));
    return Partials(at, a.c.batch, a.n);
  };
  const ScoreScale zs(a.cap);
  const bool cap = a.cap > 0.f;
  each_piece(a, s_start, [&](int b, int first, int p0, int p1) {
    const Sequence seq = Sequence(a.c, a.counts, a.n, b).uniform();
    const int whole = min(p1, first + seq.len / TR_PAIR);  // pairs of committed keys alone come first
    stage_queries<WAVES * 64>(a.q, b, g, TILES, seq.rows, s_buf);
    for (int r = threadIdx.x; r < TILES * 16; r += WAVES * 64)
      s_bits[r] = r < seq.rows ? row_mask(a.tree, a.n, b, r / H) & seq.there() : 0;
    if (threadIdx.x == 0) s_nan = 0;
    Tile t[2];
    uint4 kx[2][4], vx[2][4];
    auto tiles = [&](int pair) {
#pragma unroll
      for (int x = 0; x < 2; ++x) t[x] = tile_at<PAGED>(a.c, b, g, (pair - first) * TR_PAIR + 16 * x, seq.keys);
    };
    int j = p0 + kw;
    if (j < whole) {
      tiles(j);
#pragma unroll
      for (int x = 0; x < 2; ++x) load_k<true>(kx[x], t[x], lane);
      __builtin_amdgcn_sched_barrier(0);  // (in the loop's order, which its waits count)
#pragma unroll
      for (int x = 0; x < 2; ++x) load_v<true, RW == 1>(vx[x], t[x], lane);
    }
    __syncthreads();

    RowSums<RT> sums;
    sums.clear();
    // one pair; EDGE: some of its keys are drafts or past the end (it loads
    // its records itself); MORE: the wave's next pair is loaded, by code of its
    // own, since a wait behind a branch that may not load is one for all loads
    auto step = [&](auto edge, auto more) {
      constexpr bool EDGE = decltype(edge)::value, MORE = decltype(more)::value;
      const int at = (j - first) * TR_PAIR;
      if (EDGE) {
        tiles(j);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          load_k<false>(kx[x], t[x], lane);
          load_v<false, RW == 1>(vx[x], t[x], lane);
        }
      }
      const bool bad0 = t[0].bad, bad1 = t[1].bad;
      if (MORE) tiles(j + KW);
      v4f acc[RT][2];
      scores<RT>(kx, s_buf + rw * RT * IMG_TILE, lane, acc);
      // (done before their records' registers are loaded anew)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int x = 0; x < 2; ++x) asm volatile("" : "+v"(acc[rt][x]));
      if (MORE) {
#pragma unroll
        for (int x = 0; x < 2; ++x) load_k<true>(kx[x], t[x], lane);
      }
      v8h pb[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (cap) zs.squash(acc[rt]);
        if (EDGE || bad0 || bad1)
          hide<EDGE>(acc[rt], EDGE ? s_bits[(rw * RT + rt) * 16 + col] : 0, at + 4 * kb - seq.len, bad0, bad1);
        pb[rt] = sums.weigh(rt, acc[rt], zs.unit);
      }
      if (bad0 || bad1) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (bad0) vx[0][r] = make_uint4(0, 0, 0, 0);
          if (bad1) vx[1][r] = make_uint4(0, 0, 0, 0);
        }
      }
      if (EDGE) {
        uint32_t any = 0;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) any |= drop_nan(vx[x][r]);
        if (__ballot(any != 0) && lane == 0) s_nan = 1;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        v8h va[4];
        v_operands(vx, w, va);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            sums.o[rt][4 * w + i] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(va[i], pb[rt], sums.o[rt][4 * w + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);  // one word's operands live at a time
      }
      if (MORE) {
#pragma unroll
        for (int x = 0; x < 2; ++x) load_v<true, RW == 1>(vx[x], t[x], lane);
      }
      j += KW;
    };
#pragma nounroll
    while (j + KW < whole) step(std::false_type{}, std::true_type{});
    if (j < whole) step(std::false_type{}, std::false_type{});
#pragma nounroll
    while (j < p1) step(std::true_type{}, std::false_type{});
    sums.total();
    sums.template join<RW>(min(KW, p1 - p0), rw, kw, seq.rows, lane, s_buf, s_ml);  // (waves without a pair hold nothing)
    const Partials part = partials();
    if (kw == 0)
      sums.store(part, part.tile(g, k, b), rw * RT, seq.rows, lane);
    __syncthreads();  // the buffer is formed anew
    if (threadIdx.x == 0) part.nan[g * part.shares + k + b] = s_nan;
  });
}

// More than 16 drafts: 8 row waves of 16 RT rows would each widen the same
// records.  Here they load and widen two pairs together into LDS, twice
// buffered, and every wave reads its operands there; the queries stay in
// registers.
template <int RT, bool PAGED>
__global__ __launch_bounds__(512) void k_tree_wide(TreeArgs a) {
  constexpr int TILES = RT * 8;
  constexpr int KBUF = 2 * 2 * IMG_TILE;   // uint4: [pair][tile][step][lane]
  constexpr int VBUF = 2 * 16 * WAVE;      // uint4: [pair][dim of 16][lane], tile x in half x
  constexpr int BUF = KBUF + VBUF;         // 64 KB
  __shared__ uint4 s_buf[2 * BUF];
  __shared__ uint64_t s_bits[TILES * 16];
  __shared__ uint32_t s_bad[2];  // of the four tiles in a buffer, a byte each
  __shared__ int s_start[CACHE_MAX_BATCH + 1];
  __shared__ int s_nan;
  const int g = blockIdx.y, k = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kb = lane >> 4;
  // what the wave loads: tile sx of pair sp, K or V (each SIMD has one of both)
  const int sx = wave & 1, sp = (wave >> 1) & 1;
  const bool sv = wave >= 4;
  // (formed where it is used: its addresses do not stay in registers)
  auto partials = [&] {
    float* at = a.part;
    asm volatile("" : "+s"(at));
    return Partials(at, a.c.batch, a.n);
  };
  const ScoreScale zs(a.cap);
  const bool cap = a.cap > 0.f;
  each_piece(a, s_start, [&](int b, int first, int p0, int p1) {
    const Sequence seq = Sequence(a.c, a.counts, a.n, b).uniform();
    for (int r = threadIdx.x; r < TILES * 16; r += 512)
      s_bits[r] = r < seq.rows ? row_mask(a.tree, a.n, b, r / H) & seq.there() : 0;
    if (threadIdx.x == 0) s_nan = 0;
    v8bf q[RT][STEPS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = (wave * RT + rt) * 16 + col;
      const bool real = row < seq.rows;
      const uint16_t* src = static_cast<const uint16_t*>(a.q.data) + b * a.q.sb +
                            (real ? row / H : 0) * a.q.st + (g * H + row % H) * a.q.sh;
#pragma unroll
      for (int step = 0; step < STEPS; ++step)
        q[rt][step] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(src + step_dim(step, kb)));
    }
    // waited for here: a wait in the loop would be one for the records too
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int step = 0; step < STEPS; ++step) asm volatile("" : "+v"(q[rt][step]));
    __syncthreads();  // (s_nan is 0 before any wave may set it)
    const int steps = (p1 - p0 + 1) / 2;
    // (formed anew where it is used: what is made of it does not stay in
    // registers; a spill of loaded records would wait for them)
    auto anew = [](int x) {
      asm volatile("" : "+v"(x));
      return x;
    };
    RowSums<RT> sums;
    sums.clear();
    // What a wave does, in two forms, of waves that load and widen K and of
    // those that do V: registers that two branches load are copied where the
    // branches meet, which waits for the loads.  Both take the same barriers.
    auto walk = [&](auto values) {
      constexpr bool V = decltype(values)::value;
      uint4 in[4];
      Tile t;
      auto load = [&](int it) {  // (past the last pair: its last tile again, not used)
        const int pair = min(p0 + 2 * it + sp, p1 - 1);
        t = tile_at<PAGED>(a.c, b, g, (pair - first) * TR_PAIR + 16 * sx, seq.keys);
        if (V) load_v<false, true>(in, t, anew(lane));
        else load_k<false>(in, t, anew(lane));
      };
      auto widen = [&](int it) {
        uint4* buf = s_buf + (it & 1) * BUF;
        const int pair = min(p0 + 2 * it + sp, p1 - 1);
        const int lane = anew(threadIdx.x) & 63;
        if (V) {
          if (PAGED && t.bad) {
#pragma unroll
            for (int r = 0; r < 4; ++r) in[r] = make_uint4(0, 0, 0, 0);
          }
          if ((pair - first + 1) * TR_PAIR > seq.len) {
            uint32_t any = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) any |= drop_nan(in[r]);
            if (__ballot(any != 0) && lane == 0) s_nan = 1;
          }
          uint2* out = reinterpret_cast<uint2*>(buf + KBUF + sp * 16 * WAVE + lane) + sx;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint2 half[4];
            v_halves(in, w, half);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[(4 * w + i) * WAVE * 2] = half[i];
          }
        } else {
          uint4* out = buf + (sp * 2 + sx) * IMG_TILE + lane;
#pragma unroll
          for (int step = 0; step < STEPS; ++step) {
            const uint4 w = in[step >> 1];
            out[step * WAVE] = __builtin_bit_cast(uint4, (step & 1) ? k_operand(w.z, w.w) : k_operand(w.x, w.y));
          }
          if (PAGED && lane == 0) reinterpret_cast<uint8_t*>(&s_bad[it & 1])[sp * 2 + sx] = t.bad;
        }
      };
      auto advance = [&](int it) {
        if (it + 1 < steps) widen(it + 1);
        if (it + 2 < steps) load(it + 2);
      };
      load(0);
      widen(0);
      if (steps > 1) load(1);
      __syncthreads();
#pragma nounroll
      for (int it = 0; it < steps; ++it) {
        const uint4* buf = s_buf + (it & 1) * BUF;
        uint32_t bad = 0;  // a byte for each of the buffer's tiles
        if constexpr (PAGED) bad = __builtin_amdgcn_readfirstlane(s_bad[it & 1]);
        // the two waves of a SIMD take turns: one widens the next pairs before
        // it computes, the other after, and one has priority, so that one
        // weighs while the other multiplies (64 drafts over 131072 keys: 201 us
        // a call without, 189 with the priority alone, 183 with both, before
        // the waits for records were taken out)
        if (V) advance(it);
#pragma nounroll
        for (int pair = 0; pair < 2; ++pair) {
          const int j = p0 + 2 * it + pair;
          if (j >= p1) break;
          const int at = (j - first) * TR_PAIR;
          const int ln = anew(lane);
          v4f acc[RT][2];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][0] = acc[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int step = 0; step < STEPS; ++step)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const v8bf kk = __builtin_bit_cast(v8bf, buf[((pair * 2 + x) * STEPS + step) * WAVE + ln]);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                acc[rt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[rt][step], acc[rt][x], 0, 0, 0);
            }
          const bool edge = at + TR_PAIR > seq.len;
          const bool bad0 = (bad >> (16 * pair)) & 0xffu, bad1 = (bad >> (16 * pair + 8)) & 0xffu;
          v8h pb[RT];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if (cap) zs.squash(acc[rt]);
            if (edge)
              hide<true>(acc[rt], s_bits[(wave * RT + rt) * 16 + (ln & 15)], at + 4 * (ln >> 4) - seq.len, bad0, bad1);
            else if (bad0 || bad1)
              hide<false>(acc[rt], 0, 0, bad0, bad1);
            pb[rt] = sums.weigh(rt, acc[rt], zs.unit);
          }
          const uint4* vb = buf + KBUF + pair * 16 * WAVE + ln;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const v8h va = __builtin_bit_cast(v8h, vb[i * WAVE]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              sums.o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[rt], sums.o[rt][i], 0, 0, 0);
          }
        }
        if (!V) advance(it);
        __syncthreads();
      }
    };
    if (sv) {
      __builtin_amdgcn_s_setprio(1);
      walk(std::true_type{});
    } else {
      walk(std::false_type{});
    }
    sums.total();
    const Partials part = partials();
    sums.store(part, part.tile(g, k, b), wave * RT, seq.rows, lane);
    __syncthreads();
    if (threadIdx.x == 0) part.nan[g * part.shares + k + b] = s_nan;
  });
}

// Joins the partials of a tile of rows, NI of the 16 sums i at a time (unit =
// (b, g, tile, i / NI)).  SLICES waves each add every SLICES-th share and the
// slices are added in order: 8 for few sequences, which have up to 64 shares
// each, with NI 1 where there are few rows too, so that all of a wave's shares
// are in flight at once (one draft, 64 shares: 5.5 us, 8.3 with NI 4); 1 (4
// units a block) for many rows with few shares (24 sequences x 48 rows: 7.8
// us, 23.5 when 16 slices had 3.7 shares to add).
// Where a share met NaN in V among the last keys (it took them as 0), those
// keys are gone through once more and the dims in which the row sees one
// become NaN.
template <int SLICES, int NI>
__global__ __launch_bounds__(SLICES == 1 ? 256 : SLICES * 64) void k_tree_merge(TreeArgs a, int shares) {
  constexpr int PER = 16 / NI;  // units of a tile
  const Partials part(a.part, a.c.batch, a.n);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int unit = SLICES == 1 ? blockIdx.x * 4 + wave : blockIdx.x, sl = SLICES == 1 ? 0 : wave;
  const int i0 = unit % PER * NI, tile = unit / PER % part.tiles, g = unit / PER / part.tiles % G,
            b = unit / (PER * part.tiles * G);
  __shared__ float4 s_o[SLICES == 1 ? 1 : SLICES][NI][WAVE];
  __shared__ float2 s_ml[SLICES == 1 ? 1 : SLICES][16];
  const Sequence seq = Sequence(a.c, a.counts, a.n, b).uniform();
  int total, start = 0;
  int stop = total = sequence_pairs<false>(seq);
  if (a.c.batch > 1) {
    total = part.starts[a.c.batch];
    start = part.starts[b];
    stop = part.starts[b + 1];
  }
  float m = -INFINITY, l = 0.f;
  v4f o[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
  int nan = 0;
  // the factors of what is held and of one more share
  auto join = [&](float2 ml, float& f0, float& f1) {
    const float mn = fmaxf(m, ml.x);
    f0 = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    f1 = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - mn);
    m = mn;
    l = fmaf(l, f0, ml.y * f1);
  };
  const int row = tile * 16 + (lane & 15);
  if (row < seq.rows && start < stop) {
    const int blocks = min(shares, total);
    const int k1 = share_of(total, blocks, stop - 1);
    constexpr int U = NI == 1 ? 8 : 4;  // shares in flight
    for (int k = share_of(total, blocks, start) + sl; k <= k1; k += U * SLICES) {
      float2 ml[U];
      float4 x[U][NI];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int ku = min(k + u * SLICES, k1);
        const size_t at = part.tile(g, ku, b) + tile;
        ml[u] = part.stats[at * 16 + (lane & 15)];
        if (k + u * SLICES > k1) ml[u] = make_float2(-INFINITY, 0.f);  // (none left: adds nothing)
        nan |= part.nan[g * part.shares + ku + b];
#pragma unroll
        for (int i = 0; i < NI; ++i) x[u][i] = part.o[(at * 16 + i0 + i) * WAVE + lane];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f0, f1;
        join(ml[u], f0, f1);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const float v[4] = {x[u][i].x, x[u][i].y, x[u][i].z, x[u][i].w};
#pragma unroll
          for (int r = 0; r < 4; ++r) o[i][r] = fmaf(o[i][r], f0, v[r] * f1);
        }
      }
    }
  }
  // dims 64 kb + 16 r + i0 + [0, NI) of the row, for r = r0 .. r1 - 1
  int r0 = 0, r1 = 4;
  if constexpr (SLICES > 1) {
#pragma unroll
    for (int i = 0; i < NI; ++i) s_o[sl][i][lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    if (lane < 16) s_ml[sl][lane] = make_float2(m, l);
    nan = __syncthreads_or(nan);
    if (sl >= 4) return;  // wave r < 4 finishes its dims
    r0 = sl;
    r1 = sl + 1;
    m = -INFINITY;
    l = 0.f;
    float sum[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) sum[i] = 0.f;
#pragma unroll
    for (int s = 0; s < SLICES; ++s) {
      float f0, f1;
      join(s_ml[s][lane & 15], f0, f1);
#pragma unroll
      for (int i = 0; i < NI; ++i)
        sum[i] = fmaf(sum[i], f0, reinterpret_cast<const float*>(&s_o[s][i][lane])[sl] * f1);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) o[i] = v4f{sum[i], sum[i], sum[i], sum[i]};
  }
  if (row >= a.n * H) return;
  const size_t at = ((size_t)b * a.n + row / H) * G * H + g * H + row % H;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r < r0 || r >= r1) continue;
    const int dim = 64 * (lane >> 4) + 16 * r + i0;
    float y[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) y[i] = l == 0.f ? 0.f : o[i][r] * inv;
    if (nan && row < seq.rows) {
      const uint64_t bits = row_mask(a.tree, a.n, b, row / H);
      for (int t = seq.len & ~(TR_PAIR - 1); t < seq.keys; ++t) {
        const uint32_t page = a.c.table ? a.c.page(b, t) : 0;
        if (!sees(seq, bits, t) || (a.c.table && page >= a.c.n_pages)) continue;
        const size_t record = a.c.table ? a.c.row_in(page, g, t) : a.c.row(b, g, t);
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if ((a.c.records[record * 512 + dim + i] & 0x7f) == 0x7f) y[i] = __builtin_nanf("");
      }
    }
    uint16_t* out = a.out + at * D + dim;
    if constexpr (NI == 4)
      *reinterpret_cast<uint2*>(out) =
          make_uint2(bf16_rne(y[0]) | bf16_rne(y[1]) << 16, bf16_rne(y[2]) | bf16_rne(y[3]) << 16);
    else
      out[0] = (uint16_t)bf16_rne(y[0]);
  }
  if (i0 == 0 && r0 == 0 && lane < 16) a.lse[at] = l == 0.f ? -INFINITY : (m + __log2f(l)) * TR_LN2;
}

// ------------------------------------------------------------ key weights
// A block takes a share of the pairs of KV head g like k_tree's; its waves
// stride the share, each with all rows of its 32 keys: the queries' image is
// in LDS, the K halves widened once in registers, and a key's weight is summed
// over the rows in registers and then over the 16 lanes of a row group: no
// atomics, the same bits every time.  Bound by matrix cores, vector units and
// LDS about alike for many rows, so 4 waves on a SIMD do more than records
// loaded ahead (32 rows over 131072 keys: 46 us, 70 with 2 waves and a pair
// ahead; 64 rows 67); by the K halves, 256 bytes of every 512, for few (one row
// 28 us a call, 4.8 TB/s).  4 waves leave 128 registers: 8 are spilled, outside
// the loop over row tiles.
// (the 128 KB image of 64 drafts leaves room for one block, of 16 waves then)
constexpr int weight_waves(int tiles) { return tiles > 8 ? 16 : 8; }

template <int TILES, bool PAGED>
__global__ __launch_bounds__(weight_waves(TILES) * 64, 4) void k_key_weights(WeightArgs a) {
  constexpr int WAVES = weight_waves(TILES);
  __shared__ uint4 s_img[TILES * IMG_TILE];
  __shared__ float s_lse[TILES * 16];
  __shared__ uint64_t s_bits[TILES * 16];
  __shared__ int s_start[CACHE_MAX_BATCH + 1];
  const int g = blockIdx.y, k = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kb = lane >> 4;
  const ScoreScale zs(a.cap);
  const bool cap = a.cap > 0.f;
  const int total = a.c.batch == 1 ? sequence_pairs<true>(Sequence(a.c, a.counts, a.n, 0).uniform())
                                   : sequence_starts<true>(a.c, a.counts, a.n, s_start);
  const int blocks = min((int)gridDim.x, total);
  if (k >= blocks) return;
  const int end = share_start(total, blocks, k + 1);
  for (int p0 = share_start(total, blocks, k); p0 < end;) {
    int b = 0, first = 0, p1 = end;
    if (a.c.batch > 1) {
      b = sequence_of(s_start, a.c.batch, p0);
      first = __builtin_amdgcn_readfirstlane(s_start[b]);
      p1 = min(end, __builtin_amdgcn_readfirstlane(s_start[b + 1]));
    }
    const Sequence seq = Sequence(a.c, a.counts, a.n, b).uniform();
    uint4 kx[2][4];
    Tile t0, t1;
    int j = p0 + wave;
    auto tiles = [&](int pair, Tile& x, Tile& y) {
      const int t = (pair - first) * TR_PAIR;
      x = tile_at<PAGED>(a.c, b, g, t, seq.keys);
      y = tile_at<PAGED>(a.c, b, g, t + 16, seq.keys);
    };
    stage_queries<WAVES * 64>(a.q, b, g, TILES, seq.rows, s_img);
    for (int r = threadIdx.x; r < TILES * 16; r += WAVES * 64) {
      const int i = r / H;
      const bool row = r < seq.rows;
      s_bits[r] = row ? row_mask(a.tree, a.n, b, i) : 0;
      const float lse = row ? a.lse[((size_t)b * a.n + i) * G * H + g * H + r % H] : -INFINITY;
      s_lse[r] = lse == -INFINITY ? INFINITY : lse * DN_LOG2E;  // such a row adds 2^-inf
    }
    __syncthreads();
    const int used = (seq.rows + 15) / 16;
#pragma nounroll
    for (; j < p1; j += WAVES) {
      const int at = (j - first) * TR_PAIR;
      // nothing is loaded ahead: with 4 waves on a SIMD the others compute
      tiles(j, t0, t1);
      load_k<false>(kx[0], t0, lane);
      load_k<false>(kx[1], t1, lane);
      const bool bad0 = t0.bad, bad1 = t1.bad;
      const bool edge = at + TR_PAIR > seq.len || bad0 || bad1;
      // widened once for all rows; the records' registers are loaded anew
      v8bf ka[2][STEPS];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
          const uint4 w = kx[x][step >> 1];
          ka[x][step] = (step & 1) ? k_operand(w.z, w.w) : k_operand(w.x, w.y);
        }
      float sum[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = 0.f;
#pragma nounroll
      for (int tile = 0; tile < used; ++tile) {
        const int row = tile * 16 + col;
        const float lse = s_lse[row];
        v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
          const v8bf q = __builtin_bit_cast(v8bf, s_img[tile * IMG_TILE + step * WAVE + lane]);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            acc[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[x][step], q, acc[x], 0, 0, 0);
        }
        if (cap) zs.squash(acc);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float p = __builtin_amdgcn_exp2f(fmaf(acc[e >> 2][e & 3], zs.unit, -lse));
          if (edge) {
            const bool seen = !(e < 4 ? bad0 : bad1) &&
                              sees(seq, s_bits[row], at + 16 * (e >> 2) + 4 * kb + (e & 3));
            p = seen ? p : 0.f;
          }
          sum[e] += p;
        }
      }
      float mine = 0.f;  // lane col = 4 x + r of a row group keeps key 16 x + 4 kb + r
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = sum[e];
        v += dpp_f<0xB1>(v);   // quad_perm [1,0,3,2]
        v += dpp_f<0x4E>(v);   // quad_perm [2,3,0,1]
        v += dpp_f<0x141>(v);  // row_half_mirror
        v += dpp_f<0x140>(v);  // row_mirror
        mine = col == e ? v : mine;
      }
      const int t = at + 16 * (col >> 2) + 4 * kb + (col & 3);
      if (col < 8 && t < seq.keys) {
        float* w = a.weights + a.c.row(b, g, t);
        *w = a.accumulate ? *w + mine : mine;
      }
    }
    p0 = p1;
    __syncthreads();
  }
}

template <bool PAGED>
void tree_rows(const TreeArgs& a, hipStream_t st) {
  const dim3 grid(TR_BLOCKS, G);
  const int tiles = (a.n * H + 15) / 16;
  // up to 4 drafts: one tile of rows a wave (49 us a call on one cache of 131072
  // keys over and over; 57 with two, the second empty; 62 with 12 waves, whose
  // 168 registers spill)
  if (tiles <= 1) hipLaunchKernelGGL((k_tree<1, 1, 8, PAGED>), grid, dim3(512), 0, st, a);
  // two tiles a wave: widened records serve both (16 drafts 66 us, 99 with
  // one); row waves that hold the same records as far as 16 drafts (12 in 64
  // paged sequences of 2000 keys 72 us, 80 when they are widened once into
  // LDS), widened once past them (32 drafts 93 us, 122 by 4 row waves each for
  // itself; 64 drafts 154 us, 219 by 8)
  else if (tiles <= 2) hipLaunchKernelGGL((k_tree<2, 1, 8, PAGED>), grid, dim3(512), 0, st, a);
  else if (tiles <= 4) hipLaunchKernelGGL((k_tree<2, 2, 4, PAGED>), grid, dim3(512), 0, st, a);
  else if (tiles <= 8) hipLaunchKernelGGL((k_tree_wide<1, PAGED>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((k_tree_wide<2, PAGED>), grid, dim3(512), 0, st, a);
}

template <bool PAGED>
void weight_rows(const WeightArgs& a, hipStream_t st) {
  const int tiles = (a.n * H + 15) / 16;
  const dim3 block(weight_waves(tiles) * 64);
  const dim3 grid(tiles <= 8 ? 2 * TR_BLOCKS : TR_BLOCKS, G);
  if (tiles <= 1) hipLaunchKernelGGL((k_key_weights<1, PAGED>), grid, block, 0, st, a);
  else if (tiles <= 2) hipLaunchKernelGGL((k_key_weights<2, PAGED>), grid, block, 0, st, a);
  else if (tiles <= 4) hipLaunchKernelGGL((k_key_weights<4, PAGED>), grid, block, 0, st, a);
  else if (tiles <= 8) hipLaunchKernelGGL((k_key_weights<8, PAGED>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_key_weights<16, PAGED>), grid, block, 0, st, a);
}

}  // namespace

size_t tree_workspace(int batch, int n) {
  const Partials p(nullptr, batch, n);
  return reinterpret_cast<size_t>(p.starts + batch + 1);
}

void launch_tree(const TreeArgs& a, hipStream_t st) {
  (a.c.table ? tree_rows<true> : tree_rows<false>)(a, st);
  const int tiles = a.c.batch * G * ((a.n * H + 15) / 16);
  if (tiles <= 16)
    hipLaunchKernelGGL((k_tree_merge<8, 1>), dim3(tiles * 16), dim3(512), 0, st, a, TR_BLOCKS);
  else if (a.c.batch <= 4)
    hipLaunchKernelGGL((k_tree_merge<8, 4>), dim3(tiles * 4), dim3(512), 0, st, a, TR_BLOCKS);
  else if (a.c.batch <= 16)
    hipLaunchKernelGGL((k_tree_merge<4, 4>), dim3(tiles * 4), dim3(256), 0, st, a, TR_BLOCKS);
  else
    hipLaunchKernelGGL((k_tree_merge<1, 4>), dim3(tiles), dim3(256), 0, st, a, TR_BLOCKS);
}

void launch_key_weights(const WeightArgs& a, hipStream_t st) {
  (a.c.table ? weight_rows<true> : weight_rows<false>)(a, st);
}

}  // namespace skv
