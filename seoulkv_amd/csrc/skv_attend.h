// What the attention of a record cache's operators shares: what rows see, the
// records' two forms, scores, softmax sums (the mathematics: skv_tree.hip).
#pragma once

#include <type_traits>

#include "skv_cache.h"
#include "skv_device.h"
#include "skv_tile.h"

namespace skv {

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

// The pairs of a sequence that some row may see, those first that every row sees
// whole: pair(i) for i < whole, then the others, edges.  Without a window they
// come in slot order; with one the pairs between the sink's and the window's
// are left out.
struct Reach {
  static constexpr bool ENDS = true;  // see WideBuffers
  int whole, all;       // numbers of pairs
  int sink, sink_pairs; // whole ones in the sink; pairs of the sink
  int late, window;     // first whole pair of every window; first pair of some window
  int open;             // first pair with a draft or past the committed slots
  // Rows that all see slots below `seen` but for the window, the earliest of
  // which begins at slot `from`, the latest at `until`; no row sees slot `keys`.
  __device__ Reach(int seen, int keys, int from, int until, const Window& w) {
    const int pairs = (keys + TR_PAIR - 1) / TR_PAIR;
    open = seen / TR_PAIR;
    late = sink = sink_pairs = window = 0;
    if (w.size) {
      sink = min(w.sink, seen) / TR_PAIR;
      late = min(max((until + TR_PAIR - 1) / TR_PAIR, sink), open);
      sink_pairs = min((min(w.sink, keys) + TR_PAIR - 1) / TR_PAIR, late);
      window = min(max(from / TR_PAIR, sink_pairs), late);
    }
    whole = sink + open - late;
    all = whole + sink_pairs - sink + late - window + pairs - open;
  }
  // A sequence's drafts: the earliest window is that of a row that sees none of
  // them, the latest that of one that sees all.
  __device__ Reach(const Sequence& s, const Window& w)
      : Reach(s.len, s.keys, max(0, s.len - w.size), min(s.len, max(0, s.len - w.size + s.drafts)), w) {}
  __device__ __forceinline__ int pair(int i) const {
    if (i < whole) return i < sink ? i : late + i - sink;
    i -= whole;
    if (i < sink_pairs - sink) return sink + i;
    i -= sink_pairs - sink;
    return i < late - window ? window + i : open + i - (late - window);
  }
};

// The same without a window: the pairs in slot order.
struct AllPairs {
  static constexpr bool ENDS = false;
  int whole, all;
  __device__ AllPairs(const Sequence& s, const Window&) : whole(s.len / TR_PAIR), all((s.keys + TR_PAIR - 1) / TR_PAIR) {}
  __device__ __forceinline__ int pair(int i) const { return i; }
};

// Pairs of a sequence; with WHOLE one without rows counts too.
template <bool WHOLE>
__device__ __forceinline__ int sequence_pairs(const Sequence& s, const Window& w) {
  return WHOLE || s.rows ? Reach(s, w).all : 0;
}

// s_start[b]: pairs of the sequences before b; s_start[batch]: all.
template <bool WHOLE>
__device__ __forceinline__ int sequence_starts(const CacheView& c, const int* counts, int n, const Window& w,
                                               int* s_start) {
  if (threadIdx.x < WAVE) {
    int carry = 0;
    for (int b0 = 0; b0 < c.batch; b0 += WAVE) {
      const int b = b0 + threadIdx.x;
      const int pairs = b < c.batch ? sequence_pairs<WHOLE>(Sequence(c, counts, n, b), w) : 0;
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
template <int BYTES, bool PAGED>
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
    x.at = c.records + (x.bad ? 0 : c.row_in(page, g, ta) * BYTES);
  } else {
    x.at = c.records + c.row(b, g, ta) * BYTES;
  }
  return x;
}

// ---------------------------------------------------------------- formats
// The two forms of records.  A tile's registers: K, of key lane % 16 the dims
// step_dim(step, kb) .. +7 of every step; V, of keys 4 kb + r the dims 16 c ..
// +15.  Both are widened exactly, K to BF16 and V to FP16.
__device__ __forceinline__ v8bf join8(v2bf a, v2bf b, v2bf c, v2bf d) {
  return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

struct Eight {
  static constexpr int BYTES = RECORD_EIGHT;
  struct K { uint4 w[4]; };
  struct V { uint4 w[4]; };

  // Step 2 j + half takes the dims that half `half` of a lane's K word j holds.
  __device__ __forceinline__ static int step_dim(int step, int kb) {
    return 64 * (step >> 1) + 16 * kb + 8 * (step & 1);
  }
  // WHOLE: all 16 keys are in reach.
  template <bool WHOLE>
  __device__ __forceinline__ static void load_k(K& k, const Tile& x, int lane) {
    const uint32_t at = (WHOLE ? lane & 15 : min(lane & 15, x.last)) * BYTES + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) k.w[j] = *reinterpret_cast<const uint4*>(x.at + 256 + 64 * j + at);
  }
  // ONCE: no other wave reads the tile.  Where two row waves do, streaming loads
  // brought a fifth of the records from memory twice (12 drafts of 24 ragged
  // sequences: 557 MB and 124 us, 455 MB and 118 us with plain ones).
  template <bool WHOLE, bool ONCE>
  __device__ __forceinline__ static void load_v(V& v, const Tile& x, int lane) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * (lane >> 4) + r;
      const uint8_t* at = x.at + (uint32_t)((WHOLE ? row : min(row, x.last)) * BYTES + 16 * (lane & 15));
      v.w[r] = ONCE ? load_stream(at) : *reinterpret_cast<const uint4*>(at);
    }
  }
  template <bool HI>
  __device__ __forceinline__ static v2bf bf16x2(uint32_t w) {
    return __builtin_bit_cast(v2bf, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, HI));
  }
  // The row operand of a step.
  __device__ __forceinline__ static v8bf k_operand(const K& k, int step) {
    const uint4 w = k.w[step >> 1];
    const uint32_t lo = (step & 1) ? w.z : w.x, hi = (step & 1) ? w.w : w.y;
    return join8(bf16x2<false>(lo), bf16x2<true>(lo), bf16x2<false>(hi), bf16x2<true>(hi));
  }
  template <bool HI>
  __device__ __forceinline__ static v2h f16x2(uint32_t w) {
    return __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, HI));
  }
  // Dims 16 c + 4 w + i of the 4 keys, transposed and widened: half i's 4 values.
  __device__ __forceinline__ static void v_halves(const V& v, int w, uint2 (&half)[4]) {
    const uint32_t y[4] = {(&v.w[0].x)[w], (&v.w[1].x)[w], (&v.w[2].x)[w], (&v.w[3].x)[w]};
    const uint32_t lo01 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u);
    const uint32_t hi01 = __builtin_amdgcn_perm(y[1], y[0], 0x07030602u);
    const uint32_t lo23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
    const uint32_t hi23 = __builtin_amdgcn_perm(y[3], y[2], 0x07030602u);
    const uint32_t d[4] = {__builtin_amdgcn_perm(lo23, lo01, 0x05040100u), __builtin_amdgcn_perm(lo23, lo01, 0x07060302u),
                           __builtin_amdgcn_perm(hi23, hi01, 0x05040100u), __builtin_amdgcn_perm(hi23, hi01, 0x07060302u)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      half[i] = make_uint2(__builtin_bit_cast(uint32_t, f16x2<false>(d[i])), __builtin_bit_cast(uint32_t, f16x2<true>(d[i])));
  }
  __device__ __forceinline__ static void clear_v(V& v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v.w[r] = make_uint4(0, 0, 0, 0);
  }
  // Takes NaN as 0 (see k_tree_merge); whether there was one.
  __device__ __forceinline__ static uint32_t drop_nan(V& v) {
    uint32_t any = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t& u = (&v.w[r].x)[w];
        const uint32_t flag = (((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
        u &= ~(flag * 0xffu);
        any |= flag;
      }
    return any;
  }
  __device__ __forceinline__ static bool v_is_nan(const uint8_t* record, int dim) {
    return (record[dim] & 0x7f) == 0x7f;
  }
};

struct Four {
  static constexpr int BYTES = RECORD_FOUR;
  // A tile as it lies in memory, 272 pieces of 16 bytes: whole lines, where K, V
  // and scales of records that begin anywhere in a line touch four times as many.
  // A wave holds it in registers and parts it in LDS of its own.
  typedef uint32_t Word4 __attribute__((ext_vector_type(4)));
  struct Raw { Word4 w[5]; };
  template <bool WHOLE>
  __device__ __forceinline__ static void load_raw(Raw& raw, const Tile& x, int lane) {
    const int end = WHOLE ? 16 * BYTES / 16 - 1 : (x.last + 1) * (BYTES / 16) - 1;
    const Word4* at = reinterpret_cast<const Word4*>(x.at);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const int piece = i < 4 ? 64 * i + lane : 256 + (lane & 15);
      raw.w[i] = at[WHOLE ? piece : min(piece, end)];
    }
  }
  __device__ __forceinline__ static void put_raw(const Raw& raw, uint4* stage, int lane) {
    Word4* to = reinterpret_cast<Word4*>(stage);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[64 * i + lane] = raw.w[i];
    to[256 + (lane & 15)] = raw.w[4];  // (the same by four lanes)
  }
  struct K { uint4 w[2]; uint2 scale; };
  struct V { uint2 w[4]; uint32_t scale[4]; };

  // Step 4 j + s takes word s of a lane's K word j, which is of one block of 32.
  __device__ __forceinline__ static int step_dim(int step, int kb) {
    return 32 * (4 * (step >> 2) + kb) + 8 * (step & 3);
  }
  template <bool WHOLE>
  __device__ __forceinline__ static void load_k(K& k, const Tile& x, int lane) {
    const uint32_t key = (WHOLE ? lane & 15 : min(lane & 15, x.last)) * BYTES, at = key + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < 2; ++j) k.w[j] = *reinterpret_cast<const uint4*>(x.at + 128 + 64 * j + at);
    // bytes kb and 4 + kb of the 8
    const uint2 s = *reinterpret_cast<const uint2*>(x.at + 264 + key);
    k.scale = s;
  }
  template <bool WHOLE, bool ONCE>
  __device__ __forceinline__ static void load_v(V& v, const Tile& x, int lane) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * (lane >> 4) + r;
      const uint8_t* at = x.at + (uint32_t)((WHOLE ? row : min(row, x.last)) * BYTES);
      v.w[r] = *reinterpret_cast<const uint2*>(at + 8 * (lane & 15));
      v.scale[r] = at[256 + ((lane & 15) >> 1)];
    }
  }
  // 2^(byte - 127) as FP32; NaN or infinity, which widen to NaN, for what no write gives
  __device__ __forceinline__ static float scale_of(uint32_t byte) {
    return __uint_as_float((byte > (uint32_t)FOUR_MAX ? (uint32_t)FOUR_NAN : byte) << 23);
  }
  template <int BYTE>
  __device__ __forceinline__ static v2bf bf16x2(uint32_t w, float s) {
    return __builtin_bit_cast(v2bf, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, BYTE));
  }
  __device__ __forceinline__ static v8bf k_operand(const K& k, int step) {
    const uint32_t kb = (threadIdx.x >> 4) & 3u;
    const float s = scale_of(((step >> 2 ? k.scale.y : k.scale.x) >> (8 * kb)) & 0xffu);
    const uint32_t w = (&k.w[step >> 2].x)[step & 3];
    return join8(bf16x2<0>(w, s), bf16x2<1>(w, s), bf16x2<2>(w, s), bf16x2<3>(w, s));
  }
  template <int BYTE>
  __device__ __forceinline__ static uint32_t f16x2(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, BYTE));
  }
  __device__ __forceinline__ static void v_halves(const V& v, int w, uint2 (&half)[4]) {
    uint32_t y[4][2];  // of key r dims 4 w, +1 and 4 w + 2, +3
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t u = w >> 1 ? v.w[r].y : v.w[r].x;
      const float s = scale_of(v.scale[r]);
      y[r][0] = (w & 1) ? f16x2<2>(u, s) : f16x2<0>(u, s);
      y[r][1] = (w & 1) ? f16x2<3>(u, s) : f16x2<1>(u, s);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t pick = i & 1 ? 0x07060302u : 0x05040100u;
      half[i] = make_uint2(__builtin_amdgcn_perm(y[1][i >> 1], y[0][i >> 1], pick),
                           __builtin_amdgcn_perm(y[3][i >> 1], y[2][i >> 1], pick));
    }
  }
  __device__ __forceinline__ static void clear_v(V& v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v.w[r] = make_uint2(0, 0);
      v.scale[r] = 127;
    }
  }
  __device__ __forceinline__ static uint32_t drop_nan(V& v) {
    uint32_t any = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool nan = v.scale[r] > (uint32_t)FOUR_MAX;
      v.w[r] = nan ? make_uint2(0, 0) : v.w[r];
      v.scale[r] = nan ? 127u : v.scale[r];
      any |= nan;
    }
    return any;
  }
  __device__ __forceinline__ static bool v_is_nan(const uint8_t* record, int dim) {
    return record[256 + dim / 32] > FOUR_MAX;
  }
};

// ---------------------------------------------------------------- queries
// The score step's column operands of 16 rows: [step][lane] 16 bytes, the dims
// F::step_dim(step, kb) .. +7 of row col for lane 16 kb + col.
constexpr int STEPS = D / 32;
constexpr int IMG_TILE = STEPS * WAVE;  // uint4 per 16 rows

// Copies the rows of a sequence into the image of `tiles` tiles; rows past
// `rows` are 0.
template <typename F, int THREADS>
__device__ __forceinline__ void stage_queries(const Rows& q, int b, int g, int tiles, int rows, uint4* img) {
  for (int at = threadIdx.x; at < tiles * IMG_TILE; at += THREADS) {
    const int lane = at & 63, step = (at >> 6) & (STEPS - 1), row = (at / IMG_TILE) * 16 + (lane & 15);
    uint4 w = make_uint4(0, 0, 0, 0);
    if (row < rows)
      w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q.data) + b * q.sb +
                                          (row / H) * q.st + (g * H + row % H) * q.sh +
                                          F::step_dim(step, lane >> 4));
    img[at] = w;
  }
}

// q . k of two tiles of 16 keys (lane: keys 4 kb + r) for RT tiles of 16 rows
// (lane: row col).
template <typename F, int RT>
__device__ __forceinline__ void scores(const typename F::K (&k)[2], const uint4* img, int lane, v4f (&acc)[RT][2]) {
  // the image is read from LDS for every pair: held in registers it would
  // leave too few for the records in flight
  asm volatile("" : "+v"(lane));
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) acc[rt][0] = acc[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int step = 0; step < STEPS; ++step) {
    v8bf a[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) a[x] = F::k_operand(k[x], step);
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

// What a row sees of a sequence: of the drafts that are there those in `bits`, of
// the committed slots those before `sink` and those from `first` on.
struct Sight {
  uint64_t bits;
  int first;
};
// With a window the last `size` of what a row that sees the drafts `bits` sees
// stay, and what lies in the first `sink` slots.
__device__ __forceinline__ Sight sight_of(const Sequence& s, const Window& w, uint64_t bits) {
  bits &= s.there();
  if (w.size == 0) return {bits, 0};
  const int seen = __popcll(bits);
  if (seen <= w.size) return {bits, max(0, s.len - (w.size - seen))};
  const int room = w.sink - s.len;  // drafts in the first slots
  uint64_t late = bits;
  for (int drop = seen - w.size; drop > 0; --drop) late &= late - 1;
  return {late | (room <= 0 ? 0ull : room < 64 ? bits & ((1ull << room) - 1ull) : bits), s.len};
}

// Whether the key in slot t is visible to a row with mask `bits`, without a window
// and with one.
__device__ __forceinline__ bool sees_drafts(const Sequence& s, uint64_t bits, int t) {
  const int j = t - s.len;
  return j < 0 || (j < s.drafts && ((bits >> j) & 1ull));
}
__device__ __forceinline__ bool sees(const Sequence& s, const Window& w, const Sight& r, int t) {
  const int j = t - s.len;
  return j < 0 ? t >= r.first || t < w.sink : j < s.drafts && ((r.bits >> j) & 1ull);
}

// Row operands of softmax x V: element 4 x + r is key 4 kb + r of tile x.
template <typename F>
__device__ __forceinline__ void v_operands(const typename F::V (&v)[2], int w, v8h (&va)[4]) {
  uint2 half[2][4];
#pragma unroll
  for (int x = 0; x < 2; ++x) F::v_halves(v[x], w, half[x]);
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

// Which of slots t .. t + 3 a row sees (bits 0 .. 3): of the drafts those in `bits`;
// with a window.
__device__ __forceinline__ uint32_t seen4(const Sequence& s, const Window&, uint64_t bits, int t) {
  const int j = t - s.len;
  if (j < 0) return (uint32_t)((bits << min(-j, 63)) | ((1ull << min(-j, 63)) - 1ull));
  return j < 64 ? (uint32_t)(bits >> j) : 0u;
}
__device__ __forceinline__ uint32_t seen4(const Sequence& s, const Window& w, const Sight& r, int t) {
  const int j = t - s.len;
  uint64_t drafts = r.bits;
  if (j < 0) drafts = (drafts << min(-j, 63)) | ((1ull << min(-j, 63)) - 1ull);
  else drafts = j < 64 ? drafts >> j : 0ull;
  // (a draft that is seen lies behind `first`)
  const uint32_t late = ~0u << min(max(r.first - t, 0), 31), early = (1u << min(max(w.sink - t, 0), 31)) - 1u;
  return (uint32_t)drafts & (late | early);
}

// The scores of invisible keys of a pair become -inf: of tiles without a page,
// and with EDGE of those that the row does not see.  t: the lane's first key.
template <bool EDGE, typename Row>
__device__ __forceinline__ void hide(v4f (&s)[2], const Sequence& seq, const Window& w, const Row& row, int t,
                                     bool bad0, bool bad1) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t seen = (x ? bad1 : bad0) ? 0u : EDGE ? seen4(seq, w, row, t + 16 * x) : ~0u;
#pragma unroll
    for (int r = 0; r < 4; ++r) s[x][r] = (seen >> r) & 1u ? s[x][r] : -INFINITY;
  }
}

// The queries of 16 RT rows of a wave as column operands: row0 is the lane's row of
// its first tile, row / H the token after `token`; rows past `rows` repeat one.
template <typename F, int RT>
__device__ __forceinline__ void load_queries(v8bf (&q)[RT][STEPS], const Rows& in, int b, int g, int token, int rows,
                                             int row0, int kb) {
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = row0 + rt * 16;
    const uint16_t* src = static_cast<const uint16_t*>(in.data) + b * in.sb +
                          (token + (row < rows ? row / H : 0)) * in.st + (g * H + row % H) * in.sh;
#pragma unroll
    for (int step = 0; step < STEPS; ++step)
      q[rt][step] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(src + F::step_dim(step, kb)));
  }
  // waited for here: a wait in the walk's loop would be one for the records too
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int step = 0; step < STEPS; ++step) asm volatile("" : "+v"(q[rt][step]));
}

// x formed anew where it is used: what is made of it does not stay in registers.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Eight waves of 16 RT rows each load and widen two pairs together into LDS,
// twice buffered, and every wave reads its operands there; the queries stay in
// registers.  (So what is not needed in the walk is formed anew after it: a spill of
// loaded records would wait for them.)
//
// Pairs without ENDS, a tree's without a window, are walked with less beside the
// operands: pages are read with their tiles, holes tested in every step.  With the
// window's form scalar registers ran out and operands were read from LDS one by one
// (paged, 32 drafts over 131072 keys 120 us, 103 so; of 24 ragged sequences 99 and 87;
// 64 capped drafts, contiguous, 221 and 214).
struct WideBuffers {
  static constexpr int KBUF = 2 * 2 * IMG_TILE;   // uint4: [pair][tile][step][lane]
  static constexpr int VBUF = 2 * 16 * WAVE;      // uint4: [pair][dim of 16][lane], tile x in half x
  static constexpr int BUF = KBUF + VBUF;         // 64 KB
  uint4 buf[2 * BUF];
  uint32_t bad[2];  // of the four tiles in a buffer, a byte each
  int nan;          // whether V had NaN in an edge, taken as 0

  // Adds pairs p0 .. p1 - 1 of `reach` to the sums of the wave's rows; waves
  // that are not `active` only load.  hide_rows(edge, rt, scores, pair, lane,
  // bad0, bad1) hides what a row does not see.
  template <typename F, int RT, bool PAGED, typename Pairs, typename Hide>
  __device__ __forceinline__ void walk(const CacheView& c, int b, int g, int keys, const Pairs& reach, int p0, int p1,
                                       const v8bf (&q)[RT][STEPS], RowSums<RT>& sums, float cap, bool active,
                                       Hide hide_rows) {
    if constexpr (PAGED && Pairs::ENDS) {
      // (pages that are none are rare: looked for once and not in every step,
      // whose wait for the flags took a sixth of the time)
      int hole = 0;
      for (int i = p0 + (int)threadIdx.x; i < p1; i += 512) {
        const int t = reach.pair(i) * TR_PAIR;
        hole |= c.page(b, t) >= c.n_pages || c.page(b, min(t + 16, keys - 1)) >= c.n_pages;
      }
      if (__syncthreads_or(hole)) {
        forms<F, RT, true, true>(c, b, g, keys, reach, p0, p1, q, sums, cap, active, hide_rows);
        return;
      }
    }
    forms<F, RT, PAGED, PAGED && !Pairs::ENDS>(c, b, g, keys, reach, p0, p1, q, sums, cap, active, hide_rows);
  }

 private:
  // What a wave does, in two forms, of waves that load and widen K and of those
  // that do V (each SIMD has one of both): registers that two branches load are
  // copied where the branches meet, which waits for the loads.  Both take the
  // same barriers.
  template <typename F, int RT, bool PAGED, bool HOLES, typename Pairs, typename Hide>
  __device__ __forceinline__ void forms(const CacheView& c, int b, int g, int keys, const Pairs& reach, int p0, int p1,
                                        const v8bf (&q)[RT][STEPS], RowSums<RT>& sums, float cap, bool active,
                                        Hide hide_rows) {
    if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= 4) {
      __builtin_amdgcn_s_setprio(1);
      form<F, RT, PAGED, HOLES, true>(c, b, g, keys, reach, p0, p1, q, sums, cap, active, hide_rows);
    } else {
      form<F, RT, PAGED, HOLES, false>(c, b, g, keys, reach, p0, p1, q, sums, cap, active, hide_rows);
    }
  }

  template <typename F, int RT, bool PAGED, bool HOLES, bool V, typename Pairs, typename Hide>
  __device__ __forceinline__ void form(const CacheView& c, int b, int g, int keys, const Pairs& reach, int p0, int p1,
                                       const v8bf (&q)[RT][STEPS], RowSums<RT>& sums, float cap_at, bool active,
                                       Hide hide_rows) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sx = wave & 1, sp = (wave >> 1) & 1;  // it loads tile sx of pair sp
    const int steps = (p1 - p0 + 1) / 2;
    const ScoreScale zs(cap_at);
    const bool cap = cap_at > 0.f;
    // Tiles in flight: with one tile of rows registers are left for more, and 4
    // bits are half the bytes (32 drafts over 131072 keys 110 us with one, 98 with
    // three when that was chosen, then LDS bound, 87 now; in 8 bits 98 with one or
    // two, 91 now)
    constexpr int SETS = RT == 1 && F::BYTES == RECORD_FOUR ? 3 : 1;
    std::conditional_t<V, typename F::V, typename F::K> in[SETS];
    bool hole[SETS];    // of the tile in registers
    Tile ahead;         // the next to load: with ENDS its page is read a step before it is used
    auto find = [&](int it) {  // (past the last pair: its last tile again, not used)
      const int pair = min(p0 + 2 * it + sp, p1 - 1);
      ahead = tile_at<F::BYTES, PAGED>(c, b, g, reach.pair(pair) * TR_PAIR + 16 * sx, keys);
    };
    // (set: it % SETS, known to the compiler)
    auto load = [&](int it, int set) {
      if constexpr (!Pairs::ENDS) find(it);
      if constexpr (V) F::template load_v<false, true>(in[set], ahead, anew(lane));
      else F::template load_k<false>(in[set], ahead, anew(lane));
      hole[set] = ahead.bad;
      if constexpr (Pairs::ENDS) find(it + 1);
    };
    auto widen = [&](int it, int set) {
      uint4* to = buf + (it & 1) * BUF;
      const int pair = min(p0 + 2 * it + sp, p1 - 1);
      const int lane = anew(threadIdx.x) & 63;
      if constexpr (V) {
        if (HOLES && hole[set]) F::clear_v(in[set]);
        if (pair >= reach.whole) {
          const uint32_t any = F::drop_nan(in[set]);
          if (__ballot(any != 0) && lane == 0) nan = 1;
        }
        uint2* out = reinterpret_cast<uint2*>(to + KBUF + sp * 16 * WAVE + lane) + sx;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint2 half[4];
          F::v_halves(in[set], w, half);
#pragma unroll
          for (int i = 0; i < 4; ++i) out[(4 * w + i) * WAVE * 2] = half[i];
        }
      } else {
        uint4* out = to + (sp * 2 + sx) * IMG_TILE + lane;
#pragma unroll
        for (int step = 0; step < STEPS; ++step)
          out[step * WAVE] = __builtin_bit_cast(uint4, F::k_operand(in[set], step));
        if (HOLES && lane == 0) reinterpret_cast<uint8_t*>(&bad[it & 1])[sp * 2 + sx] = hole[set];
      }
    };
    auto advance = [&](int it, int set) {
      if (SETS > 1 || it + 1 < steps) widen(it + 1, set);
      if (SETS > 1 || it + 2 < steps) load(it + 1 + SETS, set);
    };
    if constexpr (Pairs::ENDS) find(0);
#pragma unroll
    for (int d = 0; d < SETS; ++d) load(d, d);
    widen(0, 0);
    if (SETS > 1 || steps > 1) load(SETS, 0);
    __syncthreads();
    // (several sets: loads without a branch, also past the end, since a wait behind
    // one is a wait for all of them)
#pragma nounroll
    for (int it0 = 0; it0 < steps; it0 += SETS)
#pragma unroll
    for (int d = 0; d < SETS; ++d) {
      const int it = it0 + d, set = (d + 1) % SETS;
      const uint4* from = buf + (it & 1) * BUF;
      uint32_t holes = 0;  // a byte for each of the buffer's tiles
      if constexpr (HOLES) holes = __builtin_amdgcn_readfirstlane(bad[it & 1]);
      // the two waves of a SIMD take turns: one widens the next pairs before
      // it computes, the other after, and one has priority, so that one
      // weighs while the other multiplies (64 drafts over 131072 keys: 201 us
      // a call without, 189 with the priority alone, 183 with both, before
      // the waits for records were taken out)
      if (V) advance(it, set);
#pragma nounroll
      for (int pair = 0; pair < 2; ++pair) {
        const int j = p0 + 2 * it + pair;
        if (j >= p1 || !active) break;
        const bool edge = j >= reach.whole;
        const int ln = anew(lane);
        v4f acc[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][0] = acc[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int step = 0; step < STEPS; ++step)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const v8bf kk = __builtin_bit_cast(v8bf, from[((pair * 2 + x) * STEPS + step) * WAVE + ln]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              acc[rt][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[rt][step], acc[rt][x], 0, 0, 0);
          }
        const bool bad0 = HOLES && (holes >> (16 * pair)) & 0xffu, bad1 = HOLES && (holes >> (16 * pair + 8)) & 0xffu;
        v8h pb[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          if (cap) zs.squash(acc[rt]);
          if (edge) hide_rows(std::true_type{}, rt, acc[rt], j, ln, bad0, bad1);
          else if (bad0 || bad1) hide_rows(std::false_type{}, rt, acc[rt], j, ln, bad0, bad1);
          pb[rt] = sums.weigh(rt, acc[rt], zs.unit);
        }
        const uint4* vb = from + KBUF + pair * 16 * WAVE + ln;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const v8h va = __builtin_bit_cast(v8h, vb[i * WAVE]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            sums.o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[rt], sums.o[rt][i], 0, 0, 0);
        }
      }
      if (!V) advance(it, set);
      __syncthreads();
    }
  }
};

}  // namespace skv
