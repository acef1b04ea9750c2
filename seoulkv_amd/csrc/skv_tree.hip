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
// 44, 6.0 TB/s, the record stream; 8 drafts 55, 16 66 (71 in turns): the wait for
// records, since 256 registers a wave leave 8 waves a CU and one pair ahead; 32
// drafts 89, 64 drafts 151, with a cap 173: multiplying and weighing, which two
// waves a SIMD overlap little (loads two or three steps ahead changed nothing
// there).  One draft of many ragged paged sequences: 64 of up to 8192 keys
// (279530 in all) 113 us, 5.1 TB/s, 256 of up to 4096 (504279) 195 us, 5.3 TB/s:
// a share holds pieces of several sequences, each with queries to stage and a
// partial to store.  Loads pay where no wait stands between their issue and
// their use: see the loops' notes on branches and spills (of the two-tile instances
// 4 to 9 registers, outside those loops; of the wide ones with a window 8 to 19, those
// over pages partly inside).
//
// With a window the pairs that no row sees are left out (Reach) and the others
// come whole ones first, so the loop over them is the same: a token of 32 ragged
// paged sequences of up to 32768 keys in windows of 4096 (73000 keys) 40 us, 3.9
// TB/s, pieces of several sequences in a share.
//
// Records of 4 bits (Four) are widened with their scales by the converter.  One
// token over 131072 keys 35 to 38 us (8 bits 51), 8 drafts 43 (55), 16 drafts 58
// (71): 4.6 TB/s at most, since a pair takes as many vector instructions as one of
// 8 bits and half the bytes are in flight (two pairs ahead spilled: 41 us); from
// 17 drafts on as 8 bits, LDS bound.  Two key halves of 4 row waves that widen
// together: 16 drafts 76 us, 12 drafts of ragged sequences 132 against 101.
#include <type_traits>

#include "skv_attend.h"

namespace skv {

namespace {

// A block's share of the pairs of KV head g: the piece of one sequence after
// the other, `piece` called for each.  A single sequence (the latency of short
// contexts) needs no starts.
template <typename F>
__device__ __forceinline__ void each_piece(const TreeArgs& a, int* s_start, F piece) {
  const int g = blockIdx.y, k = blockIdx.x;
  int total;
  if (a.c.batch == 1) {
    total = sequence_pairs<false>(Sequence(a.c, a.counts, a.n, 0).uniform(), a.window);
  } else {
    total = sequence_starts<false>(a.c, a.counts, a.n, a.window, s_start);
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
template <typename F, int RT, int RW, int KW, bool PAGED>
__global__ __launch_bounds__(RW * KW * 64) void k_tree(TreeArgs a) {
  constexpr int WAVES = RW * KW, TILES = RT * RW;
  // Records of 4 bits come through LDS (Four::Raw): one token over 131072 keys 36
  // us a call, 39 without; two tiles of rows leave no registers for it (16 drafts
  // 63, 70 with it).
  constexpr bool STAGED = F::BYTES == RECORD_FOUR && RT == 1;
  constexpr int JOIN = (KW / 2) * RW * RT * 16 * WAVE;
  constexpr int STAGE = 16 * F::BYTES / 16;  // uint4 of a tile
  constexpr int IMG = TILES * IMG_TILE, LOOP = IMG + (STAGED ? WAVES * 2 * STAGE : 0);
  __shared__ uint4 s_buf[LOOP > JOIN ? LOOP : JOIN];  // the queries' image and tiles, then the sums in transit
  __shared__ float2 s_ml[(KW / 2) * RW * RT * WAVE];
  __shared__ Sight s_sight[TILES * 16];
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
    const Reach reach(seq, a.window);
    const int whole = min(p1, first + reach.whole);
    stage_queries<F, WAVES * 64>(a.q, b, g, TILES, seq.rows, s_buf);
    for (int r = threadIdx.x; r < TILES * 16; r += WAVES * 64)
      s_sight[r] = r < seq.rows ? sight_of(seq, a.window, row_mask(a.tree, a.n, b, r / H)) : Sight{0, 0};
    if (threadIdx.x == 0) s_nan = 0;
    Tile t[2];
    typename F::K kx[2];
    typename F::V vx[2];
    auto tiles = [&](int pair) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
        t[x] = tile_at<F::BYTES, PAGED>(a.c, b, g, reach.pair(pair - first) * TR_PAIR + 16 * x, seq.keys);
    };
    int j = p0 + kw;
    std::conditional_t<STAGED, Four::Raw, int> raw[2];
    uint4* const stage = s_buf + IMG + wave * 2 * STAGE;
    if (j < whole) {
      tiles(j);
      if constexpr (STAGED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_raw<true>(raw[x], t[x], lane);
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_k<true>(kx[x], t[x], lane);
        __builtin_amdgcn_sched_barrier(0);  // (in the loop's order, which its waits count)
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_v<true, RW == 1>(vx[x], t[x], lane);
      }
    }
    __syncthreads();

    RowSums<RT> sums;
    sums.clear();
    // one pair; EDGE: some of its keys are drafts or past the end (it loads
    // its records itself); MORE: the wave's next pair is loaded, by code of its
    // own, since a wait behind a branch that may not load is one for all loads
    auto step = [&](auto edge, auto more) {
      constexpr bool EDGE = decltype(edge)::value, MORE = decltype(more)::value;
      const int at = EDGE ? reach.pair(j - first) * TR_PAIR : 0;
      if (EDGE) {
        tiles(j);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if constexpr (STAGED) {
            F::template load_raw<false>(raw[x], t[x], lane);
          } else {
            F::template load_k<false>(kx[x], t[x], lane);
            F::template load_v<false, RW == 1>(vx[x], t[x], lane);
          }
        }
      }
      const bool bad0 = t[0].bad, bad1 = t[1].bad;
      Tile here[2];  // the staged tiles
      if constexpr (STAGED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          F::put_raw(raw[x], stage + x * STAGE, lane);
          here[x] = Tile{reinterpret_cast<const uint8_t*>(stage + x * STAGE), t[x].last, false};
        }
        __builtin_amdgcn_wave_barrier();  // (other lanes read it, below)
      }
      if (MORE) tiles(j + KW);
      if constexpr (STAGED) {
        if (MORE) {
#pragma unroll
          for (int x = 0; x < 2; ++x) F::template load_raw<true>(raw[x], t[x], lane);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_k<!EDGE>(kx[x], here[x], lane);
      }
      v4f acc[RT][2];
      scores<F, RT>(kx, s_buf + rw * RT * IMG_TILE, lane, acc);
      // (done before their records' registers are loaded anew)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int x = 0; x < 2; ++x) asm volatile("" : "+v"(acc[rt][x]));
      if (MORE && !STAGED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_k<true>(kx[x], t[x], lane);
      }
      v8h pb[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (cap) zs.squash(acc[rt]);
        if (EDGE || bad0 || bad1)
          hide<EDGE>(acc[rt], seq, a.window, EDGE ? s_sight[(rw * RT + rt) * 16 + col] : Sight{0, 0}, at + 4 * kb, bad0,
                     bad1);
        pb[rt] = sums.weigh(rt, acc[rt], zs.unit);
      }
      if constexpr (STAGED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_v<!EDGE, false>(vx[x], here[x], lane);
        __builtin_amdgcn_wave_barrier();  // (before it is written again)
      }
      if (bad0) F::clear_v(vx[0]);
      if (bad1) F::clear_v(vx[1]);
      if (EDGE) {
        uint32_t any = 0;
#pragma unroll
        for (int x = 0; x < 2; ++x) any |= F::drop_nan(vx[x]);
        if (__ballot(any != 0) && lane == 0) s_nan = 1;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        v8h va[4];
        v_operands<F>(vx, w, va);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            sums.o[rt][4 * w + i] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(va[i], pb[rt], sums.o[rt][4 * w + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);  // one word's operands live at a time
      }
      if (MORE && !STAGED) {
#pragma unroll
        for (int x = 0; x < 2; ++x) F::template load_v<true, RW == 1>(vx[x], t[x], lane);
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
// records.  Here they widen them together (WideBuffers).
template <typename F, int RT, bool PAGED, bool WINDOW>
__global__ __launch_bounds__(512) void k_tree_wide(TreeArgs a) {
  constexpr int TILES = RT * 8;
  typedef std::conditional_t<WINDOW, Sight, uint64_t> Row;  // (the drafts alone)
  __shared__ WideBuffers wide;
  __shared__ Row s_sight[TILES * 16];
  __shared__ int s_start[CACHE_MAX_BATCH + 1];
  const int g = blockIdx.y, k = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kb = lane >> 4;
  // (formed where it is used: its addresses do not stay in registers)
  auto partials = [&] {
    float* at = a.part;
    asm volatile("" : "+s"(at));
    return Partials(at, a.c.batch, a.n);
  };
  each_piece(a, s_start, [&](int b, int first, int p0, int p1) {
    const Sequence seq = Sequence(a.c, a.counts, a.n, b).uniform();
    const std::conditional_t<WINDOW, Reach, AllPairs> reach(seq, a.window);
    for (int r = threadIdx.x; r < TILES * 16; r += 512) {
      const uint64_t bits = r < seq.rows ? row_mask(a.tree, a.n, b, r / H) : 0;
      if constexpr (WINDOW) s_sight[r] = sight_of(seq, a.window, bits);
      else s_sight[r] = bits & seq.there();
    }
    if (threadIdx.x == 0) wide.nan = 0;
    v8bf q[RT][STEPS];
    load_queries<F>(q, a.q, b, g, 0, seq.rows, wave * RT * 16 + col, kb);
    __syncthreads();  // (wide.nan is 0 before any wave may set it)
    RowSums<RT> sums;
    sums.clear();
    auto hide_rows = [&](auto edge, int rt, v4f (&scores)[2], int pair, int ln, bool bad0, bool bad1) {
      constexpr bool EDGE = decltype(edge)::value;
      hide<EDGE>(scores, seq, a.window, EDGE ? s_sight[(wave * RT + rt) * 16 + (ln & 15)] : Row{},
                 EDGE ? reach.pair(pair) * TR_PAIR + 4 * (ln >> 4) : 0, bad0, bad1);
    };
    wide.template walk<F, RT, PAGED>(a.c, b, g, seq.keys, reach, p0 - first, p1 - first, q, sums, a.cap, true, hide_rows);
    sums.total();
    const Partials part = partials();
    sums.store(part, part.tile(g, k, b), wave * RT, seq.rows, lane);
    __syncthreads();
    if (threadIdx.x == 0) part.nan[g * part.shares + k + b] = wide.nan;
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
template <typename F, int SLICES, int NI>
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
  int stop = total = sequence_pairs<false>(seq, a.window);
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
      const Sight sight = sight_of(seq, a.window, row_mask(a.tree, a.n, b, row / H));
      const Reach reach(seq, a.window);
      for (int e = reach.whole * TR_PAIR; e < reach.all * TR_PAIR; ++e) {
        const int t = reach.pair(e / TR_PAIR) * TR_PAIR + e % TR_PAIR;
        if (t >= seq.keys || !sees(seq, a.window, sight, t)) continue;
        const uint32_t page = a.c.table ? a.c.page(b, t) : 0;
        if (a.c.table && page >= a.c.n_pages) continue;
        const uint8_t* record = a.c.records + (a.c.table ? a.c.row_in(page, g, t) : a.c.row(b, g, t)) * F::BYTES;
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (F::v_is_nan(record, dim + i)) y[i] = __builtin_nanf("");
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
// loaded ahead (32 rows over 131072 keys: 45 us, 70 with 2 waves and a pair
// ahead; 64 rows 70); by the K halves, 256 bytes of every 512, for few (one row
// 28 us a call, 4.8 TB/s).  4 bits as long, bound by their widening (28, 45, 70).  In
// a window of 4096 10, 18 and 26 us, of 100000 27, 44 and 65.  4 waves leave 128
// registers: 8 to 10 are spilled, outside the loop over row tiles, 18 to 23 with a
// window.
// (the 128 KB image of 64 drafts leaves room for one block, of 16 waves then)
constexpr int weight_waves(int tiles) { return tiles > 8 ? 16 : 8; }

template <typename F, int TILES, bool PAGED, bool WINDOW>
__global__ __launch_bounds__(weight_waves(TILES) * 64, 4) void k_key_weights(WeightArgs a) {
  constexpr int WAVES = weight_waves(TILES);
  __shared__ uint4 s_img[TILES * IMG_TILE];
  __shared__ float s_lse[TILES * 16];
  __shared__ std::conditional_t<WINDOW, Sight, uint64_t> s_sight[TILES * 16];  // (the drafts alone)
  __shared__ int s_start[CACHE_MAX_BATCH + 1];
  const int g = blockIdx.y, k = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kb = lane >> 4;
  const ScoreScale zs(a.cap);
  const bool cap = a.cap > 0.f;
  const Window window = WINDOW ? a.window : Window{0, 0};
  const int total = a.c.batch == 1 ? sequence_pairs<true>(Sequence(a.c, a.counts, a.n, 0).uniform(), window)
                                   : sequence_starts<true>(a.c, a.counts, a.n, window, s_start);
  if (WINDOW && !a.accumulate) {
    // the pairs that no row sees: several blocks a sequence, or several sequences a
    // block (every block at all of them, 1024 sequences of 400 slots 568 us, 61 so)
    const int parts = max((int)gridDim.x / a.c.batch, 1);
    for (int u = k; u < a.c.batch * parts; u += gridDim.x) {
      const int b = u / parts, part = u % parts;
      const Reach reach(Sequence(a.c, a.counts, a.n, b), window);
      for (int t = reach.sink_pairs * TR_PAIR + part * WAVES * 64 + threadIdx.x; t < reach.window * TR_PAIR;
           t += parts * WAVES * 64)
        a.weights[a.c.row(b, g, t)] = 0.f;
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
    const Sequence seq = Sequence(a.c, a.counts, a.n, b).uniform();
    const Reach reach(seq, window);
    typename F::K kx[2];
    Tile t0, t1;
    int j = p0 + wave;
    stage_queries<F, WAVES * 64>(a.q, b, g, TILES, seq.rows, s_img);
    for (int r = threadIdx.x; r < TILES * 16; r += WAVES * 64) {
      const int i = r / H;
      const bool row = r < seq.rows;
      if constexpr (WINDOW) s_sight[r] = row ? sight_of(seq, window, row_mask(a.tree, a.n, b, i)) : Sight{0, 0};
      else s_sight[r] = row ? row_mask(a.tree, a.n, b, i) : 0;
      const float lse = row ? a.lse[((size_t)b * a.n + i) * G * H + g * H + r % H] : -INFINITY;
      s_lse[r] = lse == -INFINITY ? INFINITY : lse * DN_LOG2E;  // such a row adds 2^-inf
    }
    __syncthreads();
    const int used = (seq.rows + 15) / 16;
#pragma nounroll
    for (; j < p1; j += WAVES) {
      const int at = (WINDOW ? reach.pair(j - first) : j - first) * TR_PAIR;
      // nothing is loaded ahead: with 4 waves on a SIMD the others compute
      t0 = tile_at<F::BYTES, PAGED>(a.c, b, g, at, seq.keys);
      t1 = tile_at<F::BYTES, PAGED>(a.c, b, g, at + 16, seq.keys);
      F::template load_k<false>(kx[0], t0, lane);
      F::template load_k<false>(kx[1], t1, lane);
      const bool bad0 = t0.bad, bad1 = t1.bad;
      const bool edge = (WINDOW ? j - first >= reach.whole : at + TR_PAIR > seq.len) || bad0 || bad1;
      // widened once for all rows; the records' registers are loaded anew
      v8bf ka[2][STEPS];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int step = 0; step < STEPS; ++step) ka[x][step] = F::k_operand(kx[x], step);
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
            // (a row that adds nothing has no window that would hide a NaN key)
            bool seen = !(e < 4 ? bad0 : bad1);
            const int t = at + 16 * (e >> 2) + 4 * kb + (e & 3);
            if constexpr (WINDOW) seen = seen && lse != INFINITY && sees(seq, window, s_sight[row], t);
            else seen = seen && sees_drafts(seq, s_sight[row], t);
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

template <typename F, bool PAGED>
void tree_rows(const TreeArgs& a, hipStream_t st) {
  const dim3 grid(TR_BLOCKS, G);
  const int tiles = (a.n * H + 15) / 16;
  // up to 4 drafts: one tile of rows a wave (49 us a call on one cache of 131072
  // keys over and over; 57 with two, the second empty; 62 with 12 waves, whose
  // 168 registers spill)
  if (tiles <= 1) hipLaunchKernelGGL((k_tree<F, 1, 1, 8, PAGED>), grid, dim3(512), 0, st, a);
  // two tiles a wave: widened records serve both (16 drafts 66 us, 99 with
  // one); row waves that hold the same records as far as 16 drafts (12 in 64
  // paged sequences of 2000 keys 72 us, 80 when they are widened once into
  // LDS), widened once past them (32 drafts 93 us then, 122 by 4 row waves each for
  // itself; 64 drafts 154 us, 219 by 8)
  else if (tiles <= 2) hipLaunchKernelGGL((k_tree<F, 2, 1, 8, PAGED>), grid, dim3(512), 0, st, a);
  else if (tiles <= 4) hipLaunchKernelGGL((k_tree<F, 2, 2, 4, PAGED>), grid, dim3(512), 0, st, a);
  else {
    auto wide = tiles <= 8 ? (a.window.size ? k_tree_wide<F, 1, PAGED, true> : k_tree_wide<F, 1, PAGED, false>)
                           : (a.window.size ? k_tree_wide<F, 2, PAGED, true> : k_tree_wide<F, 2, PAGED, false>);
    hipLaunchKernelGGL(wide, grid, dim3(512), 0, st, a);
  }
}

template <typename F, bool PAGED, bool WINDOW>
void weight_rows(const WeightArgs& a, hipStream_t st) {
  const int tiles = (a.n * H + 15) / 16;
  const dim3 block(weight_waves(tiles) * 64);
  const dim3 grid(tiles <= 8 ? 2 * TR_BLOCKS : TR_BLOCKS, G);
  if (tiles <= 1) hipLaunchKernelGGL((k_key_weights<F, 1, PAGED, WINDOW>), grid, block, 0, st, a);
  else if (tiles <= 2) hipLaunchKernelGGL((k_key_weights<F, 2, PAGED, WINDOW>), grid, block, 0, st, a);
  else if (tiles <= 4) hipLaunchKernelGGL((k_key_weights<F, 4, PAGED, WINDOW>), grid, block, 0, st, a);
  else if (tiles <= 8) hipLaunchKernelGGL((k_key_weights<F, 8, PAGED, WINDOW>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((k_key_weights<F, 16, PAGED, WINDOW>), grid, block, 0, st, a);
}

}  // namespace

size_t tree_workspace(int batch, int n) {
  const Partials p(nullptr, batch, n);
  return reinterpret_cast<size_t>(p.starts + batch + 1);
}

template <typename F>
static void tree(const TreeArgs& a, hipStream_t st) {
  (a.c.table ? tree_rows<F, true> : tree_rows<F, false>)(a, st);
  const int tiles = a.c.batch * G * ((a.n * H + 15) / 16);
  if (tiles <= 16)
    hipLaunchKernelGGL((k_tree_merge<F, 8, 1>), dim3(tiles * 16), dim3(512), 0, st, a, TR_BLOCKS);
  else if (a.c.batch <= 4)
    hipLaunchKernelGGL((k_tree_merge<F, 8, 4>), dim3(tiles * 4), dim3(512), 0, st, a, TR_BLOCKS);
  else if (a.c.batch <= 16)
    hipLaunchKernelGGL((k_tree_merge<F, 4, 4>), dim3(tiles * 4), dim3(256), 0, st, a, TR_BLOCKS);
  else
    hipLaunchKernelGGL((k_tree_merge<F, 1, 4>), dim3(tiles), dim3(256), 0, st, a, TR_BLOCKS);
}

void launch_tree(const TreeArgs& a, hipStream_t st) { (a.c.four ? tree<Four> : tree<Eight>)(a, st); }

template <typename F, bool WINDOW>
static void key_weights(const WeightArgs& a, hipStream_t st) {
  (a.c.table ? weight_rows<F, true, WINDOW> : weight_rows<F, false, WINDOW>)(a, st);
}

void launch_key_weights(const WeightArgs& a, hipStream_t st) {
  // (a window's bookkeeping in every instance: 32 rows over 131072 keys 58 us, 47 without)
  if (a.window.size) (a.c.four ? key_weights<Four, true> : key_weights<Eight, true>)(a, st);
  else (a.c.four ? key_weights<Four, false> : key_weights<Eight, false>)(a, st);
}

}  // namespace skv
