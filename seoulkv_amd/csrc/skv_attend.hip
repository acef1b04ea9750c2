// Attention of a chain of any length over a record cache (interface in
// skv_cache.h; scores, sums and their precision: skv_tree.hip).
//
// A block takes 64 tokens of a sequence with the 4 query heads of a KV head,
// 256 rows: eight waves of 32 rows that widen the records together (WideBuffers).
// Row i of the chain sees what lies before slot lengths + i + 1; only the pairs
// at the chain's end and at the window's two ends are masked, the others run
// without a test.
//
// Neighbours, 64-token blocks of one list (sequence and KV head), run side by
// side on one XCD, so that its L2 reads a record once for them.
//
// Many blocks (a prompt): one each, those with the most keys first.  Fewer than
// AT_FEW (a piece of a prompt, a ragged batch) would leave CUs idle or busy for
// unlike times: k_attend_plan cuts the pairs of neighbours at the same places into
// pieces of like length that fill the CUs once or twice, and k_attend_merge joins
// the pieces of a block in order (equal shares of all pairs, each a loop over
// what it holds of several blocks: 700 tokens over 20000 keys 258 us against 255,
// over 100000 1128 against 1035; the loop's registers spilled loaded records).
//
// Bounds: a pair of tiles takes 256 KB of LDS reads (2048 cycles) beside as many
// cycles of matrix cores and four fifths of that of vector units, which two waves
// a SIMD overlap in part.  Whole calls: prompt of 16384 all visible 1900 us, 1157
// TFLOP/s (a library product of 16384^3: 1364), 4-bit records 1845, 1192; in a window
// of 4096 with 128 sinks 970, 1019; 2000 capped tokens of 4 bits in a window of
// 8192 317, 855; ragged paged pieces of 6 prompts 452, 800.
#include "skv_attend.h"

namespace skv {

namespace {

constexpr int AT_TOKENS = 64, AT_ROWS = AT_TOKENS * H, AT_RT = 2, AT_TILES = AT_ROWS / 16;
// Fewer blocks are cut into pieces (fresh prompts: 4096 tokens, 256 blocks, 199 us,
// 239 a block each; 7000, 440 blocks, 432 and 394; 700 tokens over 20000 keys, 44
// blocks, 256 and 1088)
constexpr int AT_FEW = 384;
constexpr int AT_CUS = 256, AT_PIECES = 2 * AT_CUS;
constexpr int AT_NEAR = 4;      // neighbours that are cut alike
constexpr int AT_LEAST = 4;     // pairs of a piece (512 fresh tokens 35 to 37 us, 47 with 16)
constexpr int AT_COST = 12;     // pairs that a piece costs beside its own: some 25 us of 2 a pair

// What row `token` of a chain sees: slots [first, last] and the sink.
struct Span {
  int first, last;
  __device__ Span(int len, int keys, int token, const Window& w)
      : last(min(len + token, keys - 1)) {
    first = w.size ? max(0, last + 1 - w.size) : 0;
  }
  __device__ __forceinline__ bool sees(const Window& w, int t) const { return t <= last && (t >= first || t < w.sink); }
};

// 64 tokens of a sequence.
struct Tokens {
  int len, keys, first, rows;  // first token; rows that are no padding
  // alike: the whole wave is at this block
  __device__ Tokens(const AttendArgs& a, int b, int block, bool alike = true) {
    len = a.c.length(b);
    int count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
    if (alike) {
      len = __builtin_amdgcn_readfirstlane(len);
      count = __builtin_amdgcn_readfirstlane(count);
    }
    first = block * AT_TOKENS;
    rows = H * min(max(count - first, 0), AT_TOKENS);
    keys = len + min(count, a.c.capacity - len);
  }
  __device__ Reach reach(const Window& w) const {
    const Span early(len, keys, first, w), late(len, keys, first + rows / H - 1, w);
    return Reach(early.last + 1, late.last + 1, early.first, late.first, w);
  }
};

// Some pairs of a block of tokens; index: of their sums, -1 if they are all;
// p1 = 0: none.
struct Piece {
  int item, p0, p1, index;
};
// Of a block: the index of its first piece, from one to the next, their number
// (0: no rows).
struct Parts {
  int first, step, count;
};

// Pieces' sums, as the waves hold them, flags of NaN, the plan.
struct AttendPartials {
  float4* o;
  float2* stats;
  Piece* plan;  // of block x of the grid
  Parts* parts;
  int* nan;
  __host__ __device__ explicit AttendPartials(void* work) {
    o = static_cast<float4*>(work);
    stats = reinterpret_cast<float2*>(o + (size_t)AT_PIECES * AT_TILES * 16 * WAVE);
    plan = reinterpret_cast<Piece*>(stats + AT_PIECES * AT_TILES * 16);
    parts = reinterpret_cast<Parts*>(plan + AT_PIECES);
    nan = reinterpret_cast<int*>(parts + AT_FEW);
  }
  __host__ size_t end() const { return reinterpret_cast<size_t>(nan + AT_PIECES); }
};

// Sum over the threads before this one of a block of 512; sums: of its waves.
__device__ __forceinline__ int block_before(int v, int* sums) {
  const int inc = wave_incl_scan(v), wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) sums[wave] = inc;
  __syncthreads();
  int before = inc - v;
  for (int w = 0; w < wave; ++w) before += sums[w];
  __syncthreads();
  return before;
}

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Thread u takes neighbours u, AT_NEAR blocks of a list, or those that are left,
// and then piece u (65 tokens over 8000 keys 5.3 us; threads that write their
// neighbours' pieces one after the other 9.0).
__global__ __launch_bounds__(512) void k_attend_plan(AttendArgs a, int blocks) {
  static_assert(AT_PIECES == 512 && AT_FEW <= 512, "a thread each");
  __shared__ int s_pairs[512], s_blocks[512], s_own[512], s_even[512], s_by_rank[512], s_at_rank[512], s_sums[8];
  const AttendPartials part(a.work);
  const int per = (blocks + AT_NEAR - 1) / AT_NEAR, groups = a.c.batch * G * per, u = threadIdx.x;
  const int list = u / per, first = u % per * AT_NEAR, count = min(AT_NEAR, blocks - first);
  int own[AT_NEAR], most = 0, live = 0;  // pairs of each; blocks that have rows
#pragma unroll
  for (int r = 0; r < AT_NEAR; ++r) {
    own[r] = 0;
    if (u < groups && r < count) {
      const Tokens tok(a, list / G, first + r, /*alike=*/false);
      if (tok.rows) own[r] = tok.reach(a.window).all;
      s_own[list * blocks + first + r] = own[r];
    }
    most = max(most, own[r]);
    live += own[r] > 0;
  }
  s_pairs[u] = most;
  s_blocks[u] = live;
  __syncthreads();
  // The least length of a piece for which there are at most `limit` of them
  // (every wave finds it by itself).
  int longest = 0, all = 0, total = 0;  // (fewer than 2^24 pairs: 512 blocks of 2^15)
  for (int v = u & 63; v < groups; v += 64) {
    longest = max(longest, s_pairs[v]);
    all += s_blocks[v];
    total += s_pairs[v] * s_blocks[v];
  }
  longest = wave_max(longest);
  all = wave_sum(all);
  total = wave_sum(total);
  auto least = [&](int limit) {
    // the answer lies in [lo, hi]: total / x to total / x + all pieces of x
    int lo = min(max(AT_LEAST, ceil_div(total, limit)), longest), hi = longest;
    if (all < limit) hi = max(lo, min(hi, ceil_div(total, limit - all)));
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      int pieces = 0;
      for (int v = u & 63; v < groups; v += 64) pieces += s_blocks[v] * ceil_div(s_pairs[v], mid);
      if (wave_sum(pieces) <= limit) hi = mid;
      else lo = mid + 1;
    }
    return max(lo, 1);
  };
  int length = least(AT_PIECES);
  if (all <= AT_CUS) {  // filled once if that ends no later than filled twice
    const int once = least(AT_CUS);
    if (once + AT_COST <= 2 * (length + AT_COST)) length = once;
  }
  // neighbours with the most pairs first
  int rank = 0;
  for (int v = 0; v < groups; ++v) rank += s_pairs[v] > most || (s_pairs[v] == most && v < u);
  const int shares = ceil_div(most, length), even = shares ? ceil_div(most, shares) : 1;
  s_even[u] = even;
  s_by_rank[u] = 0;
  __syncthreads();
  if (u < groups) {
    s_by_rank[rank] = live * shares;
    s_at_rank[rank] = u;
  }
  __syncthreads();
  const int held = s_by_rank[u], before = block_before(held, s_sums);
  s_by_rank[u] = before;
  if (u == 511) s_sums[0] = before + held;
  __syncthreads();
  if (u < groups)
#pragma unroll
    for (int r = 0; r < AT_NEAR; ++r)  // (neighbours with rows come first in a list)
      if (r < count) part.parts[list * blocks + first + r] = Parts{s_by_rank[rank] + r, live, ceil_div(own[r], even)};
  // piece u is of the last neighbours that begin at or before it
  Piece piece{0, 0, 0, 0};
  if (u < s_sums[0]) {
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_by_rank[mid] <= u) lo = mid;
      else hi = mid;
    }
    const int v = s_at_rank[lo], local = u - s_by_rank[lo], r = local % s_blocks[v], p0 = local / s_blocks[v] * s_even[v];
    const int item = v / per * blocks + v % per * AT_NEAR + r;
    if (p0 < s_own[item]) piece = Piece{item, p0, min(s_own[item], p0 + s_even[v]), s_own[item] > s_even[v] ? u : -1};
  }
  // blocks x % 8 are on one XCD: it gets AT_NEAR pieces in a row
  part.plan[(u / (8 * AT_NEAR) * AT_NEAR + u % AT_NEAR) * 8 + u / AT_NEAR % 8] = piece;
}

// Whether a key that a row sees and that lies in an edge has NaN in `dim` (the
// walk took it as 0).
template <typename F>
__device__ bool edge_nan(const AttendArgs& a, int b, int g, const Reach& reach, int keys, const Span& span, int dim) {
  for (int e = reach.whole * TR_PAIR; e < reach.all * TR_PAIR; ++e) {
    const int t = reach.pair(e / TR_PAIR) * TR_PAIR + e % TR_PAIR;
    if (t >= keys || !span.sees(a.window, t)) continue;
    const uint32_t page = a.c.table ? a.c.page(b, t) : 0;
    if (a.c.table && page >= a.c.n_pages) continue;
    if (F::v_is_nan(a.c.records + (a.c.table ? a.c.row_in(page, g, t) : a.c.row(b, g, t)) * F::BYTES, dim)) return true;
  }
  return false;
}

// Rows of padding give 0 and -inf.
__device__ __forceinline__ void clear_padding(const AttendArgs& a, int b, int g, const Tokens& tok) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int end = min(a.n - tok.first, AT_TOKENS) * H;
  for (int row = tok.rows + wave; row < end; row += 8) {
    const size_t at = (((size_t)b * a.n + tok.first + row / H) * G + g) * H + row % H;
    reinterpret_cast<uint2*>(a.out + at * D)[lane] = make_uint2(0, 0);
    if (lane == 0) a.lse[at] = -INFINITY;
  }
}

template <typename F, bool PAGED, bool PIECES>
__global__ __launch_bounds__(512) void k_attend(AttendArgs a, int blocks) {
  __shared__ WideBuffers wide;
  __shared__ int2 s_span[AT_ROWS];
  const int lists = a.c.batch * G;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // pairs p0 .. p1 - 1 of 64 tokens, all of them or (index >= 0) some
  auto piece = [&](int list, int block, int p0, int p1, int index) {
    const int b = list / G, g = list % G;
    const Tokens tok(a, b, block);
    const Reach reach = tok.reach(a.window);
    for (int r = anew(threadIdx.x); r < AT_ROWS; r += 512) {
      const Span s(tok.len, tok.keys, tok.first + min(r, tok.rows - 1) / H, a.window);
      s_span[r] = make_int2(s.first, s.last);
    }
    if (threadIdx.x == 0) wide.nan = 0;
    v8bf q[AT_RT][STEPS];
    {
      const int lane = anew(threadIdx.x) & 63;
      load_queries<F>(q, a.q, b, g, tok.first, tok.rows, wave * AT_RT * 16 + (lane & 15), lane >> 4);
    }
    __syncthreads();  // (wide.nan is 0 before any wave may set it)
    RowSums<AT_RT> sums;
    sums.clear();
    auto hide_rows = [&](auto edge, int rt, v4f (&scores)[2], int pair, int ln, bool bad0, bool bad1) {
      constexpr bool EDGE = decltype(edge)::value;
      const int2 span = EDGE ? s_span[(wave * AT_RT + rt) * 16 + (ln & 15)] : make_int2(0, 0);
      const int at = EDGE ? reach.pair(pair) * TR_PAIR + 4 * (ln >> 4) : 0;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int t = at + 16 * x;
        uint32_t seen = ~0u;
        if (EDGE) {
          const uint32_t late = ~0u << min(max(span.x - t, 0), 31), early = (1u << min(max(a.window.sink - t, 0), 31)) - 1u;
          seen = (late | early) & ((1u << min(max(span.y + 1 - t, 0), 31)) - 1u);
        }
        if (x ? bad1 : bad0) seen = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) scores[x][r] = (seen >> r) & 1u ? scores[x][r] : -INFINITY;
      }
    };
    wide.template walk<F, AT_RT, PAGED>(a.c, b, g, tok.keys, reach, p0, p1, q, sums, a.cap,
                                        wave * AT_RT * 16 < tok.rows, hide_rows);
    sums.total();
    const int lane = anew(threadIdx.x) & 63, kb = lane >> 4, row0 = wave * AT_RT * 16 + (lane & 15);
    if (PIECES && index >= 0) {
      const AttendPartials part(a.work);
#pragma unroll
      for (int rt = 0; rt < AT_RT; ++rt) {
        if (row0 + rt * 16 >= tok.rows) continue;
        const size_t at = (size_t)index * AT_TILES + wave * AT_RT + rt;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          part.o[(at * 16 + i) * WAVE + lane] =
              make_float4(sums.o[rt][i][0], sums.o[rt][i][1], sums.o[rt][i][2], sums.o[rt][i][3]);
        if (lane < 16) part.stats[at * 16 + lane] = make_float2(sums.m[rt], sums.l[rt]);
      }
      if (threadIdx.x == 0) part.nan[index] = wide.nan;
      return;
    }
    auto out_row = [&](int row) { return (((size_t)b * a.n + tok.first + row / H) * G + g) * H + row % H; };
#pragma unroll
    for (int rt = 0; rt < AT_RT; ++rt) {
      const int row = row0 + rt * 16;
      if (row >= tok.rows) continue;
      const float l = sums.l[rt], inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t* out = a.out + out_row(row) * D + 64 * kb;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)  // (a row that saw nothing has sums of 0)
          w[i] = bf16_rne(sums.o[rt][2 * i][r] * inv) | bf16_rne(sums.o[rt][2 * i + 1][r] * inv) << 16;
        reinterpret_cast<uint4*>(out + 16 * r)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(out + 16 * r)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
      if (kb == 0) a.lse[out_row(row)] = l == 0.f ? -INFINITY : (sums.m[rt] + __log2f(l)) * TR_LN2;
    }
    if (wide.nan) {
      __syncthreads();
      for (int at = threadIdx.x; at < tok.rows * D; at += 512) {
        const int row = at / D, dim = at % D;
        const Span span(tok.len, tok.keys, tok.first + row / H, a.window);
        if (edge_nan<F>(a, b, g, reach, tok.keys, span, dim)) a.out[out_row(row) * D + dim] = 0x7fc0;
      }
    }
  };

  if constexpr (!PIECES) {
    // blocks x % 8 are on one XCD; 8 there in turn are neighbours of one list, the
    // lists turned by one XCD from one group of neighbours to the next, so that
    // long sequences are spread
    const int k = blockIdx.x / 8, eight = k / 8, turn = eight * 8 / lists;
    const int group = eight * 8 + (blockIdx.x + turn) % 8, list = group % lists;
    const int block = blocks - 1 - (group / lists * 8 + k % 8);
    if (block < 0) return;
    const Tokens tok(a, list / G, block);
    clear_padding(a, list / G, list % G, tok);
    if (tok.rows) piece(list, block, 0, tok.reach(a.window).all, -1);
  } else {
    if ((int)blockIdx.x < lists * blocks) {
      const int list = blockIdx.x / blocks;
      clear_padding(a, list / G, list % G, Tokens(a, list / G, blockIdx.x % blocks));
    }
    const Piece x = AttendPartials(a.work).plan[blockIdx.x];
    const int p1 = __builtin_amdgcn_readfirstlane(x.p1), item = __builtin_amdgcn_readfirstlane(x.item);
    if (p1)
      piece(item / blocks, item % blocks, __builtin_amdgcn_readfirstlane(x.p0), p1,
            __builtin_amdgcn_readfirstlane(x.index));
  }
}

// Joins the pieces of a tile of 16 rows; wave w the sums 4 w .. +3.
template <typename F>
__global__ __launch_bounds__(256) void k_attend_merge(AttendArgs a, int blocks) {
  const int tile = blockIdx.x % AT_TILES, item = blockIdx.x / AT_TILES;
  const int list = item / blocks, b = list / G, g = list % G;
  const int lane = threadIdx.x & 63, i0 = 4 * (threadIdx.x >> 6), row = tile * 16 + (lane & 15);
  const AttendPartials part(a.work);
  const Parts parts = part.parts[item];
  if (parts.count < 2) return;
  const Tokens tok(a, b, item % blocks);
  if (row >= tok.rows) return;
  const Reach reach = tok.reach(a.window);
  float m = -INFINITY, l = 0.f;
  v4f o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v4f{0.f, 0.f, 0.f, 0.f};
  int nan = 0;
#pragma unroll 2
  for (int k = 0; k < parts.count; ++k) {
    const int index = parts.first + k * parts.step;
    const size_t at = (size_t)index * AT_TILES + tile;
    const float2 ml = part.stats[at * 16 + (lane & 15)];
    nan |= part.nan[index];
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = part.o[(at * 16 + i0 + i) * WAVE + lane];
    const float mn = fmaxf(m, ml.x);
    const float f0 = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    const float f1 = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - mn);
    m = mn;
    l = fmaf(l, f0, ml.y * f1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int r = 0; r < 4; ++r) o[i][r] = fmaf(o[i][r], f0, v[r] * f1);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const size_t out_row = (((size_t)b * a.n + tok.first + row / H) * G + g) * H + row % H;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int dim = 64 * (lane >> 4) + 16 * r + i0;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = o[i][r] * inv;
    if (nan) {
      const Span span(tok.len, tok.keys, tok.first + row / H, a.window);
#pragma nounroll
      for (int i = 0; i < 4; ++i)
        if (edge_nan<F>(a, b, g, reach, tok.keys, span, dim + i)) y[i] = __builtin_nanf("");
    }
    *reinterpret_cast<uint2*>(a.out + out_row * D + dim) =
        make_uint2(bf16_rne(y[0]) | bf16_rne(y[1]) << 16, bf16_rne(y[2]) | bf16_rne(y[3]) << 16);
  }
  if (i0 == 0 && lane < 16) a.lse[out_row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * TR_LN2;
}

int blocks_of(int n) { return (n + AT_TOKENS - 1) / AT_TOKENS; }

template <typename F>
void attend(const AttendArgs& a, hipStream_t st) {
  const int blocks = blocks_of(a.n), lists = a.c.batch * G, items = lists * blocks;
  if (items >= AT_FEW) {
    const int groups = lists * ((blocks + 7) / 8);
    auto kernel = a.c.table ? k_attend<F, true, false> : k_attend<F, false, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((groups + 7) / 8 * 64)), dim3(512), 0, st, a, blocks);
    return;
  }
  auto kernel = a.c.table ? k_attend<F, true, true> : k_attend<F, false, true>;
  hipLaunchKernelGGL(k_attend_plan, dim3(1), dim3(512), 0, st, a, blocks);
  hipLaunchKernelGGL(kernel, dim3(AT_PIECES), dim3(512), 0, st, a, blocks);
  hipLaunchKernelGGL((k_attend_merge<F>), dim3((unsigned)(items * AT_TILES)), dim3(256), 0, st, a, blocks);
}

}  // namespace

size_t attend_workspace(int batch, int n) {
  if (n <= TREE_MAX_DRAFTS) return tree_workspace(batch, n);
  if ((int64_t)batch * G * blocks_of(n) >= AT_FEW) return 0;
  return AttendPartials(nullptr).end();
}

void launch_attend(const AttendArgs& a, hipStream_t st) {
  if (a.n <= TREE_MAX_DRAFTS) {
    TreeArgs t{};
    t.c = a.c;
    t.q = a.q;
    t.n = a.n;
    t.counts = a.counts;
    t.cap = a.cap;
    t.window = a.window;
    t.part = static_cast<float*>(a.work);
    t.out = a.out;
    t.lse = a.lse;
    launch_tree(t, st);
    return;
  }
  (a.c.four ? attend<Four> : attend<Eight>)(a, st);
}

}  // namespace skv
