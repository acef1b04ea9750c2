// Eviction by accumulated attention weight (interface in skv_cache.h).
//
// Which slots stay: the weights are ordered by a 32-bit image, and the value
// at the cut is found digit by digit (11, 11 and 10 bits) from histograms; of
// the slots at that value the lowest ones stay.  Up to EV_ONE middle slots are
// one block's work per (sequence, KV head), the weights read once and held in
// registers: 16000 slots in 13.8 us, against 61 with a pass over memory per 8
// bits and one thread walking the bins, and 26 spread over blocks.  Longer
// lists are spread over blocks of EV_CHUNK slots: a launch per digit, one for
// the counts of every chunk, one for the list; 131072 slots in pages in 27 us
// (3.0 to clear and look for holes, 3 x 4.6, 4.5, 5.7), against 250 by one
// block.  These launches are
// bound by their latency (a chain of load, scan, atomic), not by their bytes.
//
// A slot whose page is none holds no key, so it neither stays nor counts: all
// of this works on the ranks of the slots that have a page (Held), which are
// the slots themselves unless a table has such holes (34.4 us a call for these
// 131072 slots, 32.9 without the search).
//
// The list holds the ranks of the middle that stay, in order; what lies before
// and behind them is sink and local.  k_evict_copy moves the records, 32 lanes
// a record: 4 x 4 x 8192 records in 30 us, 4.6 TB/s read and written (35 where
// weight and position were stored before the record was loaded).
#include "skv_cache.h"
#include "skv_device.h"

namespace skv {

namespace {

constexpr int EV_BLOCK = 1024;
constexpr int EV_ONE = 32 * EV_BLOCK;       // most middle slots that one block takes: 32 a thread
constexpr int EV_CHUNK = 4096;              // slots of a block of the long path: 4 a thread
constexpr int EV_CHUNKS = CACHE_MAX_SLOTS / EV_CHUNK;
constexpr int EV_BINS = 2048;
constexpr int EV_SHIFT[3] = {21, 10, 0};    // the digits: bits 31..21, 20..10, 9..0
constexpr int EV_COPY = 256;                // threads of a copy block: 8 records at a time
constexpr int EV_COPY_SLOTS = 32;

// Larger weight, larger value; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t weight_order(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return w != w ? 0u : o;
}

// The committed slots of a sequence that have a page, in order.
struct Held {
  int count;
  const int* before;  // of those, before each page; NULL: all slots have one
  int pages, shift;

  __device__ __forceinline__ int slot(int rank) const {
    if (!before) return rank;
    int lo = 0, hi = pages;  // the last page that has no more before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= rank) lo = mid;
      else hi = mid;
    }
    return (lo << shift) + rank - before[lo];
  }
};

__device__ __forceinline__ int pages_of(const CacheView& c, int len) {
  return (len + (1 << c.shift) - 1) >> c.shift;
}

// Finds them, by a whole block, and notes them for the launches that follow.
__device__ __forceinline__ Held find_held(const EvictArgs& a, int list, int* scratch) {
  const int b = list / G, len = a.from.length(b);
  if (!a.from.table) return {len, nullptr, 0, 0};
  const int pages = pages_of(a.from, len), page_tokens = 1 << a.from.shift;
  int* before = a.before + (size_t)list * a.before_stride;
  bool hole = false;
  for (int p = threadIdx.x; p < pages; p += EV_BLOCK)
    hole |= a.from.page(b, p << a.from.shift) >= a.from.n_pages;
  int count = len;
  if (__syncthreads_or(hole)) {
    count = 0;
    for (int p0 = 0; p0 < pages; p0 += EV_BLOCK) {
      const int p = p0 + (int)threadIdx.x, t = p << a.from.shift;
      const bool there = p < pages && a.from.page(b, t) < a.from.n_pages;
      int total;
      const int n = block_excl_scan(there ? min(page_tokens, len - t) : 0, scratch, &total);
      if (p < pages) before[p] = count + n;
      count += total;
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) a.held[list] = count;
  return {count, count < len ? before : nullptr, pages, a.from.shift};
}

// What find_held noted in an earlier launch.
__device__ __forceinline__ Held noted_held(const EvictArgs& a, int list) {
  const int len = a.from.length(list / G);
  if (!a.from.table) return {len, nullptr, 0, 0};
  const int count = a.held[list];
  return {count, count < len ? a.before + (size_t)list * a.before_stride : nullptr, pages_of(a.from, len),
              a.from.shift};
}

// What stays of `len` slots: all of them (need 0), or the first sink, the last
// local and `need` of [sink, last).
struct Split {
  int last, need;
  __device__ Split(const EvictArgs& a, int len) {
    last = len - a.local;
    need = len <= a.keep ? 0 : a.keep - a.sink - a.local;
  }
};

// The bin of `hist` (EV_BINS, by all 1024 threads) in which the left-th item
// from the top lies; *above: items in higher bins.
__device__ __forceinline__ int cut_bin(const int* hist, int left, int* scratch, int* s_cut, int* above) {
  const int hi = EV_BINS - 1 - 2 * (int)threadIdx.x;  // the thread's bins: hi, hi - 1
  const int a = hist[hi], b = hist[hi - 1];
  int total;
  const int before = block_excl_scan(a + b, scratch, &total);
  if (before < left && left <= before + a + b) {
    const bool lower = left > before + a;
    s_cut[0] = hi - lower;
    s_cut[1] = before + (lower ? a : 0);
  }
  __syncthreads();
  *above = s_cut[1];
  return s_cut[0];
}

// Adds the bin of every lane to a histogram in LDS; a wave whose lanes agree
// adds once.
__device__ __forceinline__ void count_bin(int* hist, bool on, int bin) {
  const uint64_t lanes = __ballot(on);
  if (!lanes) return;
  const int first = __builtin_amdgcn_readlane(bin, __builtin_ctzll(lanes));
  if (__ballot(on && bin == first) == lanes) {
    if ((threadIdx.x & 63) == __builtin_ctzll(lanes)) atomicAdd(&hist[first], __popcll(lanes));
  } else if (on) {
    atomicAdd(&hist[bin], 1);
  }
}

// A wave holds 64 N consecutive ranks, lane l the ranks t + 64 i + l (loads of
// whole lines; a thread with N consecutive slots read every line N times).
template <int N>
struct Items {
  uint32_t o[N];
  int t, last;  // lane 0's first rank; ranks from `last` on are none

  __device__ Items(const float* w, const Held& held, int begin, int last) : last(last) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    t = begin + wave * WAVE * N;
    if (!held.before) {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = weight_order(on(i) ? w[rank(i)] : 0.f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = weight_order(on(i) ? w[held.slot(rank(i))] : 0.f);
    }
  }
  __device__ __forceinline__ int rank(int i) const { return t + WAVE * i + (int)(threadIdx.x & 63); }
  __device__ __forceinline__ bool on(int i) const { return rank(i) < last; }
  // The wave's items above, and at, the cut.
  __device__ __forceinline__ int above(uint32_t cut) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(on(i) && o[i] > cut));
    return n;
  }
  __device__ __forceinline__ int tied(uint32_t cut) const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(on(i) && o[i] == cut));
    return n;
  }
};

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The sum of a value per wave over the waves before this one; *total: over all.
__device__ __forceinline__ int waves_before(int v, int* scratch, int* total) {
  return __builtin_amdgcn_readfirstlane(block_excl_scan((threadIdx.x & 63) == 0 ? v : 0, scratch, total));
}

// Writes the ranks that stay, those above the cut and the first `left` at it,
// from list[at] on (`ties`: items at the cut before this block's).
template <int N>
__device__ __forceinline__ void list_staying(const Items<N>& x, uint32_t cut, int left, int ties, int at,
                                             int (*scan)[SCAN_WAVES], int* list) {
  int total;
  int tie_rank = ties + waves_before(x.tied(cut), scan[0], &total);
  uint64_t stay[N];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool tie = x.on(i) && x.o[i] == cut;
    const uint64_t tied = __ballot(tie);
    stay[i] = __ballot((x.on(i) && x.o[i] > cut) || (tie && tie_rank + lanes_below(tied) < left));
    tie_rank += __popcll(tied);
    mine += __popcll(stay[i]);
  }
  at += waves_before(mine, scan[1], &total);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((stay[i] >> (threadIdx.x & 63)) & 1) list[at + lanes_below(stay[i])] = x.rank(i);
    at += __popcll(stay[i]);
  }
}

// A whole list by one block, PER slots a thread; sets to_lengths.
template <int PER>
__global__ __launch_bounds__(EV_BLOCK) void k_evict_one(EvictArgs a, int* kept) {
  const int b = blockIdx.x / G;
  __shared__ int s_hist[EV_BINS], s_cut[2], s_scan[3][SCAN_WAVES];
  const Held held = find_held(a, blockIdx.x, s_scan[0]);
  const Split s(a, held.count);
  if (blockIdx.x % G == 0 && threadIdx.x == 0) a.to_lengths[b] = min(held.count, a.keep);
  if (s.need == 0) return;
  const Items<PER> x(a.weights + a.from.row(b, blockIdx.x % G, 0), held, a.sink, s.last);
  uint32_t cut = 0;   // the digits found so far
  int left = s.need;  // items to take among those with these digits
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int shift = EV_SHIFT[d];
    s_hist[threadIdx.x] = 0;
    s_hist[threadIdx.x + EV_BLOCK] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int up = EV_SHIFT[d ? d - 1 : 0];
      const bool in = x.on(i) && (d == 0 || (x.o[i] >> up) == (cut >> up));
      count_bin(s_hist, in, (int)((x.o[i] >> shift) & (d == 2 ? 1023 : 2047)));
    }
    __syncthreads();
    int above;
    cut |= (uint32_t)cut_bin(s_hist, left, s_scan[d], s_cut, &above) << shift;
    left -= above;
    __syncthreads();
  }
  list_staying(x, cut, left, 0, 0, s_scan, kept + (size_t)blockIdx.x * a.keep);
}

// ----------------------------------------------------------- the long path
// Workspace beside the list, per list: a histogram per digit, the cut and what
// is left to take at it after each digit, (items above, items at the cut) of
// every chunk.
struct LongWork {
  int* hist;    // [lists][3][EV_BINS]
  int2* found;  // [lists][3]
  int2* count;  // [lists][chunks]
};

// Clears n words; with `lists` more blocks, one for each list, finds what its
// sequence holds.
__global__ __launch_bounds__(EV_BLOCK) void k_evict_clear(EvictArgs a, int* hist, int n, int lists) {
  __shared__ int s_scan[SCAN_WAVES];
  if ((int)blockIdx.x < lists) {
    (void)find_held(a, blockIdx.x, s_scan);
    return;
  }
  const int i = (blockIdx.x - lists) * EV_BLOCK + threadIdx.x;
  if (i < n) hist[i] = 0;
}

// The cut and what is left to take at it after `digits` digits, from the last
// one's histogram and what was found before it; block 0 of a list notes it.
__device__ __forceinline__ uint32_t cut_so_far(const LongWork& work, int list, int digits, int need, int* scan,
                                               int* s_cut, int* left) {
  uint32_t cut = 0;
  *left = need;
  if (digits == 0) return cut;
  if (digits > 1) {
    const int2 found = work.found[list * 3 + digits - 2];
    cut = (uint32_t)found.x;
    *left = found.y;
  }
  int above;
  cut |= (uint32_t)cut_bin(work.hist + ((size_t)list * 3 + digits - 1) * EV_BINS, *left, scan, s_cut, &above)
         << EV_SHIFT[digits - 1];
  *left -= above;
  if (blockIdx.x == 0 && threadIdx.x == 0) work.found[list * 3 + digits - 1] = make_int2((int)cut, *left);
  return cut;
}

constexpr int EV_LPER = EV_CHUNK / EV_BLOCK;

// Histogram of digit d over one chunk (grid x) of a list (grid y).
__global__ __launch_bounds__(EV_BLOCK) void k_evict_digit(EvictArgs a, LongWork work, int d) {
  const int b = blockIdx.y / G;
  const Held held = noted_held(a, blockIdx.y);
  const Split s(a, held.count);
  if (d == 0 && blockIdx.x == 0 && blockIdx.y % G == 0 && threadIdx.x == 0)
    a.to_lengths[b] = min(held.count, a.keep);
  const int t0 = a.sink + blockIdx.x * EV_CHUNK;
  if (s.need == 0 || t0 >= s.last) return;
  __shared__ int s_hist[EV_BINS], s_cut[2], s_scan[SCAN_WAVES];
  int* hist = work.hist + ((size_t)blockIdx.y * 3 + d) * EV_BINS;
  const Items<EV_LPER> x(a.weights + a.from.row(b, blockIdx.y % G, 0), held, t0, s.last);
  s_hist[threadIdx.x] = 0;
  s_hist[threadIdx.x + EV_BLOCK] = 0;
  int left;
  const uint32_t cut = cut_so_far(work, blockIdx.y, d, s.need, s_scan, s_cut, &left);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EV_LPER; ++i) {
    const int up = d == 0 ? 0 : EV_SHIFT[d - 1];
    const bool in = x.on(i) && (d == 0 || (x.o[i] >> up) == (cut >> up));
    count_bin(s_hist, in, (int)((x.o[i] >> EV_SHIFT[d]) & (d == 2 ? 1023 : 2047)));
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < EV_BINS; i += EV_BLOCK)
    if (const int n = s_hist[i]) atomicAdd(&hist[i], n);
}

// PASS 0: a chunk's items above and at the cut; PASS 1: its part of the list.
template <int PASS>
__global__ __launch_bounds__(EV_BLOCK) void k_evict_list(EvictArgs a, LongWork work, int* kept) {
  const int b = blockIdx.y / G, chunks = gridDim.x;
  const Held held = noted_held(a, blockIdx.y);
  const Split s(a, held.count);
  const int t0 = a.sink + blockIdx.x * EV_CHUNK;
  if (s.need == 0 || t0 >= s.last) return;
  __shared__ int s_cut[2], s_scan[3][SCAN_WAVES];
  int2* count = work.count + (size_t)blockIdx.y * chunks;
  const Items<EV_LPER> x(a.weights + a.from.row(b, blockIdx.y % G, 0), held, t0, s.last);
  // (at most EV_CHUNKS chunks: one per thread)
  static_assert(EV_CHUNKS <= EV_BLOCK, "a block reads the chunks before its own at once");
  int2 mine = make_int2(0, 0);
  if (PASS == 1 && (int)threadIdx.x < (int)blockIdx.x) mine = count[threadIdx.x];
  int left;
  const uint32_t cut = cut_so_far(work, blockIdx.y, 3, s.need, s_scan[2], s_cut, &left);
  if (PASS == 0) {
    int above, ties;
    (void)waves_before(x.above(cut), s_scan[0], &above);
    (void)waves_before(x.tied(cut), s_scan[1], &ties);
    if (threadIdx.x == 0) count[blockIdx.x] = make_int2(above, ties);
    return;
  }
  int above, ties;
  (void)block_excl_scan(mine.x, s_scan[0], &above);
  (void)block_excl_scan(mine.y, s_scan[1], &ties);
  __syncthreads();  // (the scratch is used again)
  list_staying(x, cut, left, ties, above + min(ties, left), s_scan, kept + (size_t)blockIdx.y * a.keep);
}

// 32 lanes copy a record (512 bytes), its position and its weight.
__global__ __launch_bounds__(EV_COPY) void k_evict_copy(EvictArgs a, const int* kept) {
  const int b = blockIdx.y / G, g = blockIdx.y % G, lane = threadIdx.x & 31;
  const Held held = noted_held(a, blockIdx.y);
  const int count = min(held.count, a.keep);
  const Split s(a, held.count);
  const int* list = kept + (size_t)blockIdx.y * a.keep - a.sink;
  const int end = min(count, (int)(blockIdx.x + 1) * EV_COPY_SLOTS);
  for (int i = blockIdx.x * EV_COPY_SLOTS + (threadIdx.x >> 5); i < end; i += EV_COPY / 32) {
    const int t = held.slot(held.count <= a.keep || i < a.sink ? i
                            : i < a.sink + s.need ? list[i] : held.count - count + i);
    const size_t slot = a.from.row(b, g, t), to_slot = a.to.row(b, g, i);
    size_t from = slot, to = to_slot;
    if (a.from.table) from = a.from.row_in(a.from.page(b, t), g, t);
    // (loaded together before anything is stored)
    const uint4 x = reinterpret_cast<const uint4*>(a.from.records + from * 512)[lane];
    const float w = a.weights[slot];
    const int p = a.to_positions ? a.positions[slot] : 0;
    if (a.to.table) {
      const uint32_t page = a.to.page(b, i);
      if (page >= a.to.n_pages) {  // dropped
        if (lane == 0 && a.to_status) atomicOr(a.to_status, STATUS_PAGE);
        continue;
      }
      to = a.to.row_in(page, g, i);
    }
    if (lane == 0) {
      if (a.to_weights) a.to_weights[to_slot] = w;
      if (a.to_positions) a.to_positions[to_slot] = p;
    }
    reinterpret_cast<uint4*>(a.to.records + to * 512)[lane] = x;
  }
}

// Pages of a sequence, if it has any (of 16 tokens at least).
int most_pages(int capacity) { return (capacity + 15) / 16; }
int chunks_of(int capacity) { return (capacity + EV_CHUNK - 1) / EV_CHUNK; }

}  // namespace

size_t evict_workspace(int batch, int capacity, int keep) {
  const size_t lists = (size_t)batch * G;
  size_t bytes = lists * ((size_t)keep + 1 + most_pages(capacity)) * sizeof(int);
  if (capacity > EV_ONE)  // (fewer middle slots may still take the short path)
    bytes = ((bytes + 15) & ~(size_t)15) +
            lists * (3 * EV_BINS * sizeof(int) + (3 + chunks_of(capacity)) * sizeof(int2));
  return bytes;
}

void launch_evict(EvictArgs a, hipStream_t st) {
  int* kept = static_cast<int*>(a.workspace);
  const int lists = a.from.batch * G;
  a.held = kept + (size_t)lists * a.keep;
  a.before = a.held + lists;
  a.before_stride = most_pages(a.from.capacity);
  const int middle = a.from.capacity - a.sink - a.local;  // at most; a longer list takes the long path
  if (middle <= EV_ONE) {
    // as few slots a thread as hold the list (4 lists, whole calls: 4096 slots 16
    // us, 20 with 16 a thread, 27 with 32, 34 on the long path; 8192: 22, 24, 31,
    // 38; 16384: 44, 50 with 32, 56; 32768: 54, 56 on the long path)
    auto one = middle <= 4 * EV_BLOCK ? k_evict_one<4> : middle <= 8 * EV_BLOCK ? k_evict_one<8>
               : middle <= 16 * EV_BLOCK ? k_evict_one<16> : k_evict_one<32>;
    hipLaunchKernelGGL(one, dim3(lists), dim3(EV_BLOCK), 0, st, a, kept);
  } else {
    const size_t bytes = (size_t)lists * ((size_t)a.keep + 1 + a.before_stride) * sizeof(int);
    LongWork work;
    work.hist = reinterpret_cast<int*>(static_cast<char*>(a.workspace) + ((bytes + 15) & ~(size_t)15));
    work.found = reinterpret_cast<int2*>(work.hist + (size_t)lists * 3 * EV_BINS);
    work.count = work.found + (size_t)lists * 3;
    const int words = lists * 3 * EV_BINS, finders = a.from.table ? lists : 0;
    const dim3 grid(chunks_of(a.from.capacity), lists);
    hipLaunchKernelGGL(k_evict_clear, dim3(finders + (words + EV_BLOCK - 1) / EV_BLOCK), dim3(EV_BLOCK), 0, st, a,
                       work.hist, words, finders);
    for (int d = 0; d < 3; ++d) hipLaunchKernelGGL(k_evict_digit, grid, dim3(EV_BLOCK), 0, st, a, work, d);
    hipLaunchKernelGGL(k_evict_list<0>, grid, dim3(EV_BLOCK), 0, st, a, work, kept);
    hipLaunchKernelGGL(k_evict_list<1>, grid, dim3(EV_BLOCK), 0, st, a, work, kept);
  }
  hipLaunchKernelGGL(k_evict_copy, dim3((a.keep + EV_COPY_SLOTS - 1) / EV_COPY_SLOTS, lists), dim3(EV_COPY),
                     0, st, a, (const int*)kept);
}

}  // namespace skv
