// Eviction by accumulated attention weight (interface in skv_cache.h).
//
// Which slots stay: the weights are ordered by a 32-bit image, and the value
// at the cut is found digit by digit (11, 11 and 10 bits) from histograms; of
// the slots at that value the lowest ones stay.  Up to EV_ONE middle slots are
// one block's work per (sequence, KV head), the weights read once and held in
// registers: 16000 slots in 13.8 us, against 61 with a pass over memory per 8
// bits and one thread walking the bins, and 26 spread over blocks.  Longer
// lists are spread over blocks of EV_CHUNK slots: a launch per digit, one for
// the counts of every chunk, one for the list; 131072 slots in 24 us (1.8 to
// clear, 3 x 4.3, 4.3, 5.6), against 250 by one block.  These launches are
// bound by their latency (a chain of load, scan, atomic), not by their bytes.
//
// The list holds the middle slots that stay, in order; what lies before and
// behind them is sink and local.  k_evict_copy moves the records, 32 lanes a
// record: 4 x 4 x 8192 records in 31 us, 4.4 TB/s read and written.
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

// What stays of a sequence of `len` slots: all of them (need 0), or the first
// sink, the last local and `need` of [sink, last).
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

// A wave holds 64 N consecutive slots, lane l the slots t + 64 i + l (loads of
// whole lines; a thread with N consecutive slots read every line N times).
template <int N>
struct Items {
  uint32_t o[N];
  int t, last;  // lane 0's first slot; slots from `last` on are none

  __device__ Items(const float* w, int begin, int last) : last(last) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    t = begin + wave * WAVE * N;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = weight_order(on(i) ? w[slot(i)] : 0.f);
  }
  __device__ __forceinline__ int slot(int i) const { return t + WAVE * i + (int)(threadIdx.x & 63); }
  __device__ __forceinline__ bool on(int i) const { return slot(i) < last; }
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

// Writes the slots that stay, those above the cut and the first `left` at it,
// from list[at] on (`ties`: items at the cut in slots before this block's).
template <int N>
__device__ __forceinline__ void list_staying(const Items<N>& x, uint32_t cut, int left, int ties, int at,
                                             int (*scan)[SCAN_WAVES], int* list) {
  int total;
  int rank = ties + waves_before(x.tied(cut), scan[0], &total);
  uint64_t stay[N];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool tie = x.on(i) && x.o[i] == cut;
    const uint64_t tied = __ballot(tie);
    stay[i] = __ballot((x.on(i) && x.o[i] > cut) || (tie && rank + lanes_below(tied) < left));
    rank += __popcll(tied);
    mine += __popcll(stay[i]);
  }
  at += waves_before(mine, scan[1], &total);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((stay[i] >> (threadIdx.x & 63)) & 1) list[at + lanes_below(stay[i])] = x.slot(i);
    at += __popcll(stay[i]);
  }
}

// A whole list by one block, PER slots a thread; sets to_lengths.
template <int PER>
__global__ __launch_bounds__(EV_BLOCK) void k_evict_one(EvictArgs a, int* kept) {
  const int b = blockIdx.x / G;
  const int len = a.from.length(b);
  const Split s(a, len);
  if (blockIdx.x % G == 0 && threadIdx.x == 0) a.to_lengths[b] = min(len, a.keep);
  if (s.need == 0) return;
  const float* w = a.weights + a.from.row(b, blockIdx.x % G, 0);
  __shared__ int s_hist[EV_BINS], s_cut[2], s_scan[3][SCAN_WAVES];
  const Items<PER> x(w, a.sink, s.last);
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

__global__ __launch_bounds__(256) void k_evict_clear(int* hist, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
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
  const int len = a.from.length(b);
  const Split s(a, len);
  if (d == 0 && blockIdx.x == 0 && blockIdx.y % G == 0 && threadIdx.x == 0) a.to_lengths[b] = min(len, a.keep);
  const int t0 = a.sink + blockIdx.x * EV_CHUNK;
  if (s.need == 0 || t0 >= s.last) return;
  __shared__ int s_hist[EV_BINS], s_cut[2], s_scan[SCAN_WAVES];
  int* hist = work.hist + ((size_t)blockIdx.y * 3 + d) * EV_BINS;
  const Items<EV_LPER> x(a.weights + a.from.row(b, blockIdx.y % G, 0), t0, s.last);
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
  const Split s(a, a.from.length(b));
  const int t0 = a.sink + blockIdx.x * EV_CHUNK;
  if (s.need == 0 || t0 >= s.last) return;
  __shared__ int s_cut[2], s_scan[3][SCAN_WAVES];
  int2* count = work.count + (size_t)blockIdx.y * chunks;
  const Items<EV_LPER> x(a.weights + a.from.row(b, blockIdx.y % G, 0), t0, s.last);
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
  const int len = a.from.length(b), count = min(len, a.keep);
  const Split s(a, len);
  const int* list = kept + (size_t)blockIdx.y * a.keep - a.sink;
  const int end = min(count, (int)(blockIdx.x + 1) * EV_COPY_SLOTS);
  for (int i = blockIdx.x * EV_COPY_SLOTS + (threadIdx.x >> 5); i < end; i += EV_COPY / 32) {
    const int t = len <= a.keep || i < a.sink ? i : i < a.sink + s.need ? list[i] : len - count + i;
    size_t from = a.from.row(b, g, t), to = a.to.row(b, g, i);
    if (lane == 0) {
      if (a.to_weights) a.to_weights[to] = a.weights[from];
      if (a.to_positions) a.to_positions[to] = a.positions[from];
    }
    uint4 x = make_uint4(0, 0, 0, 0);
    bool held = true;
    if (a.from.table) {
      const uint32_t page = a.from.page(b, t);
      held = page < a.from.n_pages;
      from = a.from.row_in(page, g, t);
    }
    if (held) x = reinterpret_cast<const uint4*>(a.from.records + from * 512)[lane];
    if (a.to.table) {
      const uint32_t page = a.to.page(b, i);
      if (page >= a.to.n_pages) continue;
      to = a.to.row_in(page, g, i);
    }
    reinterpret_cast<uint4*>(a.to.records + to * 512)[lane] = x;
  }
}

int chunks_of(int capacity) { return (capacity + EV_CHUNK - 1) / EV_CHUNK; }

}  // namespace

size_t evict_workspace(int batch, int capacity, int keep) {
  const size_t lists = (size_t)batch * G;
  size_t bytes = lists * (size_t)keep * sizeof(int);
  if (capacity > EV_ONE)  // (fewer middle slots may still take the short path)
    bytes = ((bytes + 15) & ~(size_t)15) +
            lists * (3 * EV_BINS * sizeof(int) + (3 + chunks_of(capacity)) * sizeof(int2));
  return bytes;
}

void launch_evict(const EvictArgs& a, hipStream_t st) {
  int* kept = static_cast<int*>(a.workspace);
  const int lists = a.from.batch * G;
  const int middle = a.from.capacity - a.sink - a.local;  // at most; a longer list takes the long path
  if (middle <= EV_ONE) {
    auto one = middle <= 4 * EV_BLOCK ? k_evict_one<4> : middle <= 8 * EV_BLOCK ? k_evict_one<8>
               : middle <= 16 * EV_BLOCK ? k_evict_one<16> : k_evict_one<32>;
    hipLaunchKernelGGL(one, dim3(lists), dim3(EV_BLOCK), 0, st, a, kept);
  } else {
    const size_t bytes = (size_t)lists * a.keep * sizeof(int);
    LongWork work;
    work.hist = reinterpret_cast<int*>(static_cast<char*>(a.workspace) + ((bytes + 15) & ~(size_t)15));
    work.found = reinterpret_cast<int2*>(work.hist + (size_t)lists * 3 * EV_BINS);
    work.count = work.found + (size_t)lists * 3;
    const int words = lists * 3 * EV_BINS;
    const dim3 grid(chunks_of(a.from.capacity), lists);
    hipLaunchKernelGGL(k_evict_clear, dim3((words + 255) / 256), dim3(256), 0, st, work.hist, words);
    for (int d = 0; d < 3; ++d) hipLaunchKernelGGL(k_evict_digit, grid, dim3(EV_BLOCK), 0, st, a, work, d);
    hipLaunchKernelGGL(k_evict_list<0>, grid, dim3(EV_BLOCK), 0, st, a, work, kept);
    hipLaunchKernelGGL(k_evict_list<1>, grid, dim3(EV_BLOCK), 0, st, a, work, kept);
  }
  hipLaunchKernelGGL(k_evict_copy, dim3((a.keep + EV_COPY_SLOTS - 1) / EV_COPY_SLOTS, lists), dim3(EV_COPY),
                     0, st, a, (const int*)kept);
}

}  // namespace skv
