// Eviction by accumulated attention weight (interface in skv_cache.h).
//
// k_evict_select, one block per (sequence, KV head): the weight of the last
// slot that stays, by a radix search over the order-preserving 32-bit image of
// the weights (8 bits a pass), then the list of slots that stay, in order.
// k_evict_copy moves their records, 32 lanes a record.
#include "skv_cache.h"
#include "skv_device.h"

namespace skv {

namespace {

constexpr int EV_BLOCK = 1024;
constexpr int EV_COPY = 256;  // threads of a copy block: 8 records at a time
constexpr int EV_PER_BLOCK = 32;

// Larger weight, larger value; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t weight_order(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return w != w ? 0u : o;
}

// What stays of a sequence of `len` slots: all of them, or the first sink, the
// last local and `need` of [sink, last).
struct Split {
  int last, need;
  bool all;
  __device__ Split(const EvictArgs& a, int len) {
    all = len <= a.keep;
    last = len - a.local;
    need = a.keep - a.sink - a.local;
  }
};

__global__ __launch_bounds__(EV_BLOCK) void k_evict_select(EvictArgs a, int* kept) {
  const int b = blockIdx.x / G;
  const int len = a.from.length(b);
  const Split s(a, len);
  int* list = kept + (size_t)blockIdx.x * a.keep;
  if (blockIdx.x % G == 0 && threadIdx.x == 0) a.to_lengths[b] = s.all ? len : a.keep;
  if (s.all) {
    for (int t = threadIdx.x; t < len; t += EV_BLOCK) list[t] = t;
    return;
  }
  const float* w = a.weights + a.from.row(b, blockIdx.x % G, 0);
  __shared__ int s_hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_scan[SCAN_WAVES];
  uint32_t prefix = 0;  // the digits found so far; bits below `shift` are open
  int left = s.need;    // items to take among those with this prefix
  for (int shift = 24; shift >= 0 && s.need > 0; shift -= 8) {
    if (threadIdx.x < 256) s_hist[threadIdx.x] = 0;
    __syncthreads();
    for (int t = a.sink + threadIdx.x; t < s.last; t += EV_BLOCK) {
      const uint32_t o = weight_order(w[t]);
      if (shift == 24 || (o >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(o >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int d = 255, above = 0;
      while (d > 0 && above + s_hist[d] < left) above += s_hist[d--];
      s_prefix = prefix | (uint32_t)d << shift;
      s_left = left - above;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
  }
  // slots in order: those above the last weight, and the first `left` at it
  int out = 0, tied = 0;
  for (int t0 = 0; t0 < len; t0 += EV_BLOCK) {
    const int t = t0 + threadIdx.x;
    int fixed = 0, tie = 0;
    if (t < len) {
      fixed = t < a.sink || t >= s.last;
      if (!fixed && s.need > 0) {
        const uint32_t o = weight_order(w[t]);
        fixed = o > prefix;
        tie = o == prefix;
      }
    }
    int ties, count;
    const int rank = block_excl_scan(tie, s_scan, &ties) + tied;
    __syncthreads();
    const int stays = fixed || (tie && rank < left);
    const int at = block_excl_scan(stays, s_scan, &count) + out;
    if (stays && at < a.keep) list[at] = t;
    out += count;
    tied += ties;
    __syncthreads();
  }
}

// 32 lanes copy a record (512 bytes), its position and its weight.
__global__ __launch_bounds__(EV_COPY) void k_evict_copy(EvictArgs a, const int* kept) {
  const int b = blockIdx.y / G, g = blockIdx.y % G, lane = threadIdx.x & 31;
  const int len = a.from.length(b), count = min(len, a.keep);
  const int* list = kept + (size_t)blockIdx.y * a.keep;
  const int end = min(count, (int)(blockIdx.x + 1) * EV_PER_BLOCK);
  for (int i = blockIdx.x * EV_PER_BLOCK + (threadIdx.x >> 5); i < end; i += EV_COPY / 32) {
    const int t = list[i];
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

}  // namespace

size_t evict_workspace(int batch, int capacity, int keep) {
  return (size_t)batch * G * (size_t)keep * sizeof(int);
}

void launch_evict(const EvictArgs& a, hipStream_t st) {
  int* kept = static_cast<int*>(a.workspace);
  const int lists = a.from.batch * G;
  hipLaunchKernelGGL(k_evict_select, dim3(lists), dim3(EV_BLOCK), 0, st, a, kept);
  hipLaunchKernelGGL(k_evict_copy, dim3((a.keep + EV_PER_BLOCK - 1) / EV_PER_BLOCK, lists), dim3(EV_COPY),
                     0, st, a, (const int*)kept);
}

}  // namespace skv
