// The record cache's operators: kernel arguments and launches.  Every size
// here has been checked by the C entry points (skv_cache.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace skv {

constexpr int CACHE_MAX_BATCH = 1024;
constexpr int CACHE_MAX_SLOTS = 1 << 20;
constexpr int TREE_MAX_DRAFTS = 64;  // one bit of a mask word each
constexpr int STATUS_CAPACITY = 1, STATUS_PAGE = 2;

// The records of a cache and how many of them are committed.
struct CacheView {
  uint8_t* records;
  const int* table;  // paged: [batch][table_len], else NULL
  const int* lengths;
  uint32_t n_pages;
  int table_len, shift;  // paged: entries per sequence, log2 tokens per page
  int batch, capacity;

  __host__ __device__ int length(int b) const {
    const int n = lengths[b];
    return n < 0 ? 0 : n > capacity ? capacity : n;
  }
  // Index of the record of slot t of (sequence b, KV head g); contiguous.
  __host__ __device__ size_t row(int b, int g, int t) const {
    return ((size_t)b * 4 + g) * capacity + t;
  }
  // Paged: index of the record of slot t in page `page` of its sequence.
  __host__ __device__ size_t row_in(uint32_t page, int g, int t) const {
    return ((((size_t)page * 4) + g) << shift) + ((uint32_t)t & ((1u << shift) - 1u));
  }
  __host__ __device__ uint32_t page(int b, int t) const {
    return (uint32_t)table[(size_t)b * table_len + (t >> shift)];
  }
};

// BF16 (or other) rows with element strides.
struct Rows {
  const void* data;
  int64_t sb, st, sh;
};

struct RotaryArgs {
  const uint64_t* turns;
  int pairs;
  float scale;
  const void* positions;
  int64_t position_sb;
  int positions64;
};

// y = x turned; dtype as SKV_BF16 / SKV_FP16 / SKV_FP32.
void launch_rotary(const RotaryArgs& a, bool interleaved, bool transpose, const Rows& x,
                   const Rows& y, int dtype, int batch, int n, int heads, int dim, hipStream_t st);

struct WriteArgs {
  CacheView c;
  RotaryArgs r;  // pairs = 0: no turn
  int interleaved;
  Rows k, v, q, q_out;  // q.data NULL: none
  int n;
  const int* counts;
  int* positions;  // the cache's
  float* weights;
  int* status;
};
void launch_cache_write(const WriteArgs& a, hipStream_t st);

struct TreeArgs {
  CacheView c;
  Rows q;
  int n;
  const int64_t* tree;
  const int* counts;
  float cap;
  float* part;  // workspace
  uint16_t* out;
  float* lse;
};
size_t tree_workspace(int batch, int n);
void launch_tree(const TreeArgs& a, hipStream_t st);

struct WeightArgs {
  CacheView c;
  Rows q;
  int n;
  const int64_t* tree;
  const int* counts;
  float cap;
  const float* lse;
  float* weights;
  int accumulate;
};
void launch_key_weights(const WeightArgs& a, hipStream_t st);

struct EvictArgs {
  CacheView from, to;
  const int* positions;
  const float* weights;
  int* to_positions;  // NULL: not copied
  float* to_weights;
  int* to_lengths;
  int* to_status;  // NULL: not noted
  int keep, sink, local;
  void* workspace;
  // in the workspace, set by launch_evict: per list the slots that have a page,
  // and those before each page
  int *held, *before;
  int before_stride;
};
size_t evict_workspace(int batch, int capacity, int keep);
void launch_evict(EvictArgs a, hipStream_t st);

}  // namespace skv
