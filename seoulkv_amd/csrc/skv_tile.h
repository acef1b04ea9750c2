// What the attention kernels over a whole cache of FP8 [V || K] records share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace skv {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float DN_LOG2E = 1.4426950408889634f;

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// V is read with streaming loads: a row's 256 bytes are used by one
// instruction, once.  (K rows come in 64-byte runs, two instructions per
// cache line, and lose more than they gain: T = 2^20 347 us with neither
// streamed, 330 K, 311 V, 324 both; T = 131072 49.9, 53.1, 48.1, 53.0.)
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}

}  // namespace skv
