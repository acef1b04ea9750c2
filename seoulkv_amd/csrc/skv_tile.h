// Tiles of 16 FP8 [V || K] records on the matrix cores: what the attention
// kernels over a whole cache share.  The score step takes a record's K half as
// stored (16 x 16 x 128 FP8 products, two per row), in the order of dn_dim.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace skv {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));

constexpr float DN_LOG2E = 1.4426950408889634f;

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

__device__ __forceinline__ uint32_t f32_fp8_byte(float x) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false) & 0xffu;
}
__device__ __forceinline__ float fp8_byte_f32(uint32_t b) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f f = __builtin_amdgcn_cvt_pk_f32_fp8((int)b, false);
  return f[0];
}

// The four dims of word i of score step m for key block kb: the order in
// which lane 16 kb + row holds a record's K bytes 64 j + 16 kb + [0, 16).
__device__ __forceinline__ int dn_dim(int m, int i, int kb) {
  return m * 128 + (i >> 2) * 64 + kb * 16 + (i & 3) * 4;
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

__device__ __forceinline__ v8i as_v8i(uint4 a, uint4 b) {
  return v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

}  // namespace skv
