// Heads divided by their root mean square, weighted and turned to their
// positions, alone, backwards, and on the way into a record cache; and the
// record cache's writes in 4 bits.
//
//   y = R(p) (w x r),  r = 1 / sqrt(mean(x^2) + eps)
//   h = R(p)^T g,  u = w h:  dx = r u - x r^3 mean(u x),  dw = sum over rows of h x r
//
// A token is a team of L lanes of one wave; each lane holds PER units of a head
// (8 pairs, or one element an access where the width is no multiple of 16), so
// the mean is a sum in the lane and log2 L steps across lanes, and a row is
// read once.  The lane keeps its sines and cosines while the team walks the
// heads, BATCH of them in flight as they lie in memory.  All arithmetic is FP32,
// rounded once.
//
// Bound by memory: 32768 tokens x 20 heads x 256 in BF16 132 us, 5.1 TB/s, a copy's
// rate (180 where the heads in flight were widened and each BF16 rounded by
// integer instructions); 5003 x 7 x 96 in FP32 12 us, the chain load -> sum ->
// store of few blocks; the gradient of 8192 x 20 x 256 53 us, 4.8 TB/s, 5 of them
// the sum of the blocks' shares of dw (113 with 2048 shares, summed one load at
// a time); 32768 tokens into a cache with their queries 166, 4.4 TB/s, into records of
// 4 bits 170, 4.2; a token of 8 sequences 7 us, two dependent loads and the launch.
#include <type_traits>

#include "skv_rows.h"
#include "skv_tile.h"

namespace skv {

namespace {

// Sum over the L lanes of a team, in every one of them.
template <int L>
__device__ __forceinline__ float team_sum(float v) {
  if (L > 1) v += dpp_f<0xB1>(v);   // quad_perm [1,0,3,2]
  if (L > 2) v += dpp_f<0x4E>(v);   // quad_perm [2,3,0,1]
  if (L > 4) v += dpp_f<0x141>(v);  // row_half_mirror
  if (L > 8) v += dpp_f<0x140>(v);  // row_mirror
  if (L > 16) v += __shfl_xor(v, 16);
  if (L > 32) v += __shfl_xor(v, 32);
  return v;
}

// N elements of a row as they lie in memory: widened where they are used, so what
// is in flight takes half the registers.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Piece {
  T v[N];
  __device__ __forceinline__ float operator[](int i) const { return load1(&v[i]); }
};
template <typename T, int N>
__device__ __forceinline__ Piece<T, N> piece_at(const T* p) { return *reinterpret_cast<const Piece<T, N>*>(p); }

// Two values as BF16, rounded by the converter (to nearest even; NaN stays NaN).
__device__ __forceinline__ uint32_t bf16x2_rne(float a, float b) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2bf));
}
template <int N, typename T>
__device__ __forceinline__ void put(T* p, const float f[N]) { storen<N>(p, f); }
template <>
__device__ __forceinline__ void put<8, BF16>(BF16* p, const float f[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16x2_rne(f[0], f[1]), bf16x2_rne(f[2], f[3]), bf16x2_rne(f[4], f[5]),
                                            bf16x2_rne(f[6], f[7]));
}

// A lane's elements of a head: PER units, `a` at their lo and `b` at their hi
// (0 where a unit is not there or has no pairs).
template <int N, int L, int PER>
struct Lane {
  int lo[PER], hi[PER], pair[PER];
  bool there[PER], turned[PER], inter;
  float2 cs[PER][N];

  template <typename T>
  struct Raw {
    Piece<T, N> a[PER], b[PER];
  };

  __device__ __forceinline__ Lane(int lane, int units, int pairs, bool interleaved) : inter(interleaved) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int u = lane + L * p;
      there[p] = u < units;
      const Unit<N, false> half(there[p] ? u : 0, pairs);
      turned[p] = there[p] && half.turned;
      pair[p] = half.pair;
      lo[p] = half.turned && inter ? 2 * half.pair : half.lo;
      hi[p] = inter ? lo[p] + N : half.hi;
    }
  }
  __device__ __forceinline__ void angles(const RotaryArgs& r, int64_t position, float sign) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (turned[p]) unit_turns<N>(r, pair[p], position, sign, cs[p]);
  }
  // (where nothing is there element 0 is read, and not used)
  template <typename T>
  __device__ __forceinline__ void load(const T* row, Raw<T>& x) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      x.a[p] = piece_at<T, N>(row + lo[p]);
      x.b[p] = piece_at<T, N>(row + (turned[p] ? hi[p] : lo[p]));
    }
  }
  template <typename T>
  __device__ __forceinline__ void widen(const Raw<T>& x, float (&a)[PER][N], float (&b)[PER][N]) const {
#pragma unroll
    for (int p = 0; p < PER; ++p)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[p][i] = there[p] ? x.a[p][i] : 0.f;
        b[p][i] = turned[p] ? x.b[p][i] : 0.f;
      }
  }
  template <typename T>
  __device__ __forceinline__ void weights(const NormArgs& w, int head, float (&a)[PER][N], float (&b)[PER][N]) const {
    const int64_t at = head * w.sh;
    if (w.wide) {
      Raw<float> x;
      load(static_cast<const float*>(w.weight) + at, x);
      widen(x, a, b);
    } else {
      Raw<T> x;
      load(static_cast<const T*>(w.weight) + at, x);
      widen(x, a, b);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&a)[PER][N], const float (&b)[PER][N]) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      if (there[p]) put<N>(row + lo[p], a[p]);
      if (turned[p]) put<N>(row + hi[p], b[p]);
    }
  }
  __device__ __forceinline__ void turn(float (&a)[PER][N], float (&b)[PER][N]) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      if (!turned[p]) continue;
      if (inter) turn_unit<N, true>(a[p], b[p], cs[p]);
      else turn_unit<N, false>(a[p], b[p], cs[p]);
    }
  }
  // Sum of x y over the head.
  __device__ __forceinline__ static float dot(const float (&xa)[PER][N], const float (&xb)[PER][N],
                                              const float (&ya)[PER][N], const float (&yb)[PER][N]) {
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < PER; ++p)
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(xa[p][i], ya[p][i], fmaf(xb[p][i], yb[p][i], s));
    return team_sum<L>(s);
  }
  // 1 / root mean square, off by an ulp.
  __device__ __forceinline__ static float inverse_rms(const float (&a)[PER][N], const float (&b)[PER][N],
                                                      float inv_dim, float eps) {
    return __builtin_amdgcn_rsqf(fmaf(dot(a, b, a, b), inv_dim, eps));
  }
  // The normed and turned head; the weight's type decides how it is widened.
  template <typename W>
  __device__ __forceinline__ void norm(float (&a)[PER][N], float (&b)[PER][N], const Raw<W>& w, float inv_dim,
                                       float eps) const {
    const float rms = inverse_rms(a, b, inv_dim, eps);
#pragma unroll
    for (int p = 0; p < PER; ++p)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a[p][e] = a[p][e] * rms * w.a[p][e];
        b[p][e] = b[p][e] * rms * w.b[p][e];
      }
    turn(a, b);
  }
};

// Heads in flight.
template <int N, int PER>
constexpr int batch_of = 2 * N * PER <= 16 ? 4 : 2;

template <typename T, typename W, int N, int L, int PER>
__global__ __launch_bounds__(RO_BLOCK) void k_norm_rotary(RotaryArgs r, NormArgs w, Rows x, Rows y, int64_t tokens,
                                                          int units, int n, int heads, int dim, int per, int inter) {
  constexpr int BATCH = batch_of<N, PER>;
  typedef Lane<N, L, PER> Team;
  const int64_t token = ((int64_t)blockIdx.x * RO_BLOCK + threadIdx.x) / L;
  if (token >= tokens) return;
  const int b = (int)(token / n), i = (int)(token % n);
  Team lane(threadIdx.x % L, units, r.pairs, inter);
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
  const T* in = static_cast<const T*>(x.data) + b * x.sb + i * x.st;
  T* out = const_cast<T*>(static_cast<const T*>(y.data)) + b * y.sb + i * y.st;
  const W* weight = static_cast<const W*>(w.weight);
  typename Team::template Raw<W> wr[BATCH];
  if (!w.sh) lane.load(weight, wr[0]);
  lane.angles(r, position_of(r, b, i), 1.f);
  const float inv_dim = 1.f / (float)dim;
#pragma nounroll
  for (int h = h0; h < h1; h += BATCH) {
    typename Team::template Raw<T> raw[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) lane.load(in + min(h + j, h1 - 1) * x.sh, raw[j]);
    if (w.sh) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) lane.load(weight + min(h + j, h1 - 1) * w.sh, wr[j]);
    } else {
#pragma unroll
      for (int j = 1; j < BATCH; ++j) wr[j] = wr[0];
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (h + j >= h1) break;
      float a[PER][N], b[PER][N];
      lane.widen(raw[j], a, b);
      lane.norm(a, b, wr[j], inv_dim, w.eps);
      lane.store(out + (h + j) * y.sh, a, b);
    }
  }
}

// A team walks every gridDim.x-th group of tokens, and of each the heads of its
// blockIdx.y, so its share of dw stays in registers; the block's share is summed
// in LDS in a fixed order and written as FP32.  EACH (a weight for each head):
// one head, the next token's in flight.
template <typename T, int N, int L, int PER, bool EACH>
__global__ __launch_bounds__(RO_BLOCK) void k_norm_grad(RotaryArgs r, NormArgs w, Rows g, Rows x, Rows y,
                                                        int64_t tokens, int units, int n, int heads, int dim,
                                                        int per, int inter, float* partial) {
  constexpr int BATCH = EACH ? 1 : batch_of<N, PER>, TEAMS = RO_BLOCK / L, VALUES = 2 * N * PER;
  __shared__ float s_dw[VALUES][RO_BLOCK + 1];
  const int team = threadIdx.x / L;
  const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
  Lane<N, L, PER> lane(threadIdx.x % L, units, r.pairs, inter);
  float wa[PER][N], wb[PER][N], da[PER][N], db[PER][N];
  lane.template weights<T>(w, h0, wa, wb);
#pragma unroll
  for (int p = 0; p < PER; ++p)
#pragma unroll
    for (int e = 0; e < N; ++e) da[p][e] = db[p][e] = 0.f;
  const float inv_dim = 1.f / (float)dim;
  typename Lane<N, L, PER>::template Raw<T> graw[BATCH], xraw[BATCH];
  auto fetch = [&](int64_t token, int h, int j) {
    const int64_t b = token / n, i = token % n;
    lane.load(static_cast<const T*>(g.data) + b * g.sb + i * g.st + h * g.sh, graw[j]);
    lane.load(static_cast<const T*>(x.data) + b * x.sb + i * x.st + h * x.sh, xraw[j]);
  };
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  int64_t token = (int64_t)blockIdx.x * TEAMS + team;
  if (EACH && token < tokens) fetch(token, h0, 0);
  for (; token < tokens; token += step) {
    const int b = (int)(token / n), i = (int)(token % n);
    lane.angles(r, position_of(r, b, i), -1.f);
    T* out = const_cast<T*>(static_cast<const T*>(y.data)) + b * y.sb + i * y.st;
#pragma nounroll
    for (int h = h0; h < h1; h += BATCH) {
      if constexpr (!EACH) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) fetch(token, min(h + j, h1 - 1), j);
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        if (h + j >= h1) break;
        float xa[PER][N], xb[PER][N], ga[PER][N], gb[PER][N];
        lane.widen(graw[j], ga, gb);
        lane.widen(xraw[j], xa, xb);
        if (EACH && token + step < tokens) fetch(token + step, h0, 0);
        lane.turn(ga, gb);
        const float rms = lane.inverse_rms(xa, xb, inv_dim, w.eps);
#pragma unroll
        for (int p = 0; p < PER; ++p)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            // (x becomes x r, g becomes u)
            xa[p][e] *= rms;
            xb[p][e] *= rms;
            da[p][e] = fmaf(ga[p][e], xa[p][e], da[p][e]);
            db[p][e] = fmaf(gb[p][e], xb[p][e], db[p][e]);
            ga[p][e] *= wa[p][e];
            gb[p][e] *= wb[p][e];
          }
        const float mean = lane.dot(ga, gb, xa, xb) * inv_dim;
#pragma unroll
        for (int p = 0; p < PER; ++p)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            ga[p][e] = rms * fmaf(-mean, xa[p][e], ga[p][e]);
            gb[p][e] = rms * fmaf(-mean, xb[p][e], gb[p][e]);
          }
        lane.store(out + (h + j) * y.sh, ga, gb);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < PER; ++p)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      s_dw[(2 * p) * N + e][threadIdx.x] = da[p][e];
      s_dw[(2 * p + 1) * N + e][threadIdx.x] = db[p][e];
    }
  __syncthreads();
  float* row = partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * dim;
  for (int at = threadIdx.x; at < VALUES * L; at += RO_BLOCK) {
    const int value = at / L, l = at % L, p = value / (2 * N), e = value % N;
    const Lane<N, L, PER> owner(l, units, r.pairs, inter);
    const bool high = value / N & 1;
    float s = 0.f;
    for (int t = 0; t < TEAMS; ++t) s += s_dw[value][t * L + l];
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (q != p) continue;
      if (high ? owner.turned[q] : owner.there[q]) row[(high ? owner.hi[q] : owner.lo[q]) + e] = s;
    }
  }
}

// dw row blockIdx.y: the sum of `shares` partial rows, 16 slices of them in turn
// for 64 columns, the slices added in order.
__global__ __launch_bounds__(1024) void k_norm_weight(const float* partial, int shares, int dim, void* dw, int dtype) {
  __shared__ float s_sum[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
  const float* in = partial + (int64_t)blockIdx.y * shares * dim;
  float s = 0.f;
  if (col < dim) {
    int i = slice;
    for (; i + 7 * 16 < shares; i += 8 * 16) {  // 8 loads in flight
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = in[(int64_t)(i + 16 * j) * dim + col];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < shares; i += 16) s += in[(int64_t)i * dim + col];
  }
  s_sum[slice][threadIdx.x & 63] = s;
  __syncthreads();
  if (slice || col >= dim) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += s_sum[i][threadIdx.x];
  const int64_t at = (int64_t)blockIdx.y * dim + col;
  if (dtype == 0) store1(static_cast<BF16*>(dw) + at, s);
  else if (dtype == 1) store1(static_cast<FP16*>(dw) + at, s);
  else store1(static_cast<float*>(dw) + at, s);
}

// ------------------------------------------------------------ record writes
// 8 elements of a block of 32, which four neighbouring lanes hold: the block's
// scale is the smallest power of two that brings it to at most 6, 2^-20 at
// least; a block that holds NaN or more than 6 x 2^13 has none (FOUR_NAN).
__device__ __forceinline__ void pack4(const float f[8], uint32_t& codes, uint32_t& scale) {
  uint32_t most = 0;  // bits of the largest size; those of NaN are above all others
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7fffffffu);
  most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xB1, 0xf, 0xf, false));
  most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x4E, 0xf, 0xf, false));
  // 6 x 2^e is 1.5 x 2^(e + 2)
  const int e = (int)(most >> 23) - 2 + ((most & 0x7fffffu) > 0x400000u);
  scale = e > FOUR_MAX ? FOUR_NAN : max(e, FOUR_MIN);
  const float unit = __uint_as_float((uint32_t)(e > FOUR_MAX ? 127 : max(e, FOUR_MIN)) << 23);
  codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], unit, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], unit, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], unit, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], unit, 3);
}

// Elements 8 chunk .. +7 of a record's V (side 0) or K (side 1).
__device__ __forceinline__ void store4(uint8_t* record, int side, int chunk, const float f[8]) {
  uint32_t codes, scale;
  pack4(f, codes, scale);
  reinterpret_cast<uint32_t*>(record + 128 * side)[chunk] = codes;
  if (chunk % 4 == 0) record[256 + 8 * side + chunk / 4] = (uint8_t)scale;
}

// The groups of 4 rows of a token: query heads, K heads, V heads.
constexpr int WG_K = H, WG_V = H + 1, WG_ALL = H + 2;

// Teams as above; group first + blockIdx.y per .. of the token's rows.  Without
// a norm (weight NULL) rows are only turned.  With FOUR a turned K row goes
// through LDS, since the lanes' pairs do not lie in blocks of 32.
template <int N, int L, int PER, bool FOUR>
__global__ __launch_bounds__(RO_BLOCK) void k_cache_write_normed(WriteArgs a, NormArgs qw, NormArgs kw, int64_t tokens,
                                                                 int units, int first, int per) {
  constexpr int TEAMS = RO_BLOCK / L, BATCH = batch_of<N, PER>;
  __shared__ float4 s_row[FOUR ? TEAMS : 1][D / 4];
  const int64_t token = ((int64_t)blockIdx.x * RO_BLOCK + threadIdx.x) / L;
  if (token >= tokens) return;
  const int b = (int)(token / a.n), i = (int)(token % a.n), id = threadIdx.x % L;
  Lane<N, L, PER> lane(id, units, a.r.pairs, a.interleaved);
  const int slot = a.c.length(b) + i;
  const bool wanted = !a.counts || i < a.counts[b];
  const bool fits = wanted && slot < a.c.capacity;
  uint32_t page = 0;
  bool held = fits;
  if (fits && a.c.table) {
    page = a.c.page(b, slot);
    held = page < a.c.n_pages;
  }
  const int64_t p = a.r.positions ? position_of(a.r, b, i) : slot;
  lane.angles(a.r, p, 1.f);
  auto source = [&](const Rows& r, int h) {
    return static_cast<const BF16*>(r.data) + b * r.sb + i * r.st + h * r.sh;
  };
  auto record = [&](int g) {
    return a.c.records + (a.c.table ? a.c.row_in(page, g, slot) : a.c.row(b, g, slot)) * (FOUR ? 272 : 512);
  };
  const int g1 = min(first + (int)(blockIdx.y + 1) * per, WG_ALL);
#pragma nounroll
  for (int group = first + blockIdx.y * per; group < g1; ++group) {
    if (group == WG_V) {
      if (!held) continue;
#pragma unroll
      for (int h = 0; h < G; ++h) {
        const BF16* in = source(a.v, h);
        uint8_t* out = record(h);
#pragma unroll
        for (int chunk = id; chunk < D / 8; chunk += L) {
          float f[8];
          if constexpr (N == 8) load8(in + 8 * chunk, f);
          else
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = load1(in + 8 * chunk + e);
          if constexpr (FOUR) store4(out, 0, chunk, f);
          else store_fp8<8>(out + 8 * chunk, f);
        }
      }
      continue;
    }
    const bool keys = group == WG_K;
    if (keys && !held) continue;
    const Rows& rows = keys ? a.k : a.q;
    const NormArgs& w = keys ? kw : qw;
    const int h0 = keys ? 0 : group * H;
    float wa[PER][N], wb[PER][N];
    if (w.weight) lane.template weights<BF16>(w, h0, wa, wb);
#pragma unroll
    for (int hb = 0; hb < H; hb += BATCH) {
      typename Lane<N, L, PER>::template Raw<BF16> raw[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) lane.load(source(rows, h0 + hb + j), raw[j]);
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int h = h0 + hb + j;
        float xa[PER][N], xb[PER][N];
        lane.widen(raw[j], xa, xb);
        if (w.weight) {
          if (w.sh && h > h0) lane.template weights<BF16>(w, h, wa, wb);
          const float rms = lane.inverse_rms(xa, xb, 1.f / D, w.eps);
#pragma unroll
          for (int u = 0; u < PER; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              xa[u][e] = xa[u][e] * rms * wa[u][e];
              xb[u][e] = xb[u][e] * rms * wb[u][e];
            }
        }
        lane.turn(xa, xb);
        if (!keys) {
          lane.store(const_cast<BF16*>(source(a.q_out, h)), xa, xb);
        } else if constexpr (FOUR) {
          float* row = reinterpret_cast<float*>(s_row[threadIdx.x / L]);
          lane.store(row, xa, xb);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int chunk = id; chunk < D / 8; chunk += L) {
            float f[8];
            load8(row + 8 * chunk, f);
            store4(record(h), 1, chunk, f);
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        } else {
          uint8_t* out = record(h) + 256;
#pragma unroll
          for (int u = 0; u < PER; ++u) {
            if (lane.there[u]) store_fp8<N>(out + lane.lo[u], xa[u]);
            if (lane.turned[u]) store_fp8<N>(out + lane.hi[u], xb[u]);
          }
        }
      }
    }
  }
  if (id == 0 && blockIdx.y == 0) {
    if (held) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const size_t at = a.c.row(b, g, slot);
        if (a.positions) a.positions[at] = (int)p;
        if (a.weights) a.weights[at] = 0.f;
      }
    } else if (wanted && a.status) {
      atomicOr(a.status, fits ? STATUS_PAGE : STATUS_CAPACITY);
    }
  }
}

bool weight_by_8(const NormArgs& w, int size) {
  return ((uintptr_t)w.weight & 15) == 0 && w.sh * (w.wide ? 4 : size) % 16 == 0;
}

// How a call is spread: lanes a token, by the units of a head.
struct Shape {
  bool by8;
  int units, lanes;
  Shape(bool aligned, int pairs, int dim) {
    by8 = aligned && pairs % 8 == 0 && dim % 8 == 0;
    const int step = by8 ? 8 : 1;
    units = pairs / step + (dim - 2 * pairs) / step;
    lanes = !by8 ? 64 : units <= 8 ? 8 : units <= 16 ? 16 : units <= 32 ? 32 : 64;
  }
};

// Calls f<N, L, PER>(): 8 to 64 lanes of one unit for rows in 16-byte pieces
// (64 lanes: two), else 64 lanes of up to 4 or 16 elements.
template <typename F>
void with_shape(const Shape& s, F f) {
  using std::integral_constant;
  auto run = [&](auto n, auto l, auto per) { f(n, l, per); };
#define SKV_I(x) integral_constant<int, x>{}
  if (!s.by8) {
    if (s.units <= 256) run(SKV_I(1), SKV_I(64), SKV_I(4));
    else run(SKV_I(1), SKV_I(64), SKV_I(16));
  } else if (s.lanes == 8) run(SKV_I(8), SKV_I(8), SKV_I(1));
  else if (s.lanes == 16) run(SKV_I(8), SKV_I(16), SKV_I(1));
  else if (s.lanes == 32) run(SKV_I(8), SKV_I(32), SKV_I(1));
  else run(SKV_I(8), SKV_I(64), SKV_I(2));
#undef SKV_I
}

// Heads a block walks, a multiple of what is in flight: split where the tokens'
// blocks are fewer than `target`.  (One head a block, its angles formed for it
// alone: 5003 x 7 x 96 in FP32 18.7 us, 12.0 with four.)
int split_heads(int64_t blocks, int heads, int batch, int target, int& per) {
  const int groups = (heads + batch - 1) / batch;
  const int64_t wanted = (target + blocks - 1) / blocks;
  const int splits = wanted < groups ? (int)wanted : groups;
  per = (groups + splits - 1) / splits * batch;
  return (heads + per - 1) / per;
}

constexpr int NG_BLOCKS = 1024;  // blocks of the gradient: 4 of 4 waves on each of 256 CUs

// Blocks of the gradient along tokens (x) and heads (y); `per` heads each, with
// one weight for all of them a multiple of the `batch` in flight (half of it, the
// other half loaded twice, in rows of 100 BF16 elements: 1000 tokens x 8 heads 15.7
// us, 11.4 so; 256 x 20 11.9 and 10.0; 1 x 20 6.2 and 7.0, less than the host's call).
struct GradGrid {
  int x, y, per;
  GradGrid(int64_t tokens, int heads, int lanes, int batch, bool per_head) {
    const int64_t groups = (tokens * lanes + RO_BLOCK - 1) / RO_BLOCK;
    if (per_head) {
      per = 1;
      y = heads;
    } else {
      y = split_heads(groups, heads, batch, NG_BLOCKS, per);
    }
    const int64_t most = NG_BLOCKS / y > 0 ? NG_BLOCKS / y : 1;
    x = (int)(groups < most ? groups : most);
  }
};

template <typename T, typename W>
void norm_typed(const NormRows& a, const Rows& y, hipStream_t st) {
  const Shape s(rows_by_8(a.x, sizeof(T)) && rows_by_8(y, sizeof(T)) && weight_by_8(a.w, sizeof(T)), a.r.pairs, a.dim);
  const int64_t tokens = (int64_t)a.batch * a.n;
  const int64_t blocks = (tokens * s.lanes + RO_BLOCK - 1) / RO_BLOCK;
  with_shape(s, [&](auto n, auto l, auto per_lane) {
    int per;
    const int splits = split_heads(blocks, a.heads, batch_of<n(), per_lane()>, RO_TARGET_BLOCKS, per);
    hipLaunchKernelGGL((k_norm_rotary<T, W, n(), l(), per_lane()>), dim3((unsigned)blocks, splits), dim3(RO_BLOCK), 0, st,
                       a.r, a.w, a.x, y, tokens, s.units, a.n, a.heads, a.dim, per, a.interleaved);
  });
}

// Returns the partial rows of dw.
template <typename T>
int grad_typed(const NormRows& a, const Rows& g, const Rows& y, float* partial, hipStream_t st) {
  const Shape s(rows_by_8(a.x, sizeof(T)) && rows_by_8(g, sizeof(T)) && rows_by_8(y, sizeof(T)) &&
                    weight_by_8(a.w, sizeof(T)),
                a.r.pairs, a.dim);
  const int64_t tokens = (int64_t)a.batch * a.n;
  int rows = 0;
  with_shape(s, [&](auto n, auto l, auto per_lane) {
    const GradGrid grid(tokens, a.heads, l(), batch_of<n(), per_lane()>, a.w.sh != 0);
    rows = grid.x * grid.y;
    auto kernel = a.w.sh ? k_norm_grad<T, n(), l(), per_lane(), true> : k_norm_grad<T, n(), l(), per_lane(), false>;
    hipLaunchKernelGGL(kernel, dim3(grid.x, grid.y), dim3(RO_BLOCK), 0, st, a.r, a.w, g, a.x, y, tokens, s.units, a.n,
                       a.heads, a.dim, grid.per, a.interleaved, partial);
  });
  return rows;
}

}  // namespace

void launch_norm_rotary(const NormRows& a, const Rows& y, int dtype, hipStream_t st) {
  auto run = dtype == 0   ? (a.w.wide ? norm_typed<BF16, float> : norm_typed<BF16, BF16>)
             : dtype == 1 ? (a.w.wide ? norm_typed<FP16, float> : norm_typed<FP16, FP16>)
                          : norm_typed<float, float>;
  run(a, y, st);
}

size_t norm_grad_workspace(int64_t tokens, int heads, int dim, bool per_head) {
  // (x y of any GradGrid: y is `heads`, or at most NG_BLOCKS; x at most NG_BLOCKS / y, or 1)
  const int64_t least = per_head ? heads : 1;
  return (size_t)(least > NG_BLOCKS ? least : NG_BLOCKS) * dim * 4;
}

void launch_norm_grad(const NormRows& a, const Rows& g, const Rows& y, int dtype, void* dw, int dw_dtype,
                      float* partial, hipStream_t st) {
  auto run = dtype == 0 ? grad_typed<BF16> : dtype == 1 ? grad_typed<FP16> : grad_typed<float>;
  const int shares = run(a, g, y, partial, st), rows = a.w.sh ? a.heads : 1;
  hipLaunchKernelGGL(k_norm_weight, dim3((a.dim + 63) / 64, rows), dim3(1024), 0, st, partial, shares / rows, a.dim, dw,
                     dw_dtype);
}

void launch_cache_write_normed(const WriteArgs& a, const NormArgs& qw, const NormArgs& kw, hipStream_t st) {
  const bool aligned = rows_by_8(a.k, 2) && rows_by_8(a.v, 2) && weight_by_8(kw, 2) &&
                       (!a.q.data || (rows_by_8(a.q, 2) && rows_by_8(a.q_out, 2) && weight_by_8(qw, 2)));
  const Shape s(aligned, a.r.pairs, D);
  const int64_t tokens = (int64_t)a.c.batch * a.n;
  const int64_t blocks = (tokens * s.lanes + RO_BLOCK - 1) / RO_BLOCK;
  const int first = a.q.data ? 0 : WG_K;
  int per;
  const int splits = split_rows(blocks, WG_ALL - first, per);
  auto kernel = !s.by8         ? (a.c.four ? k_cache_write_normed<1, 64, 4, true> : k_cache_write_normed<1, 64, 4, false>)
                : s.lanes == 16 ? (a.c.four ? k_cache_write_normed<8, 16, 1, true> : k_cache_write_normed<8, 16, 1, false>)
                                : (a.c.four ? k_cache_write_normed<8, 32, 1, true> : k_cache_write_normed<8, 32, 1, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, splits), dim3(RO_BLOCK), 0, st, a, qw, kw, tokens, s.units, first, per);
}

}  // namespace skv
