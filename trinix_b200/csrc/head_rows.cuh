// Rows of head_dim values whose halves are rotated against each other, held by a few lanes of a warp: what the
// norms of queries and keys (qk_norm_rope.cu) and the paged cache (paged_cache.cu) share.
//
// LPR lanes hold one row: lane i has the columns (c * LPR + i) * VEC + e of either half, c < CH, so that a
// column and the one that it is rotated with are in one thread, and a sum over the row is log2(LPR) shuffles.
// A warp has 32 / LPR rows. CH is 1 where a 16-byte vector to a lane covers the half, else VEC is 1.
#pragma once

#include "common.cuh"

namespace trx {

template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Half a row as it was read: a load first, the conversion where the values are used.
template <typename T, int VEC, int CH>
struct HalfRow {
  static constexpr int N = VEC * CH;
  uint4 raw;
  float one[VEC == 1 ? CH : 1];

  template <int LPR>
  __device__ __forceinline__ void load(const T* p, int lane, int half) {
    if constexpr (VEC > 1) {
      raw = lane * VEC < half ? ld_stream16(p + lane * VEC) : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = c * LPR + lane;
        one[c] = col < half ? Pack<T>::load1(p + col) : 0.0f;
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[N]) const {
    if constexpr (VEC > 1) {
      Pack<T>::unpack(raw, f);
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) f[c] = one[c];
    }
  }
};

// The same in pairs of columns, for packed arithmetic.
template <int N>
struct HalfPairs {
  float2 v[N / 2];
  static_assert(N % 2 == 0, "pairs");
};
template <typename T, int VEC, int CH>
__device__ __forceinline__ HalfPairs<VEC * CH> pairs_of(const HalfRow<T, VEC, CH>& h) {
  HalfPairs<VEC * CH> r;
  if constexpr (VEC > 1) {
    Pack<T>::unpack2(h.raw, r.v);
  } else {
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) r.v[i] = make_float2(h.one[2 * i], h.one[2 * i + 1]);
  }
  return r;
}
template <int N>
__device__ __forceinline__ void unpair(const HalfPairs<N>& p, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    f[2 * i] = p.v[i].x;
    f[2 * i + 1] = p.v[i].y;
  }
}

template <typename T, int VEC, int CH, int LPR>
__device__ __forceinline__ void store_half(T* p, int lane, int half, const float (&f)[VEC * CH]) {
  if constexpr (VEC > 1) {
    if (lane * VEC < half) st_stream16(p + lane * VEC, Pack<T>::pack(f));
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = c * LPR + lane;
      if (col < half) Pack<T>::store1(p + col, f[c]);
    }
  }
}

// A lane's columns of a parameter or table row that is `n` long, as fp32; `fill` in the columns behind it.
template <int VEC, int CH, int LPR>
__device__ __forceinline__ void load_columns(const void* base, int dtype, int64_t first, int lane, int n,
                                             float fill, float (&f)[VEC * CH]) {
#pragma unroll
  for (int i = 0; i < VEC * CH; ++i) f[i] = fill;
  if constexpr (VEC > 1) {
    if (lane * VEC < n) load_param_vec<VEC>(base, dtype, first + lane * VEC, f);
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = c * LPR + lane;
      if (col < n) f[c] = load_param1(base, dtype, first + col);
    }
  }
}

// (x1, x2) turned by the angle of (c, s); products and sums apart, as the elementwise formula rounds them.
template <int N>
__device__ __forceinline__ void turn(float (&x1)[N], float (&x2)[N], const float (&c)[N], const float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float a = __fsub_rn(__fmul_rn(x1[i], c[i]), __fmul_rn(x2[i], s[i]));
    x2[i] = __fadd_rn(__fmul_rn(x2[i], c[i]), __fmul_rn(x1[i], s[i]));
    x1[i] = a;
  }
}
// The smallest power of two of lanes, 4 to 32, that hold `half` columns at `vec` to a lane.
inline int lanes_for(int half, int vec) {
  int lanes = 4;
  while (lanes * vec < half) lanes *= 2;
  return lanes;
}

}  // namespace trx
