// Norms of queries and keys, a row of head_dim values at a time, with the rotation by position in the same
// pass, and their gradients.
//
//   n(x) = x rsqrt(mean x^2 + eps)                    RMSNorm
//   n(x) = (x - mean x) rsqrt(mean (x - mean x)^2 + eps)   LayerNorm
//   a(x) = w n(x) (+ b);  R: the two halves of a row turned by the angles of its position
//   forward   y = R a(x)  or  y = a(R x)
//   backward  with g = R^T dy or dy, and n, rstd of x or of R x:
//             dw = sum g n,  db = sum g,  d = g w,  dz = rstd (d - n mean(d n) [- mean d])
//             dx = dz or R^T dz
// All in fp32, one rounding at the end; row statistics are recomputed in the backward pass, where the row is in
// registers anyway. A row is read once and stays with its few lanes (head_rows.cuh), no barrier in the loop,
// arithmetic in packed pairs (a half as many instructions as without: 119 us instead of 92 at a training step of 8192
// tokens, 32 / 8 heads x 128 bf16, which now is 79.6). There: forward 168 MB in 31.5 us, 5.3 TB/s; backward, with the sums
// of the weight gradients, 252 MB in 48, 5.2 TB/s. Neither the memory (47 and 60 % of its peak with cold caches) nor the
// issue slots (44 and 49 %) are full: at four and three CTAs to an SM, as registers leave room for, rows are waited for.
// Other shapes, 4096 tokens, forward, and forward and backward (floors at 6.55 TB/s): fp32 32 / 8 x 128 28.8 us (25.8),
// 74.5 (51.4); bf16 16 / 4 x 256 16.0 (13.1), 49.6 (25.9); 8 / 2 x 512 18.5 (13.5), 56.2 (26.3); rows that cannot be read
// in 16-byte vectors: 32 / 8 x 126 26.7 (12.8), 163 (25.4), 16 / 4 x 258 41.3 (13.2), 148 (26.1).
#include "head_rows.cuh"

namespace trx {

struct QkSide {
  const void* x;
  const void* dy;   // backward
  void* y;          // forward: y; backward: dx
  const void* w;
  const void* b;    // LayerNorm's bias, or null
  int64_t xs[3], dys[3], ys[3];  // (batch, seq, head) strides in elements
  int H;
};
struct QkParams {
  QkSide side[2];  // queries, keys
  const void* cos_t;
  const void* sin_t;
  const void* positions;  // null: a token's own index in its sequence
  int64_t pos_strides[2];
  int64_t table_rows, table_stride;
  int64_t tokens, S;
  int D, pos64;
  int table_dtype, w_dtype;
  int layer, first;   // LayerNorm; the norm comes before the rotation
  float eps;
  int q_chunks;       // forward: of the grid's y
  int heads_per_cta;  // backward: of an item
  int q_blocks;       // backward: of the grid's x
  float* part;        // backward: [blocks][2][D] sums of g n and of g
};

constexpr int QK_THREADS = 128;
// Backward: one wave of so many CTAs; rows of a step. 8192 tokens, 32 / 8 heads x 128 bf16, forward and backward, with
// 2 steps in shared memory: 3 CTAs of 2 rows 79.6 us; 3 steps 80.5; 6 of one row 79.5 (LayerNorm 23.9 us so, 23.3);
// 4 CTAs 82 to 86 (128 registers are too few). Rows loaded where they are used, none ahead: 88.
constexpr int QK_BWD_CTAS_PER_SM = 3;
constexpr int QK_BWD_ROWS = 2;

// A row's two halves, and what they are turned by: cos, sin, -sin.
template <int N>
struct QkRow {
  HalfPairs<N> a, b;
};
template <int N>
struct QkAngles {
  HalfPairs<N> c, s, ns;
};

template <int VEC, int CH, int LPR>
__device__ __forceinline__ HalfPairs<VEC * CH> load_pairs(const void* base, int dtype, int64_t first, int lane, int n,
                                                          float fill) {
  float f[VEC * CH];
  load_columns<VEC, CH, LPR>(base, dtype, first, lane, n, fill, f);
  HalfPairs<VEC * CH> r;
#pragma unroll
  for (int i = 0; i < VEC * CH / 2; ++i) r.v[i] = make_float2(f[2 * i], f[2 * i + 1]);
  return r;
}

// The angles of a token for a lane's columns. A position outside the tables has none: its rows become NaN.
template <int VEC, int CH, int LPR>
__device__ __forceinline__ QkAngles<VEC * CH> load_angles(const QkParams& p, int64_t b, int64_t s, int lane, int half) {
  int64_t pos = s;
  if (p.positions) {
    const int64_t at = b * p.pos_strides[0] + s * p.pos_strides[1];
    pos = p.pos64 ? __ldg(static_cast<const long long*>(p.positions) + at)
                  : __ldg(static_cast<const int*>(p.positions) + at);
  }
  const bool there = pos >= 0 && pos < p.table_rows;
  const float fill = there ? 0.0f : __int_as_float(0x7fffffff);
  QkAngles<VEC * CH> r;
  r.c = load_pairs<VEC, CH, LPR>(p.cos_t, p.table_dtype, pos * p.table_stride, lane, there ? half : 0, fill);
  r.s = load_pairs<VEC, CH, LPR>(p.sin_t, p.table_dtype, pos * p.table_stride, lane, there ? half : 0, fill);
#pragma unroll
  for (int i = 0; i < VEC * CH / 2; ++i) r.ns.v[i] = make_float2(-r.s.v[i].x, -r.s.v[i].y);
  return r;
}

// (x1, x2) turned by the angles, and back: (x1 c - x2 s, x2 c + x1 s), (x1 c + x2 s, x2 c - x1 s).
template <int N>
__device__ __forceinline__ void turn_pairs(QkRow<N>& x, const HalfPairs<N>& c, const HalfPairs<N>& s,
                                           const HalfPairs<N>& ns) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 a = fma2(x.b.v[i], ns.v[i], mul2(x.a.v[i], c.v[i]));
    x.b.v[i] = fma2(x.a.v[i], s.v[i], mul2(x.b.v[i], c.v[i]));
    x.a.v[i] = a;
  }
}

// Sum over the row of x y.
template <int LPR, int N>
__device__ __forceinline__ float row_dot(const QkRow<N>& x, const QkRow<N>& y) {
  float2 sum = mul2(x.a.v[0], y.a.v[0]);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if (i > 0) sum = fma2(x.a.v[i], y.a.v[i], sum);
    sum = fma2(x.b.v[i], y.b.v[i], sum);
  }
  return lanes_sum<LPR>(sum.x + sum.y);
}
template <int LPR, int N>
__device__ __forceinline__ float row_sum(const QkRow<N>& x) {
  float2 sum = x.a.v[0];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if (i > 0) sum = add2(sum, x.a.v[i]);
    sum = add2(sum, x.b.v[i]);
  }
  return lanes_sum<LPR>(sum.x + sum.y);
}

// A LayerNorm's row minus its mean (0 in columns behind the row).
template <int VEC, int CH, int LPR>
__device__ __forceinline__ void centre(QkRow<VEC * CH>& x, int lane, int half, float inv_d) {
  const float mean = row_sum<LPR>(x) * inv_d;
  auto inside = [&](int i) { return ((i / VEC) * LPR + lane) * VEC < half; };
#pragma unroll
  for (int i = 0; i < VEC * CH / 2; ++i) {
    const float2 m = make_float2(inside(2 * i) ? -mean : 0.0f, inside(2 * i + 1) ? -mean : 0.0f);
    x.a.v[i] = add2(x.a.v[i], m);
    x.b.v[i] = add2(x.b.v[i], m);
  }
}

// Grid (tokens, chunks of heads of q, then of k): a thread has its columns' weights and angles for all heads of
// its chunk, ROWS of them in flight.
template <typename T, int VEC, int LPR, int CH, int ROWS>
__global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_kernel(const __grid_constant__ QkParams p) {
  constexpr int N = VEC * CH;
  const int lane = threadIdx.x % LPR, half = p.D / 2;
  int64_t token = static_cast<int64_t>(blockIdx.x) * (QK_THREADS / LPR) + threadIdx.x / LPR;
  const bool live = token < p.tokens;
  if (!live) token = p.tokens - 1;  // its lanes take part in the shuffles
  const int64_t b = token / p.S, s = token - b * p.S;
  const bool keys = static_cast<int>(blockIdx.y) >= p.q_chunks;
  const QkSide& side = p.side[keys ? 1 : 0];
  const int h_begin = (static_cast<int>(blockIdx.y) - (keys ? p.q_chunks : 0)) * p.heads_per_cta;
  const int h_end = min(side.H, h_begin + p.heads_per_cta);
  const T* x = static_cast<const T*>(side.x) + b * side.xs[0] + s * side.xs[1];
  T* y = static_cast<T*>(side.y) + b * side.ys[0] + s * side.ys[1];

  const QkAngles<N> t = load_angles<VEC, CH, LPR>(p, b, s, lane, half);
  const HalfPairs<N> w1 = load_pairs<VEC, CH, LPR>(side.w, p.w_dtype, 0, lane, half, 0.0f);
  const HalfPairs<N> w2 = load_pairs<VEC, CH, LPR>(side.w, p.w_dtype, half, lane, half, 0.0f);
  const float inv_d = __fdiv_rn(1.0f, static_cast<float>(p.D));

  for (int h0 = h_begin; h0 < h_end; h0 += ROWS) {
    HalfRow<T, VEC, CH> r1[ROWS], r2[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const T* row = x + min(h0 + u, h_end - 1) * side.xs[2];
      r1[u].template load<LPR>(row, lane, half);
      r2[u].template load<LPR>(row + half, lane, half);
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      QkRow<N> z{pairs_of(r1[u]), pairs_of(r2[u])};
      if (!p.first) turn_pairs(z, t.c, t.s, t.ns);
      if (p.layer) centre<VEC, CH, LPR>(z, lane, half, inv_d);
      const float rstd = rsqrtf(fmaf(row_dot<LPR>(z, z), inv_d, p.eps));
      const float2 rstd2 = make_float2(rstd, rstd);
      if (side.b) {
        const HalfPairs<N> b1 = load_pairs<VEC, CH, LPR>(side.b, p.w_dtype, 0, lane, half, 0.0f);
        const HalfPairs<N> b2 = load_pairs<VEC, CH, LPR>(side.b, p.w_dtype, half, lane, half, 0.0f);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          z.a.v[i] = fma2(mul2(z.a.v[i], rstd2), w1.v[i], b1.v[i]);
          z.b.v[i] = fma2(mul2(z.b.v[i], rstd2), w2.v[i], b2.v[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          z.a.v[i] = mul2(mul2(z.a.v[i], rstd2), w1.v[i]);
          z.b.v[i] = mul2(mul2(z.b.v[i], rstd2), w2.v[i]);
        }
      }
      if (p.first) turn_pairs(z, t.c, t.s, t.ns);
      if (live && h0 + u < h_end) {
        T* row = y + (h0 + u) * side.ys[2];
        float f[N];
        unpair(z.a, f);
        store_half<T, VEC, CH, LPR>(row, lane, half, f);
        unpair(z.b, f);
        store_half<T, VEC, CH, LPR>(row + half, lane, half, f);
      }
    }
  }
}

// Rows of the backward pass on their way into shared memory: QK_STAGES steps of ROWS heads, 4 ROWS vectors of 16
// bytes to a thread each, which it alone reads: nobody waits for anybody.
constexpr int QK_STAGES = 2;
__device__ __forceinline__ void copy16(uint4* to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from), "r"(there ? 16 : 0)
               : "memory");
}

// Blocks [0, q_blocks) walk over the queries, the others over the keys, ROWS heads of a token at a time; every
// thread keeps the sums of its columns' weight gradients, which meet in shared memory at the end. With z the row
// that is normalised (a LayerNorm's centred) and e = rstd g w: dx = e - z rstd^2 mean(e z) [- mean e].
template <typename T, int VEC, int LPR, int CH, int ROWS, bool LAYER>
__global__ void __launch_bounds__(QK_THREADS, QK_BWD_CTAS_PER_SM)
    qk_norm_rope_bwd_kernel(const __grid_constant__ QkParams p) {
  constexpr int N = VEC * CH, GROUPS = QK_THREADS / LPR;
  const int lane = threadIdx.x % LPR, half = p.D / 2;
  const bool keys = static_cast<int>(blockIdx.x) >= p.q_blocks;
  const QkSide& side = p.side[keys ? 1 : 0];
  const int blocks = keys ? gridDim.x - p.q_blocks : p.q_blocks;
  const int block = keys ? blockIdx.x - p.q_blocks : blockIdx.x;
  const float inv_d = __fdiv_rn(1.0f, static_cast<float>(p.D));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const HalfPairs<N> w1 = load_pairs<VEC, CH, LPR>(side.w, p.w_dtype, 0, lane, half, 0.0f);
  const HalfPairs<N> w2 = load_pairs<VEC, CH, LPR>(side.w, p.w_dtype, half, lane, half, 0.0f);
  QkRow<N> dw, db;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) dw.a.v[i] = dw.b.v[i] = db.a.v[i] = db.b.v[i] = make_float2(0.0f, 0.0f);

  constexpr bool RING = VEC > 1;
  constexpr int VECTORS = 4 * ROWS;  // of a step: x's two halves, dy's two halves of each row
  __shared__ uint4 ring[(RING ? QK_STAGES : 1) * VECTORS * QK_THREADS];
  static_assert(sizeof(ring) >= sizeof(float) * (QK_THREADS / 32) * 2 * N * LPR, "the sums at the end");
  const unsigned chunks = (side.H + p.heads_per_cta - 1) / p.heads_per_cta;
  const unsigned items = static_cast<unsigned>(p.tokens) * chunks, seq = static_cast<unsigned>(p.S);
  struct Item {
    const T* x;
    const T* dy;
    int64_t b, s;
    int h, heads;  // at least one head; rows behind them are the last one again, without a gradient
    bool live;
  };
  auto item_at = [&](unsigned i) {
    Item r;
    r.live = i < items;
    i = r.live ? i : items - 1;
    const unsigned token = i / chunks;
    r.h = (i - token * chunks) * p.heads_per_cta;
    r.heads = side.H - r.h;
    r.b = token / seq;
    r.s = token - static_cast<unsigned>(r.b) * seq;
    r.x = static_cast<const T*>(side.x) + r.b * side.xs[0] + r.s * side.xs[1] + r.h * side.xs[2];
    r.dy = static_cast<const T*>(side.dy) + r.b * side.dys[0] + r.s * side.dys[1] + r.h * side.dys[2];
    return r;
  };
  const unsigned stride = blocks * GROUPS, group = (threadIdx.x % 32) / LPR;
  // whole warps leave together: the item of a warp's first row decides
  unsigned first = (block * QK_THREADS + (threadIdx.x & ~31)) / LPR;
  // what is copied next, and where to
  unsigned ahead = first;
  int ahead_h = 0, to = 0, from = 0;
  Item coming;
  auto copy_step = [&]() {
    if constexpr (RING) {
      if (ahead < items) {
        if (ahead_h == 0) coming = item_at(ahead + group);
        const bool inside = lane * VEC < half;
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
          const int h = min(ahead_h + u, coming.heads - 1), col = inside ? lane * VEC : 0;
          const bool there = inside && coming.live && ahead_h + u < coming.heads;
          uint4* slot = ring + (to * VECTORS + 4 * u) * QK_THREADS + threadIdx.x;
          const T* x = coming.x + h * side.xs[2] + col;
          const T* dy = coming.dy + h * side.dys[2] + col;
          copy16(slot, x, inside);
          copy16(slot + QK_THREADS, x + half, inside);
          copy16(slot + 2 * QK_THREADS, dy, there);
          copy16(slot + 3 * QK_THREADS, dy + half, there);
        }
        ahead_h += ROWS;
        if (ahead_h >= p.heads_per_cta) {
          ahead_h = 0;
          ahead += stride;
        }
        to = to + 1 == QK_STAGES ? 0 : to + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
#pragma unroll
  for (int i = 0; i < QK_STAGES - 1; ++i) copy_step();

  for (; first < items; first += stride) {
    const Item item = item_at(first + group);
    const bool live = item.live;
    const int heads = item.heads;
    T* dx = static_cast<T*>(side.y) + item.b * side.ys[0] + item.s * side.ys[1] + item.h * side.ys[2];
    const QkAngles<N> t = load_angles<VEC, CH, LPR>(p, item.b, item.s, lane, half);
    for (int h0 = 0; h0 < p.heads_per_cta; h0 += ROWS) {
      HalfRow<T, VEC, CH> r1[ROWS], r2[ROWS], g1[ROWS], g2[ROWS];
      if constexpr (RING) {
        asm volatile("cp.async.wait_group %0;" ::"n"(QK_STAGES - 2) : "memory");
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
          const uint4* slot = ring + (from * VECTORS + 4 * u) * QK_THREADS + threadIdx.x;
          r1[u].raw = slot[0];
          r2[u].raw = slot[QK_THREADS];
          g1[u].raw = slot[2 * QK_THREADS];
          g2[u].raw = slot[3 * QK_THREADS];
        }
        from = from + 1 == QK_STAGES ? 0 : from + 1;
        copy_step();
      } else {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
          const int h = min(h0 + u, heads - 1), there = live && h0 + u < heads ? half : 0;
          r1[u].template load<LPR>(item.x + h * side.xs[2], lane, half);
          r2[u].template load<LPR>(item.x + h * side.xs[2] + half, lane, half);
          g1[u].template load<LPR>(item.dy + h * side.dys[2], lane, there);
          g2[u].template load<LPR>(item.dy + h * side.dys[2] + half, lane, there);
        }
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        QkRow<N> z{pairs_of(r1[u]), pairs_of(r2[u])}, g{pairs_of(g1[u]), pairs_of(g2[u])};
        if (p.first) turn_pairs(g, t.c, t.ns, t.s);
        else turn_pairs(z, t.c, t.s, t.ns);
        if constexpr (LAYER) centre<VEC, CH, LPR>(z, lane, half, inv_d);
        const float rstd = rsqrtf(fmaf(row_dot<LPR>(z, z), inv_d, p.eps));
        const float2 rstd2 = make_float2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          if constexpr (LAYER) {
            db.a.v[i] = add2(db.a.v[i], g.a.v[i]);
            db.b.v[i] = add2(db.b.v[i], g.b.v[i]);
          }
          g.a.v[i] = mul2(g.a.v[i], rstd2);
          g.b.v[i] = mul2(g.b.v[i], rstd2);
          dw.a.v[i] = fma2(g.a.v[i], z.a.v[i], dw.a.v[i]);
          dw.b.v[i] = fma2(g.b.v[i], z.b.v[i], dw.b.v[i]);
          g.a.v[i] = mul2(g.a.v[i], w1.v[i]);
          g.b.v[i] = mul2(g.b.v[i], w2.v[i]);
        }
        const float k = -row_dot<LPR>(g, z) * inv_d * rstd * rstd;
        const float2 k2 = make_float2(k, k);
        float mean = 0.0f;
        if constexpr (LAYER) mean = -row_sum<LPR>(g) * inv_d;
        const float2 mean2 = make_float2(mean, mean);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          g.a.v[i] = fma2(z.a.v[i], k2, g.a.v[i]);
          g.b.v[i] = fma2(z.b.v[i], k2, g.b.v[i]);
          if constexpr (LAYER) {
            g.a.v[i] = add2(g.a.v[i], mean2);
            g.b.v[i] = add2(g.b.v[i], mean2);
          }
        }
        if (!p.first) turn_pairs(g, t.c, t.ns, t.s);
        if (live && h0 + u < heads) {
          T* row = dx + (h0 + u) * side.ys[2];
          float f[N];
          unpair(g.a, f);
          store_half<T, VEC, CH, LPR>(row, lane, half, f);
          unpair(g.b, f);
          store_half<T, VEC, CH, LPR>(row + half, lane, half, f);
        }
      }
    }
  }

  // the warp's rows, then the CTA's warps, in a fixed order
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // the ring's memory
  auto sums = reinterpret_cast<float(*)[2 * N * LPR]>(ring);
  float* part = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.D;
#pragma unroll
  for (int pass = 0; pass < (LAYER ? 2 : 1); ++pass) {
    if (pass) __syncthreads();
    float f[2][N];
    unpair(pass ? db.a : dw.a, f[0]);
    unpair(pass ? db.b : dw.b, f[1]);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float a = f[e][i];
#pragma unroll
        for (int o = 16; o >= LPR; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (threadIdx.x % 32 < LPR)
          sums[threadIdx.x / 32][e * N * LPR + ((i / VEC) * LPR + lane) * VEC + i % VEC] = a;
      }
    __syncthreads();
    for (int col = threadIdx.x; col < p.D; col += QK_THREADS) {
      const int at = col < half ? col : N * LPR + col - half;
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < QK_THREADS / 32; ++i) v += sums[i][at];
      part[pass * p.D + col] = v;
    }
  }
}

struct QkReduce {
  const float* part;
  void* out[4];      // dw of q, of k, db of q, of k; null: not asked for
  int q_blocks, blocks, D, dtype;
};
// Grid (columns / 32, 4): a block's 32 rows of threads have every 32nd partial sum of 32 columns.
__global__ void __launch_bounds__(1024) qk_norm_reduce_kernel(const QkReduce r) {
  __shared__ float sm[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  void* out = r.out[blockIdx.y];
  if (!out) return;
  const bool keys = blockIdx.y & 1;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, col = blockIdx.x * 32 + tx;
  float v = 0.0f;
  constexpr int N = 8;  // loads in flight
  const int end = keys ? r.blocks : r.q_blocks;
  for (int i0 = (keys ? r.q_blocks : 0) + ty; i0 < end; i0 += 32 * N) {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[i] = col < r.D && i0 + 32 * i < end
                 ? r.part[(static_cast<int64_t>(i0 + 32 * i) * 2 + (blockIdx.y >> 1)) * r.D + col]
                 : 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) v += f[i];
  }
  sm[ty][tx] = v;
  __syncthreads();
  const float sum = warp_reduce<false>(sm[tx][ty]);  // of column ty
  const int c = blockIdx.x * 32 + ty;
  if (tx == 0 && c < r.D) {
    if (r.dtype == TRX_F32) Pack<float>::store1(static_cast<float*>(out) + c, sum);
    else if (r.dtype == TRX_F16) Pack<__half>::store1(static_cast<__half*>(out) + c, sum);
    else Pack<__nv_bfloat16>::store1(static_cast<__nv_bfloat16*>(out) + c, sum);
  }
}

// Whether every row, of every tensor and table, can be read in 16-byte vectors of the activation type, at most
// one to a lane of a warp.
static bool qk_vector(const QkParams& p, int vec, bool backward) {
  const int half = p.D / 2;
  if (half % vec || half > 32 * vec) return false;
  const int table_vec = p.table_dtype == TRX_F32 ? 4 : 8;
  if (!aligned_to(p.cos_t, 16) || !aligned_to(p.sin_t, 16) || p.table_stride % table_vec) return false;
  for (const QkSide& s : p.side) {
    if (s.H == 0) continue;
    if (!aligned_to(s.x, 16) || !aligned_to(s.y, 16) || !aligned_to(s.w, 16) || (s.b && !aligned_to(s.b, 16)) ||
        (backward && !aligned_to(s.dy, 16)))
      return false;
    for (int i = 0; i < 3; ++i)
      if (s.xs[i] % vec || s.ys[i] % vec || (backward && s.dys[i] % vec)) return false;
  }
  return true;
}

template <typename T, int VEC, int LPR, int CH, int ROWS>
static int launch_qk(QkParams& p, cudaStream_t stream) {
  constexpr int TOKENS = QK_THREADS / LPR;
  const int64_t blocks = (p.tokens + TOKENS - 1) / TOKENS;
  // Sixteen heads to a thread where that still gives every SM eight CTAs, eight where it gives one, else four: 8192
  // tokens, 32 / 8 heads x 128 bf16 in 16, 8, 4 heads 31.5, 33.6, 36.2 us; 2103 tokens, 20 / 4 heads x 80 fp16
  // 12.9, 8.9, 9.6 us.
  const int64_t all = blocks * (p.side[0].H + p.side[1].H), sms = sm_count_of_current_device();
  p.heads_per_cta = all >= 16 * 8 * sms ? 16 : all >= 8 * sms ? 8 : ROWS;
  p.q_chunks = (p.side[0].H + p.heads_per_cta - 1) / p.heads_per_cta;
  const int chunks = p.q_chunks + (p.side[1].H + p.heads_per_cta - 1) / p.heads_per_cta;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(chunks));
  qk_norm_rope_kernel<T, VEC, LPR, CH, ROWS><<<grid, QK_THREADS, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

template <typename T>
static int launch_qk_forward(QkParams& p, cudaStream_t s) {
  constexpr int VEC = Pack<T>::VEC;
  if (!qk_vector(p, VEC, false))
    return p.D <= 128 ? launch_qk<T, 1, 32, 2, 2>(p, s) : launch_qk<T, 1, 32, 8, 1>(p, s);
  switch (lanes_for(p.D / 2, VEC)) {
    case 4: return launch_qk<T, VEC, 4, 1, 4>(p, s);
    case 8: return launch_qk<T, VEC, 8, 1, 4>(p, s);
    case 16: return launch_qk<T, VEC, 16, 1, 4>(p, s);
    default: return launch_qk<T, VEC, 32, 1, 4>(p, s);
  }
}

static int qk_bwd_blocks() { return sm_count_of_current_device() * QK_BWD_CTAS_PER_SM; }

template <typename T, int VEC, int LPR, int CH, int ROWS>
static int launch_qk_bwd(QkParams& p, QkReduce& r, cudaStream_t stream) {
  constexpr int GROUPS = QK_THREADS / LPR;
  // eight heads of a token to an item, fewer where that leaves threads without one
  const int64_t heads = p.side[0].H + p.side[1].H;
  p.heads_per_cta = 8;
  while (p.heads_per_cta > ROWS && p.tokens * heads < p.heads_per_cta * qk_bwd_blocks() * GROUPS) p.heads_per_cta /= 2;
  auto needs = [&](const QkSide& s) {
    return (p.tokens * ((s.H + p.heads_per_cta - 1) / p.heads_per_cta) + GROUPS - 1) / GROUPS;
  };
  const int64_t most = qk_bwd_blocks(), nq = needs(p.side[0]), nk = needs(p.side[1]);
  int64_t q = nq, k = nk;
  if (nq + nk > most) {  // a share each, and one block at least
    q = most * nq / (nq + nk);
    q = nq && q < 1 ? 1 : q;
    q = nk && q > most - 1 ? most - 1 : q;
    k = nk < most - q ? nk : most - q;
  }
  p.q_blocks = static_cast<int>(q);
  if (q + k > 0) {
    auto run = [&](auto kernel) { kernel<<<static_cast<unsigned>(q + k), QK_THREADS, 0, stream>>>(p); };
    if (p.layer) run(qk_norm_rope_bwd_kernel<T, VEC, LPR, CH, ROWS, true>);
    else run(qk_norm_rope_bwd_kernel<T, VEC, LPR, CH, ROWS, false>);
    if (cudaGetLastError() != cudaSuccess) return TRX_ERR_CUDA;
  }
  bool any = false;
  for (void* o : r.out) any = any || o;
  if (!any) return TRX_OK;
  r.part = p.part;
  r.q_blocks = p.q_blocks;
  r.blocks = static_cast<int>(q + k);
  r.D = p.D;
  r.dtype = p.w_dtype;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};  // prepared beside the end of the launch in front, which it waits for
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((p.D + 31) / 32, 4);
  cfg.blockDim = dim3(1024);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = q + k > 0 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, qk_norm_reduce_kernel, r) == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

template <typename T>
static int launch_qk_backward(QkParams& p, QkReduce& r, cudaStream_t s) {
  constexpr int VEC = Pack<T>::VEC;
  if (!qk_vector(p, VEC, true))
    return p.D <= 128 ? launch_qk_bwd<T, 1, 32, 2, 1>(p, r, s) : launch_qk_bwd<T, 1, 32, 8, 1>(p, r, s);
  switch (lanes_for(p.D / 2, VEC)) {
    case 4: return launch_qk_bwd<T, VEC, 4, 1, QK_BWD_ROWS>(p, r, s);
    case 8: return launch_qk_bwd<T, VEC, 8, 1, QK_BWD_ROWS>(p, r, s);
    case 16: return launch_qk_bwd<T, VEC, 16, 1, QK_BWD_ROWS>(p, r, s);
    default: return launch_qk_bwd<T, VEC, 32, 1, QK_BWD_ROWS>(p, r, s);
  }
}

// What both directions check; TRX_OK with p.tokens == 0 for nothing to do.
static int qk_check(QkParams& p, const void* q, const void* k, const void* q_weight, const void* k_weight,
                    const void* q_bias, const void* k_bias, int64_t B, int64_t S, int64_t Hq, int64_t Hk,
                    int64_t D, int norm, int x_dtype) {
  if (x_dtype != TRX_F32 && x_dtype != TRX_F16 && x_dtype != TRX_BF16) return TRX_ERR_DTYPE;
  if (p.table_dtype != TRX_F32 && p.table_dtype != x_dtype) return TRX_ERR_DTYPE;
  if (p.w_dtype != TRX_F32 && p.w_dtype != TRX_F16 && p.w_dtype != TRX_BF16) return TRX_ERR_DTYPE;
  if (norm != TRX_NORM_RMS && norm != TRX_NORM_LAYER) return TRX_ERR_UNSUPPORTED;
  if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || D <= 0 || D % 2 || p.table_rows < 0) return TRX_ERR_SHAPE;
  if (D > 512) return TRX_ERR_UNSUPPORTED;
  if (Hq > 65535 || Hk > 65535) return TRX_ERR_SHAPE;
  if (!(p.eps >= 0.0f)) return TRX_ERR_UNSUPPORTED;
  if (B > 0 && S > ((1ll << 31) - 1) / B) return TRX_ERR_SHAPE;
  if (B * S > 0 && (B * S) * (Hq > Hk ? Hq : Hk) >= (1ll << 31)) return TRX_ERR_SHAPE;
  p.tokens = B * S;
  p.S = S;
  p.D = static_cast<int>(D);
  p.layer = norm == TRX_NORM_LAYER;
  const void* x[2] = {q, k};
  const void* w[2] = {q_weight, k_weight};
  const void* b[2] = {q_bias, k_bias};
  const int64_t heads[2] = {Hq, Hk};
  for (int i = 0; i < 2; ++i) {
    p.side[i].x = x[i];
    p.side[i].w = w[i];
    p.side[i].b = b[i];
    p.side[i].H = static_cast<int>(heads[i]);
  }
  if (p.tokens == 0 || Hq + Hk == 0) {
    p.tokens = 0;
    return TRX_OK;
  }
  if (!p.cos_t || !p.sin_t) return TRX_ERR_NULL_POINTER;
  if (p.table_stride < D / 2) return TRX_ERR_STRIDE;
  for (const QkSide& s : p.side)
    if (s.H > 0) {
      if (!s.x || !s.w || !s.y) return TRX_ERR_NULL_POINTER;
      for (int i = 0; i < 3; ++i)
        if (s.xs[i] < 0 || s.ys[i] < 0) return TRX_ERR_STRIDE;
    }
  if (!p.positions && p.table_rows < S) return TRX_ERR_SHAPE;
  if (p.positions && (p.pos_strides[0] < 0 || p.pos_strides[1] < 0)) return TRX_ERR_STRIDE;
  if (p.positions && !aligned_to(p.positions, p.pos64 ? 8 : 4)) return TRX_ERR_ALIGNMENT;
  return TRX_OK;
}

static void take_strides(int64_t (&to)[3], const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

}  // namespace trx

using namespace trx;

extern "C" int trx_qk_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                    const void* q_bias_or_null, const void* k_bias_or_null,
                                    const void* cos_table, const void* sin_table,
                                    const void* positions_or_null, void* q_out, void* k_out, int64_t B,
                                    int64_t S, int64_t Hq, int64_t Hk, int64_t D, const int64_t strides[14],
                                    int64_t table_rows, int64_t table_row_stride, float eps, int norm,
                                    int norm_first, int positions_64, int table_dtype, int w_dtype,
                                    int x_dtype, void* stream) {
  if (!strides) return TRX_ERR_NULL_POINTER;
  QkParams p{};
  take_strides(p.side[0].xs, strides);
  take_strides(p.side[1].xs, strides + 3);
  take_strides(p.side[0].ys, strides + 6);
  take_strides(p.side[1].ys, strides + 9);
  p.pos_strides[0] = strides[12];
  p.pos_strides[1] = strides[13];
  p.side[0].y = q_out;
  p.side[1].y = k_out;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.positions = positions_or_null;
  p.pos64 = positions_64;
  p.table_rows = table_rows;
  p.table_stride = table_row_stride;
  p.table_dtype = table_dtype;
  p.w_dtype = w_dtype;
  p.first = norm_first;
  p.eps = eps;
  const int rc = qk_check(p, q, k, q_weight, k_weight, q_bias_or_null, k_bias_or_null, B, S, Hq, Hk, D, norm,
                          x_dtype);
  if (rc != TRX_OK || p.tokens == 0) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == TRX_F32) return launch_qk_forward<float>(p, s);
  return x_dtype == TRX_F16 ? launch_qk_forward<__half>(p, s) : launch_qk_forward<__nv_bfloat16>(p, s);
}

extern "C" size_t trx_qk_norm_rope_bwd_workspace_bytes(int64_t D) {
  if (D <= 0 || D > 512) return 0;
  return static_cast<size_t>(qk_bwd_blocks()) * 2 * D * sizeof(float);
}

extern "C" int trx_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k,
                                    const void* q_weight, const void* k_weight, const void* cos_table,
                                    const void* sin_table, const void* positions_or_null, void* dq, void* dk,
                                    void* dq_weight_or_null, void* dk_weight_or_null, void* dq_bias_or_null,
                                    void* dk_bias_or_null, int64_t B, int64_t S, int64_t Hq, int64_t Hk,
                                    int64_t D, const int64_t strides[20], int64_t table_rows,
                                    int64_t table_row_stride, float eps, int norm, int norm_first,
                                    int positions_64, int table_dtype, int w_dtype, int x_dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (!strides) return TRX_ERR_NULL_POINTER;
  QkParams p{};
  for (int i = 0; i < 2; ++i) {
    take_strides(p.side[i].dys, strides + 3 * i);
    take_strides(p.side[i].xs, strides + 6 + 3 * i);
    take_strides(p.side[i].ys, strides + 12 + 3 * i);
  }
  p.pos_strides[0] = strides[18];
  p.pos_strides[1] = strides[19];
  p.side[0].dy = dq_out;
  p.side[1].dy = dk_out;
  p.side[0].y = dq;
  p.side[1].y = dk;
  p.cos_t = cos_table;
  p.sin_t = sin_table;
  p.positions = positions_or_null;
  p.pos64 = positions_64;
  p.table_rows = table_rows;
  p.table_stride = table_row_stride;
  p.table_dtype = table_dtype;
  p.w_dtype = w_dtype;
  p.first = norm_first;
  p.eps = eps;
  const int rc = qk_check(p, q, k, q_weight, k_weight, nullptr, nullptr, B, S, Hq, Hk, D, norm, x_dtype);
  if (rc != TRX_OK) return rc;
  if (norm == TRX_NORM_RMS && (dq_bias_or_null || dk_bias_or_null)) return TRX_ERR_UNSUPPORTED;
  if (p.tokens > 0)
    for (const QkSide& s : p.side)
      if (s.H > 0) {
        if (!s.dy) return TRX_ERR_NULL_POINTER;
        for (int i = 0; i < 3; ++i)
          if (s.dys[i] < 0) return TRX_ERR_STRIDE;
      }
  if (!workspace || !aligned_to(workspace, 16) ||
      workspace_bytes < trx_qk_norm_rope_bwd_workspace_bytes(D))
    return TRX_ERR_WORKSPACE;
  p.part = static_cast<float*>(workspace);
  QkReduce r{};
  r.out[0] = dq_weight_or_null;
  r.out[1] = dk_weight_or_null;
  r.out[2] = dq_bias_or_null;
  r.out[3] = dk_bias_or_null;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == TRX_F32) return launch_qk_backward<float>(p, r, s);
  return x_dtype == TRX_F16 ? launch_qk_backward<__half>(p, r, s) : launch_qk_backward<__nv_bfloat16>(p, r, s);
}
