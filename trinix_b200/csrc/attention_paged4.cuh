// Attention forward for few query rows against many keys held in 4 bits, in the pages of a cache.
//
// A key costs D + 16 bytes (codes, step and lowest of K and of V) where 16 bits cost 4 D, so of the same memory
// bandwidth four times the keys come by, and what is done to each has to be four times cheaper than in
// attention_decode.cuh. What that rests on:
//   * The codes enter the matrix instructions as they are: a code c in the low bits of a 16-bit half is the
//     subnormal fp16 number c * 2^-24, one in the next four bits 16 times that, and mma.sync takes subnormal
//     operands. A word of eight codes becomes four operand registers by one shift and four ANDs; nothing is
//     converted, and nothing is multiplied, since with one step and lowest to a row
//         score = step_k (q . c_k) + lowest_k sum(q),    O = sum(p step_v c_v) + sum(p lowest_v).
//     The powers of two are put into Q and taken out of the results, exactly.
//   * Both products are transposed: S^T = K Q^T and O^T = V^T P^T, so that a tile's 16 is keys, or columns of V,
//     and its 8 is query rows: a group of four heads fills half of the tile where it would be a quarter. The
//     scores' fragment becomes the operand of the second product by one movmatrix per 8 keys. Which column of the
//     row a fragment's element is does not matter as long as both sides agree: a lane reads 16 (K) and 8 (V)
//     bytes of a row in one piece. Of 8 keys the fragment's rows are in the order 0, 4, 1, 5, ...: then the four
//     V rows that a load reads are neighbours.
//   * fp16 operands serve both activation types: Q's rows are scaled by a power of two to below 2^14 (what is
//     2^-28 of the row's largest value or more stays exact). Probabilities are weighed with step_v before
//     they are rounded to 11 bits, and the running maximum is that of the weighed ones, so that the largest
//     weight of a row is of the order of 1 whatever the steps are.
// The rest is as in the kernel for 16 bits: each warp has a ring of tiles of its own (32 keys; bulk copies of 16
// keys' codes and scales, which pages hold in one piece), partial results meet in shared memory and over the
// cluster. Sums, scores and O are fp32.
#pragma once

#include "attention_decode.cuh"

namespace trx {

constexpr int P4_KEYS = 32;       // keys of one tile
constexpr int P4_SUB = 16;        // of which so many lie in one page
constexpr int P4_STAGES = 4;
constexpr int P4_CTAS_PER_SM = 2;
// The steps of V that are 0, of rows of one value, are weighed as this; the others are larger (paged_cache.cuh). A
// weight over this and the keys of a sequence times 2^20 stay within fp32.
constexpr float P4_LEAST_STEP = 0x1p-80f;

struct Paged4Params : PagedAttnParams {};

template <int D, int NT>
struct P4Smem {
  static constexpr int CODES = P4_SUB * D / 2, SCALES = P4_SUB * 8;     // of 16 keys
  static constexpr int SUB_BYTES = 2 * (CODES + SCALES);                // K codes, V codes, K scales, V scales
  static constexpr int STAGE_BYTES = (P4_KEYS / P4_SUB) * SUB_BYTES;
  static constexpr int RING_BYTES = P4_STAGES * STAGE_BYTES;
  static constexpr int ROWS = 8 * NT;
  static_assert(ROWS * D * 4 <= RING_BYTES, "a warp's partial O reuses its ring");
  static constexpr int BAR_OFF = DEC_WARPS * RING_BYTES;
  static constexpr int ML_OFF = BAR_OFF + DEC_WARPS * P4_STAGES * 8;
  static constexpr int CTA_ML_OFF = ML_OFF + 2 * DEC_WARPS * ROWS * 4;
  static constexpr int FLAG_OFF = CTA_ML_OFF + 2 * ROWS * 4;
  static constexpr int TOTAL = FLAG_OFF + (DEC_WARPS + 1) * 4;
  static constexpr int DYN_BYTES = TOTAL + 128;  // slack for 128-byte alignment
};

// What is read where no page is.
__device__ uint4 p4_zeros[P4_SUB * 128 / 2 / 16];

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[WORDS]) {
  static_assert(WORDS == 1 || WORDS == 2 || WORDS == 4, "one load");
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr)
                 : "memory");
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float2 lds_float2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// Grid (splits, kv heads * row tiles, sequences), clusters of all the splits of one row tile; rows as in
// attn_decode_kernel.
template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(DEC_THREADS, P4_CTAS_PER_SM)
    attn_paged4_kernel(const __grid_constant__ Paged4Params p) {
  using L = P4Smem<D, NT>;
  constexpr int KW = D / 32;   // words of a K row to a thread
  constexpr int VW = D / 64;   // of a V row
  constexpr int MTILES = D / 16;
  constexpr int SUBS = P4_KEYS / P4_SUB;
  namespace cg = cooperative_groups;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) &
                                             ~static_cast<uintptr_t>(127));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t4 = lane & 3, g8 = lane >> 2;
  const int nsplit = gridDim.x, split = blockIdx.x;
  const int group = p.group, rows = group * p.Sq;
  const int row_tiles = (rows + L::ROWS - 1) / L::ROWS;
  const int unit = blockIdx.y / row_tiles;
  const int r0 = (blockIdx.y - unit * row_tiles) * L::ROWS;
  const int h0 = unit * group;
  const int b = by_keys(p, blockIdx.z);
  const int sk = ragged_length(p, b), shift = sk - p.Sq;

  // keys that any row of this tile sees, in tiles, and this CTA's share of them
  const int s_min = r0 / group, s_max = min(rows - 1, r0 + L::ROWS - 1) / group;
  const int hi = min(sk - 1, s_max + shift), hi_min = min(sk - 1, s_min + shift);
  int lo = 0, lo_max = 0;
  if (p.win_left >= 0) {
    lo = max(0, s_min + shift - p.win_left);
    lo_max = max(0, s_max + shift - p.win_left);
  }
  const int t_lo = lo / P4_KEYS, n_tiles = hi < lo ? 0 : hi / P4_KEYS + 1 - t_lo;
  const int share = (n_tiles + nsplit - 1) / nsplit;
  const int first = t_lo + min(n_tiles, split * share) + warp;
  const int last = t_lo + min(n_tiles, (split + 1) * share);
  int n_it = first < last ? (last - first + DEC_WARPS - 1) / DEC_WARPS : 0;

  const uint32_t ring = sbase + warp * L::RING_BYTES;
  const uint32_t bars = sbase + L::BAR_OFF + warp * P4_STAGES * 8;
  int* no_result = reinterpret_cast<int*>(smem + L::FLAG_OFF);  // [DEC_WARPS], then the CTA's
  volatile int* abort_flag = no_result + warp;

  // A lane has the page of one of the 16 keys' runs of this warp's next tiles; -1: none, or no key of it is seen.
  constexpr int TILES = 32 / SUBS;
  auto load_pages = [&](int it) {
    const int i = it + lane / SUBS, key = (first + i * DEC_WARPS) * P4_KEYS + (lane % SUBS) * P4_SUB;
    return i < n_it && key <= hi && key + P4_SUB > lo ? page_of(p.c, b, key) : -1;
  };
  // A lane's copy: run lane % SUBS, of K codes, V codes, K scales, V scales.
  const int copy_sub = lane % SUBS, copy_of = lane / SUBS;
  const bool of_codes = copy_of < 2, of_k = (copy_of & 1) == 0;
  const uint8_t* copy_src =
      of_codes ? static_cast<const uint8_t*>(of_k ? p.c.k : p.c.v) + unit * (of_k ? p.c.kp : p.c.vp)[1]
               : reinterpret_cast<const uint8_t*>((of_k ? p.c.k_scales : p.c.v_scales) +
                                                  unit * (of_k ? p.c.ksp : p.c.vsp)[1]);
  const int64_t copy_page = of_codes ? (of_k ? p.c.kp : p.c.vp)[0] : 4 * (of_k ? p.c.ksp : p.c.vsp)[0];
  const uint32_t copy_bytes = of_codes ? L::CODES : L::SCALES, copy_row = of_codes ? D / 2 : 8;
  const uint32_t copy_dst = copy_sub * L::SUB_BYTES + (of_codes ? (of_k ? 0 : L::CODES)
                                                                : 2 * L::CODES + (of_k ? 0 : L::SCALES));
  int pages_to_fill = load_pages(0);
  auto issue_fill = [&](int it) {  // the whole warp
    const int s = it % P4_STAGES;
    const int page = __shfl_sync(0xffffffffu, pages_to_fill, (it % TILES) * SUBS + copy_sub);
    if (lane == 0) mbar_expect_tx(bars + 8 * s, L::STAGE_BYTES);
    __syncwarp();
    if (lane < 4 * SUBS) {
      const int slot = ((first + it * DEC_WARPS) * P4_KEYS + copy_sub * P4_SUB) % p.c.page_size;
      const void* src = copy_src + page * copy_page + slot * copy_row;
      bulk_load(ring + s * L::STAGE_BYTES + copy_dst, page < 0 ? p4_zeros : src, copy_bytes, bars + 8 * s);
    }
  };
  if (lane == 0) {
    for (int s = 0; s < P4_STAGES; ++s) mbar_init(bars + 8 * s, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  for (int it = 0; it < min(n_it, P4_STAGES); ++it) issue_fill(it);
  // A launch that follows a recorded failure writes nothing, as in attn_decode_kernel.
  unsigned int seen = 0;
  if (lane == 0) seen = *reinterpret_cast<volatile unsigned int*>(p.status);
  const bool skip = __shfl_sync(0xffffffffu, seen, 0) != 0u;
  if (skip) n_it = min(n_it, P4_STAGES);

  // Q: row 8 n + g8 of the tile is the operand's column g8; word w of a thread has the row's columns
  // t4 * D / 4 + 8 w .. + 7, which the ANDs below take as (0, 4), (1, 5), (2, 6), (3, 7), the second and the
  // fourth pair 16 times too large.
  const float sl2 = p.scale_log2;
  uint32_t qf[NT][2 * KW][2];
  float factor[NT][2], q_sum[NT][2], slope2[NT][2];  // of rows 8 n + 2 t4, + 1, the scores' columns
  int row_s[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + g8;
    const bool live = r < rows;
    const int rr = live ? r : rows - 1;
    const uint16_t* qrow = reinterpret_cast<const uint16_t*>(p.q) + b * p.q_stride_b + (rr / group) * p.q_stride_s +
                           (h0 + rr % group) * p.q_stride_h + t4 * (D / 4);
    float x[8 * KW];
    float top = 0.0f, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const uint4 v = live ? __ldg(reinterpret_cast<const uint4*>(qrow) + w) : make_uint4(0u, 0u, 0u, 0u);
      float f[8];
      if constexpr (BF16) Pack<__nv_bfloat16>::unpack(v, f);
      else Pack<__half>::unpack(v, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[8 * w + i] = f[i];
        top = fmaxf(top, fabsf(f[i]));
        sum += f[i];
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    // the power of two that brings the row's largest value to 2^13 .. 2^14, and what takes it out again
    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 16), 240);
    const float up = __uint_as_float(static_cast<unsigned>(267 - e) << 23);
    const float down = __uint_as_float(static_cast<unsigned>(e - 13) << 23) * 0x1p24f * sl2;
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = i & 1 ? up * 0.0625f : up;
        qf[n][2 * w + i / 2][i & 1] = Pack<__half>::pack2(x[8 * w + i] * f, x[8 * w + i + 4] * f);
      }
    const float slope = p.slopes ? p.slopes[h0 + rr % group] * 1.4426950408889634f : 0.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int from = 4 * (2 * t4 + c);
      factor[n][c] = __shfl_sync(0xffffffffu, down, from);
      q_sum[n][c] = __shfl_sync(0xffffffffu, sum, from) * sl2;
      slope2[n][c] = __shfl_sync(0xffffffffu, slope, from);
      row_s[n][c] = min(rows - 1, r0 + 8 * n + 2 * t4 + c) / group;
    }
  }

  float o[MTILES][NT][4];
  float m_run[NT][2], l_run[NT][2], low_run[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m_run[n][c] = -INFINITY;
      l_run[n][c] = low_run[n][c] = 0.0f;
    }
#pragma unroll
    for (int m = 0; m < MTILES; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[m][n][i] = 0.0f;
  }
  const int key_of_row = (g8 >> 1) + ((g8 & 1) << 2);  // 0, 4, 1, 5, 2, 6, 3, 7
  const bool has_alibi = p.slopes != nullptr;
  bool ok = true;

  int it = 0;
#pragma unroll 1
  for (; it < n_it; ++it) {
    const int st = it % P4_STAGES;
    ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, (it / P4_STAGES) & 1, abort_flag, p.status,
                                           ATT_ST_SOFTMAX));
    if (!ok) break;
    const uint32_t tile = ring + st * L::STAGE_BYTES;
    const int c0 = (first + it * DEC_WARPS) * P4_KEYS;
    const bool need_mask = c0 + P4_KEYS - 1 > hi_min || c0 < lo_max;

    // scores of keys key_of_row (+ 8) of each run, weighed with V's step: x + log2 step_v
    float x[SUBS][NT][4];
    float v_low[SUBS][2], v_inv[SUBS][2];
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      const uint32_t sub = tile + u * L::SUB_BYTES;
      uint32_t ka[KW], kb[KW];
      lds_words<KW>(sub + key_of_row * (D / 2) + t4 * (D / 8), ka);
      lds_words<KW>(sub + (key_of_row + 8) * (D / 2) + t4 * (D / 8), kb);
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t a[2] = {ka[w], ka[w] >> 8}, c[2] = {kb[w], kb[w] >> 8};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t f[4] = {a[i] & 0x000F000Fu, c[i] & 0x000F000Fu, a[i] & 0x00F000F0u, c[i] & 0x00F000F0u};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816<false>(s[n], f, qf[n][2 * w + i][0], qf[n][2 * w + i][1]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = key_of_row + 8 * e, j = c0 + P4_SUB * u + key;
        const float2 ks = lds_float2(sub + 2 * L::CODES + 8 * key);
        const float2 vs = lds_float2(sub + 2 * L::CODES + L::SCALES + 8 * key);
        // fmaxf would turn a step that is not a number into the least one
        const float step = vs.x < P4_LEAST_STEP ? P4_LEAST_STEP : vs.x;
        float log_step;
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(log_step) : "f"(step));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(v_inv[u][e]) : "f"(step));
        v_low[u][e] = vs.y;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v = fmaf(s[n][2 * e + c] * factor[n][c], ks.x, fmaf(q_sum[n][c], ks.y, log_step));
            const int i = row_s[n][c] + shift;
            if (has_alibi) v = fmaf(-slope2[n][c], static_cast<float>(i - j), v);
            if (need_mask && (j > min(i, sk - 1) || (p.win_left >= 0 && j < i - p.win_left))) v = -INFINITY;
            x[u][n][2 * e + c] = v;
          }
      }
    }
    // The reference follows only when it is far behind: until a lane has a larger value the rows' maxima, 3
    // shuffles each, are not asked for.
    bool behind = false;
    float mx[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[n][c] = fmaxf(x[0][n][c], x[0][n][2 + c]);
#pragma unroll
        for (int u = 1; u < SUBS; ++u) mx[n][c] = max3(mx[n][c], x[u][n][c], x[u][n][2 + c]);
        behind = behind || mx[n][c] > m_run[n][c] + ATT_LAZY_RESCALE || (m_run[n][c] == -INFINITY && mx[n][c] > -INFINITY);
      }
    if (__any_sync(0xffffffffu, behind)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = mx[n][c];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
          if (m > m_run[n][c] + ATT_LAZY_RESCALE || (m_run[n][c] == -INFINITY && m > -INFINITY)) {
            const float f = fast_exp2(m_run[n][c] - m);  // 0 when m_run == -inf
            m_run[n][c] = m;
            l_run[n][c] *= f;
            low_run[n][c] *= f;
#pragma unroll
            for (int i = 0; i < MTILES; ++i) {
              o[i][n][c] *= f;
              o[i][n][2 + c] *= f;
            }
          }
        }
    }
    uint32_t pf[SUBS][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float ref[2] = {m_run[n][0] == -INFINITY ? 0.0f : m_run[n][0],
                            m_run[n][1] == -INFINITY ? 0.0f : m_run[n][1]};
#pragma unroll
      for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float w[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            w[c] = fast_exp2(x[u][n][2 * e + c] - ref[c]);
            float prob = w[c] * v_inv[u][e], low = prob * v_low[u][e];
            // a key that the row does not see may be anything: behind the last one there is what was there
            if (need_mask && x[u][n][2 * e + c] == -INFINITY) prob = low = 0.0f;
            l_run[n][c] += prob;
            low_run[n][c] += low;
          }
          pf[u][n][e] = transpose_8x8(Pack<__half>::pack2(w[0], w[1]));
        }
    }
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      const uint32_t sub = tile + u * L::SUB_BYTES + L::CODES + t4 * (D / 2) + g8 * (D / 16);
      uint32_t v0[VW], v1[VW], v2[VW], v3[VW];  // keys t4, + 4, + 8, + 12
      lds_words<VW>(sub, v0);
      lds_words<VW>(sub + 4 * (D / 2), v1);
      lds_words<VW>(sub + 8 * (D / 2), v2);
      lds_words<VW>(sub + 12 * (D / 2), v3);
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned pick = half ? 0x7632u : 0x5410u;
          uint32_t a = __byte_perm(v0[w], v1[w], pick), c = __byte_perm(v2[w], v3[w], pick);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t f[4] = {a & 0x000F000Fu, a & 0x00F000F0u, c & 0x000F000Fu, c & 0x00F000F0u};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816<false>(o[4 * w + 2 * half + i][n], f, pf[u][n][0], pf[u][n][1]);
            a >>= 8;
            c >>= 8;
          }
        }
    }
    __syncwarp();  // every lane has read the tile
    if ((it + P4_STAGES) % TILES == 0) pages_to_fill = load_pages(it + P4_STAGES);
    if (!skip && it + P4_STAGES < n_it) issue_fill(it + P4_STAGES);
  }
  if (!ok) {  // gave up on tile `it`: wait (bounded) for the copies still in flight
    for (int f = it; f < min(n_it, it + P4_STAGES); ++f) {
      const uint64_t t0 = global_ns();
      bool done = false;
      while (!done && global_ns() - t0 < ATT_WAIT_NS)
        done = mbar_try_wait(bars + 8 * (f % P4_STAGES), (f / P4_STAGES) & 1);
      if (!done) atomicOr(p.status, ATT_ST_DRAIN);
    }
    __syncwarp();
  }
  const bool has_result = ok && !skip;
  if (!has_result && lane == 0) {
    *abort_flag = 1;
    report_status(p.status);
  }

  // ---- this warp's partial result: O into its own ring, row maxima and sums beside it ----------
  float* ml = reinterpret_cast<float*>(smem + L::ML_OFF);          // [2][DEC_WARPS][ROWS]
  float* cta_ml = reinterpret_cast<float*>(smem + L::CTA_ML_OFF);  // [2][ROWS]
  float* ow = reinterpret_cast<float*>(smem + warp * L::RING_BYTES);
  __syncwarp();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = 8 * n + 2 * t4 + c;
      float l = l_run[n][c], low = low_run[n][c];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, w);
        low += __shfl_xor_sync(0xffffffffu, low, w);
      }
      if (g8 == 0) {
        ml[warp * L::ROWS + r] = m_run[n][c];
        ml[(DEC_WARPS + warp) * L::ROWS + r] = l;
      }
      if (has_result && r0 + r < rows)
#pragma unroll
        for (int m = 0; m < MTILES; ++m)  // columns 2 m, 2 m + 1 of this lane's D / 8
          *reinterpret_cast<float2*>(ow + r * D + g8 * (D / 8) + 2 * m) =
              make_float2(fmaf(o[m][n][c], 0x1p24f, low), fmaf(o[m][n][2 + c], 0x1p20f, low));
    }
  __syncthreads();
  bool whole = true;  // every warp (below: of the cluster) has a result; else nothing is written
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) whole = whole && no_result[w] == 0;

  auto emit = [&](int r, int c4, float4 acc, float mx, float l) {
    const int s = (r0 + r) / group, h = h0 + (r0 + r) % group;
    const float inv = l > 0.0f ? __fdividef(1.0f, l) : l == l ? 0.0f : l;
    if (whole) {
      uint2 v;
      v.x = pack16<BF16>(acc.x * inv, acc.y * inv);
      v.y = pack16<BF16>(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + b * p.o_stride_b + s * p.o_stride_s +
                                h * p.o_stride_h + 4 * c4) = v;
      if (p.lse && c4 == 0)
        p.lse[b * p.lse_stride_b + h * p.lse_stride_h + s] =
            l == 0.0f ? -INFINITY : (mx + log2f(l)) * 0.6931471805599453f;
    }
  };
  // sum of n partial results of one row: weights 2^(m_i - max m), 0 for an empty part
  const int live_rows = min(L::ROWS, rows - r0);
  float* o0 = reinterpret_cast<float*>(smem);
  for (int idx = threadIdx.x; idx < live_rows * (D / 4); idx += DEC_THREADS) {
    const int r = idx / (D / 4), c4 = idx % (D / 4);
    float mx = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < DEC_WARPS; ++w) mx = fmaxf(mx, ml[w * L::ROWS + r]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < DEC_WARPS; ++w) {
      const float f = fast_exp2(ml[w * L::ROWS + r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(smem + w * L::RING_BYTES) + r * D + 4 * c4);
      l = fmaf(f, ml[(DEC_WARPS + w) * L::ROWS + r], l);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
    if (nsplit == 1) {
      emit(r, c4, acc, mx, l);
    } else {
      *reinterpret_cast<float4*>(o0 + r * D + 4 * c4) = acc;  // this thread's own element
      if (c4 == 0) {
        cta_ml[r] = mx;
        cta_ml[L::ROWS + r] = l;
      }
    }
  }
  if (nsplit == 1) return;
  if (threadIdx.x == 0) no_result[DEC_WARPS] = whole ? 0 : 1;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  whole = __all_sync(0xffffffffu, lane >= nsplit || cluster.map_shared_rank(no_result, lane)[DEC_WARPS] == 0);
  for (int idx = split * DEC_THREADS + threadIdx.x; idx < live_rows * (D / 4); idx += nsplit * DEC_THREADS) {
    const int r = idx / (D / 4), c4 = idx % (D / 4);
    float mx = -INFINITY, l = 0.0f;
    for (int k = 0; k < nsplit; ++k) mx = fmaxf(mx, cluster.map_shared_rank(cta_ml, k)[r]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < nsplit; ++k) {
      const float* kml = cluster.map_shared_rank(cta_ml, k);
      const float f = fast_exp2(kml[r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(o0, k) + r * D + 4 * c4);
      l = fmaf(f, kml[L::ROWS + r], l);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
    emit(r, c4, acc, mx, l);
  }
  cluster.sync();  // no CTA leaves while another one reads its shared memory
}

// CTAs that share the keys of one row tile: as many as give every CTA slot of the chip work and leave a warp
// two tiles at least.
inline int paged4_splits(int64_t keys, int64_t units) {
  const int64_t slots = static_cast<int64_t>(sm_count_of_current_device()) * P4_CTAS_PER_SM;
  const int64_t tiles = (keys + P4_KEYS - 1) / P4_KEYS;
  int n = 1;
  while (n < DEC_MAX_SPLIT && units * 2 * n <= slots && tiles >= 2 * n * DEC_WARPS * 2) n *= 2;
  return n;
}

template <int D, bool BF16, int NT>
static int launch_paged4(const Paged4Params& p, cudaStream_t stream) {
  using L = P4Smem<D, NT>;
  auto kernel = attn_paged4_kernel<D, BF16, NT>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TRX_ERR_CUDA;
  const bool cacheable = dev >= 0 && dev < 64;
  if (!cacheable || !configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return TRX_ERR_CUDA;
    if (cacheable) configured[dev].store(true, std::memory_order_release);
  }
  const int64_t units = static_cast<int64_t>(p.Hq / p.group) *
                        ((static_cast<int64_t>(p.group) * p.Sq + L::ROWS - 1) / L::ROWS);
  int64_t keys = p.Sk;
  if (p.win_left >= 0 && static_cast<int64_t>(p.Sq) + p.win_left < keys) keys = p.Sq + p.win_left;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  const unsigned n = static_cast<unsigned>(paged4_splits(keys, units * p.B));
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(n, static_cast<unsigned>(units), static_cast<unsigned>(p.B));
  cfg.blockDim = dim3(DEC_THREADS);
  cfg.dynamicSmemBytes = L::DYN_BYTES;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

static int launch_paged4_rows(const Paged4Params& p, int64_t D, cudaStream_t s) {
  auto launch = [&](auto dim, auto bf16) {
    constexpr int DIM = decltype(dim)::value;
    constexpr bool BF = decltype(bf16)::value;
    return p.group * p.Sq > 8 ? launch_paged4<DIM, BF, 2>(p, s) : launch_paged4<DIM, BF, 1>(p, s);
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (D == 128) return p.is_bf16 ? launch(D128{}, std::true_type{}) : launch(D128{}, std::false_type{});
  return p.is_bf16 ? launch(D64{}, std::true_type{}) : launch(D64{}, std::false_type{});
}

}  // namespace trx
