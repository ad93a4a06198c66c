// Into and out of a paged cache of keys and values (paged_cache.cuh): appending new tokens, with the rotation of
// their keys (and queries) on the way, and reading sequences back as packed rows.
//
// Both are copies: what counts is that every row is read and written once, in 16-byte pieces, and that nothing
// is launched around it (decoding appends one token to each sequence, a few KB in all). A few lanes hold a row
// (head_rows.cuh), which makes the smallest and largest value of a 4-bit row three shuffles each.
// Measured (32 / 8 heads x 128): 64 tokens with their queries 3.5 us, a launch; prompts of 16 sequences (204 MB read
// and written, queries among them) 34.2 us, 6.0 TB/s; 2048 new tokens into a 4-bit cache and 42 thousand read back
// (230 MB) 50.6 us: the first 9 us of it, four look-ups one after the other (bounds, length, page, angles) before a
// row can be written, reading back 5.4 TB/s of mostly writes. 30 thousand rows read back from 16 bits (249 MB) 41.7 us,
// 6.0 TB/s.
#include "head_rows.cuh"
#include "paged_cache.cuh"

namespace trx {

constexpr int PC_THREADS = 128;
constexpr int PC_ROWS = 4;  // heads of a token to a thread, all in flight
constexpr float PC_LEAST_SPAN = 0x1p-76f, PC_MOST_SPAN = 0x1p120f;

struct AppendParams {
  PagedCache c;
  const void* q;  // null: none
  const void* k;
  const void* v;
  void* qo;
  int64_t qs[3], ks[3], vs[3], os[3];  // (sequence, token, head) strides; packed: sequence 0
  const int* lengths;                  // with the new tokens
  const int* cu;                       // packed: first rows; null: S tokens of every sequence
  const void* cos_t;                   // null: no rotation
  const void* sin_t;
  int64_t table_rows, angle_stride;
  int64_t tokens, S;
  int n_seq, Hq, Hk, D, table_dtype;
  int q_chunks, k_chunks;
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Eight codes of a row: rint of the IEEE quotient 15 (x - low) / span. Two FMAs with reciprocals below and above
// 1 / span round to the same integer nearly always, and then the quotient does, too (quant_pair_bracketed); the
// others, a value halfway between two codes among them, are divided.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float low, float span, float lo, float hi) {
  constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23
  uint32_t word = 0, differ = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __fmul_rn(__fsub_rn(x[i], low), 15.0f);
    const uint32_t a = __float_as_uint(fmaf(t, lo, MAGIC)), b = __float_as_uint(fmaf(t, hi, MAGIC));
    differ |= a ^ b;
    word |= (a & 15u) << (4 * i);
  }
  if (differ) {
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = __fmul_rn(__fsub_rn(x[i], low), 15.0f);
      word |= static_cast<uint32_t>(rintf(__fdiv_rn(t, span))) << (4 * i);
    }
  }
  return word;
}

template <typename T, int LPR, bool FOUR>
__global__ void __launch_bounds__(PC_THREADS) paged_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int HALF = 8 * LPR;
  const int lane = threadIdx.x % LPR;
  int64_t token = static_cast<int64_t>(blockIdx.x) * (PC_THREADS / LPR) + threadIdx.x / LPR;
  const bool live = token < p.tokens;
  if (!live) token = p.tokens - 1;  // its lanes take part in the shuffles
  // which heads, of which of the three
  int chunk = blockIdx.y, H = p.Hq;
  enum { Q, K, V } what = Q;
  if (chunk >= p.q_chunks) {
    chunk -= p.q_chunks;
    what = K;
    H = p.Hk;
    if (chunk >= p.k_chunks) {
      chunk -= p.k_chunks;
      what = V;
    }
  }
  int64_t b = 0, s = token;
  if (!p.cu) {
    b = token / p.S;
    s = token - b * p.S;
  }
  const int64_t seq = b;
  const int64_t* st = what == Q ? p.qs : what == K ? p.ks : p.vs;
  const T* x = static_cast<const T*>(what == Q ? p.q : what == K ? p.k : p.v) + seq * st[0] + s * st[1];
  const int h0 = chunk * PC_ROWS;
  HalfRow<T, 8, 1> r1[PC_ROWS], r2[PC_ROWS];
#pragma unroll
  for (int u = 0; u < PC_ROWS; ++u) {  // on their way while the place is looked up
    const T* row = x + min(h0 + u, H - 1) * st[2];
    r1[u].template load<LPR>(row, lane, HALF);
    r2[u].template load<LPR>(row + HALF, lane, HALF);
  }

  // its sequence, its place there and in the inputs
  int64_t pos;
  if (p.cu) {
    const int row = static_cast<int>(token);
    b = sequence_of(p.cu, p.n_seq, row);
    const int end = __ldg(p.cu + b + 1);
    pos = row < end && row >= __ldg(p.cu + b) ? static_cast<int64_t>(__ldg(p.lengths + b)) - end + row : -1;
  } else {
    pos = __ldg(p.lengths + b) - p.S + s;
  }
  if (p.cos_t && pos >= p.table_rows) pos = -1;
  const int at = pos < 0 || pos > 0x7fffffff ? -1 : static_cast<int>(pos);
  const int page = page_of(p.c, b, at), slot = at < 0 ? 0 : at % p.c.page_size;

  const bool turned = p.cos_t && what != V && page >= 0;
  float c[8], sn[8];
  if (turned) {
    load_columns<8, 1, LPR>(p.cos_t, p.table_dtype, at * p.angle_stride, lane, HALF, 0.0f, c);
    load_columns<8, 1, LPR>(p.sin_t, p.table_dtype, at * p.angle_stride, lane, HALF, 0.0f, sn);
  }
  const int64_t* ps = what == K ? p.c.kp : p.c.vp;
#pragma unroll
  for (int u = 0; u < PC_ROWS; ++u) {
    const int h = h0 + u;
    float x1[8], x2[8];
    r1[u].unpack(x1);
    r2[u].unpack(x2);
    if (turned) turn(x1, x2, c, sn);
    if (what == Q) {
      if (live && h < H) {
        T* row = static_cast<T*>(p.qo) + seq * p.os[0] + s * p.os[1] + h * p.os[2];
        if (page < 0)  // a token without a place
#pragma unroll
          for (int i = 0; i < 8; ++i) x1[i] = x2[i] = 0.0f;
        store_half<T, 8, 1, LPR>(row, lane, HALF, x1);
        store_half<T, 8, 1, LPR>(row + HALF, lane, HALF, x2);
      }
      continue;
    }
    const bool store = live && h < H && page >= 0;
    if constexpr (!FOUR) {
      if (store) {
        T* row = static_cast<T*>(what == K ? p.c.k : p.c.v) + page * ps[0] + h * ps[1] + slot * ps[2];
        store_half<T, 8, 1, LPR>(row, lane, HALF, x1);
        store_half<T, 8, 1, LPR>(row + HALF, lane, HALF, x2);
      }
    } else {
      float low = x1[0], high = x1[0];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        low = min_nan(low, min_nan(x1[i], x2[i]));
        high = max_nan(high, max_nan(x1[i], x2[i]));
      }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) {
        low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
      }
      const float span = __fsub_rn(high, low);
      float step = __fmul_rn(span, 1.0f / 15.0f);
      uint32_t word1 = 0u, word2 = 0u;
      if (span >= PC_LEAST_SPAN && span <= PC_MOST_SPAN) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(span));
        const float lo = __fmul_rn(r, 1.0f - 0x1p-21f), hi = __fmul_rn(r, 1.0f + 0x1p-21f);
        word1 = codes_of(x1, low, span, lo, hi);
        word2 = codes_of(x2, low, span, lo, hi);
      } else if (span < PC_LEAST_SPAN) {  // one value
        step = 0.0f;
      } else {  // infinite, not a number, or beyond what 15 (x - low) holds: the row is not a number
        step = low = __int_as_float(0x7fffffff);
      }
      if (store) {
        uint8_t* row = static_cast<uint8_t*>(what == K ? p.c.k : p.c.v) + page * ps[0] + h * ps[1] + slot * ps[2];
        st_stream4(row + 4 * lane, word1);
        st_stream4(row + HALF / 2 + 4 * lane, word2);
        if (lane == 0) {
          const int64_t* ss = what == K ? p.c.ksp : p.c.vsp;
          float* scale = (what == K ? p.c.k_scales : p.c.v_scales) + page * ss[0] + h * ss[1] + 2 * slot;
          *reinterpret_cast<float2*>(scale) = make_float2(step, low);
        }
      }
    }
  }
}

struct GatherParams {
  PagedCache c;
  void* ko;  // (rows, Hk, D)
  void* vo;
  const int* cu;
  int64_t rows;
  int n_seq, Hk, zero_rest;
};

// What a word of eight codes stands for, in T: code * step and the sum with lowest apart, as the elementwise formula
// rounds them (a packed product and sum would become one rounding). A code goes into the low byte of 2^23;
// (2^23 + code) * step - 2^23 * step, rounded once, is code * step, rounded once, where 2^23 * step is finite.
template <typename T>
__device__ __forceinline__ uint4 values_of(uint32_t word, float2 scale) {
  const uint32_t even = word & 0x0F0F0F0Fu, odd = (word >> 4) & 0x0F0F0F0Fu;
  const float2 step = make_float2(scale.x, scale.x), low = make_float2(scale.y, scale.y);
  const float2 minus = make_float2(-8388608.0f * scale.x, -8388608.0f * scale.x);
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 code = make_float2(__uint_as_float(__byte_perm(even, 0x4B000000u, 0x7650 + i)),
                                    __uint_as_float(__byte_perm(odd, 0x4B000000u, 0x7650 + i)));
    const float2 v = add2(low, fma2(code, step, minus));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
  if (scale.x >= 0x1p100f)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = __fadd_rn(scale.y, __fmul_rn(static_cast<float>((word >> (4 * i)) & 15u), scale.x));
  return Pack<T>::pack(f);
}

// Grid (rows, chunks of heads): a thread has its columns of all the chunk's heads of a row of K and of V.
template <typename T, int LPR, bool FOUR>
__global__ void __launch_bounds__(PC_THREADS) paged_gather_kernel(const __grid_constant__ GatherParams p) {
  constexpr int HALF = 8 * LPR;
  const int lane = threadIdx.x % LPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (PC_THREADS / LPR) + threadIdx.x / LPR;
  if (row >= p.rows) return;
  const int b = sequence_of(p.cu, p.n_seq, static_cast<int>(row));
  const int first = p.n_seq ? __ldg(p.cu + b) : 0, end = p.n_seq ? __ldg(p.cu + b + 1) : 0;
  const bool there = row >= first && row < end;
  if (!there && !p.zero_rest) return;
  const int at = static_cast<int>(row) - first;
  const int page = there ? page_of(p.c, b, at) : -1, slot = there ? at % p.c.page_size : 0;
  const int h0 = blockIdx.y * PC_ROWS;
  constexpr int BYTES = FOUR ? 1 : static_cast<int>(sizeof(T));
  // K's and V's loads all before the first store
  uint4 y1[2][PC_ROWS], y2[2][PC_ROWS];
  uint32_t w1[2][PC_ROWS], w2[2][PC_ROWS];
  float2 scale[2][PC_ROWS];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const int64_t* ps = kv ? p.c.vp : p.c.kp;
    const int64_t* ss = kv ? p.c.vsp : p.c.ksp;
    const uint8_t* src = static_cast<const uint8_t*>(kv ? p.c.v : p.c.k) + (page * ps[0] + slot * ps[2]) * BYTES +
                         (FOUR ? 4 : 16) * lane;
    const float* scales = (kv ? p.c.v_scales : p.c.k_scales) + page * ss[0] + 2 * slot;
#pragma unroll
    for (int u = 0; u < PC_ROWS; ++u) {
      const int h = min(h0 + u, p.Hk - 1);
      y1[kv][u] = y2[kv][u] = make_uint4(0u, 0u, 0u, 0u);
      w1[kv][u] = w2[kv][u] = 0u;
      scale[kv][u] = make_float2(0.0f, 0.0f);
      if (page < 0) continue;
      const uint8_t* from = src + h * ps[1] * BYTES;
      if constexpr (FOUR) {
        w1[kv][u] = __ldg(reinterpret_cast<const uint32_t*>(from));
        w2[kv][u] = __ldg(reinterpret_cast<const uint32_t*>(from + HALF / 2));
        scale[kv][u] = __ldg(reinterpret_cast<const float2*>(scales + h * ss[1]));
      } else {
        y1[kv][u] = ld_stream16(from);
        y2[kv][u] = ld_stream16(from + 2 * HALF);
      }
    }
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    T* out = static_cast<T*>(kv ? p.vo : p.ko) + row * p.Hk * (2 * HALF) + 8 * lane;
#pragma unroll
    for (int u = 0; u < PC_ROWS; ++u) {
      if (h0 + u >= p.Hk) break;
      if constexpr (FOUR) {  // (no page: codes, step and lowest of 0)
        y1[kv][u] = values_of<T>(w1[kv][u], scale[kv][u]);
        y2[kv][u] = values_of<T>(w2[kv][u], scale[kv][u]);
      }
      st_stream16(out + (h0 + u) * (2 * HALF), y1[kv][u]);
      st_stream16(out + (h0 + u) * (2 * HALF) + HALF, y2[kv][u]);
    }
  }
}

// Four heads of a token to a thread, whatever the sizes: eight, two after the other, for fewer look-ups of the place
// are 34.9 us instead of 34.7 (prompts of 16 sequences, 32 / 8 heads x 128, 16 bits) and 53.3 instead of 50.2 (256
// tokens behind up to 16384 in 4 bits, and all read back).
static unsigned chunks_of(int64_t heads) { return static_cast<unsigned>((heads + PC_ROWS - 1) / PC_ROWS); }

template <typename T, int LPR>
static int launch_append(AppendParams& p, cudaStream_t s) {
  const int64_t blocks = (p.tokens + PC_THREADS / LPR - 1) / (PC_THREADS / LPR);
  p.q_chunks = chunks_of(p.Hq);
  p.k_chunks = chunks_of(p.Hk);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(p.q_chunks + 2 * p.k_chunks));
  if (p.c.k_scales) paged_append_kernel<T, LPR, true><<<grid, PC_THREADS, 0, s>>>(p);
  else paged_append_kernel<T, LPR, false><<<grid, PC_THREADS, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}
template <typename T, int LPR>
static int launch_gather(GatherParams& p, cudaStream_t s) {
  const int64_t blocks = (p.rows + PC_THREADS / LPR - 1) / (PC_THREADS / LPR);
  const dim3 grid(static_cast<unsigned>(blocks), chunks_of(p.Hk));
  if (p.c.k_scales) paged_gather_kernel<T, LPR, true><<<grid, PC_THREADS, 0, s>>>(p);
  else paged_gather_kernel<T, LPR, false><<<grid, PC_THREADS, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

int make_paged_cache(PagedCache* c, const void* k_pages, const void* v_pages, const float* k_scales,
                     const float* v_scales, const int32_t* block_table, int64_t n_seq, int64_t Hk, int64_t D,
                     int64_t pages, int64_t page_size, int64_t width, const int64_t* strides) {
  if (D != 64 && D != 128) return TRX_ERR_UNSUPPORTED;
  if (n_seq < 0 || Hk <= 0 || pages < 0 || page_size <= 0 || width < 0) return TRX_ERR_SHAPE;
  if (page_size % 16) return TRX_ERR_UNSUPPORTED;
  if (Hk > 65535 || page_size > 4096 || pages > 0x7fffffff || width * page_size >= (1ll << 29) || width >= (1ll << 25))
    return TRX_ERR_SHAPE;
  if (!strides || !k_pages || !v_pages || (!block_table && n_seq * width > 0)) return TRX_ERR_NULL_POINTER;
  if (!k_scales != !v_scales) return TRX_ERR_NULL_POINTER;
  if (!aligned_to(k_pages, 16) || !aligned_to(v_pages, 16) || !aligned_to(block_table, 4) ||
      !aligned_to(k_scales, 16) || !aligned_to(v_scales, 16))
    return TRX_ERR_ALIGNMENT;
  const int64_t row = k_scales ? D / 2 : D, vec = k_scales ? 16 : 8;
  const int64_t extent[3] = {pages, Hk, page_size};  // a dim of size 1 may carry any stride
  for (int t = 0; t < 2; ++t) {
    int64_t* to = t ? c->vp : c->kp;
    for (int i = 0; i < 3; ++i) {
      to[i] = extent[i] > 1 ? strides[3 * t + i] : 0;
      if (extent[i] > 1 && to[i] < row) return TRX_ERR_STRIDE;  // rows must not share memory: they are written
      if (to[i] % vec) return TRX_ERR_ALIGNMENT;
    }
    if (k_scales && to[2] != row) return TRX_ERR_STRIDE;
    int64_t* scale = t ? c->vsp : c->ksp;
    for (int i = 0; i < 2; ++i) {
      scale[i] = k_scales && extent[i] > 1 ? strides[6 + 2 * t + i] : 0;
      if (k_scales && extent[i] > 1 && scale[i] < 2 * page_size) return TRX_ERR_STRIDE;
      if (scale[i] % 4) return TRX_ERR_ALIGNMENT;
    }
  }
  c->table_stride = strides[10];
  if (n_seq > 1 && c->table_stride < 0) return TRX_ERR_STRIDE;
  c->k = const_cast<void*>(k_pages);
  c->v = const_cast<void*>(v_pages);
  c->k_scales = const_cast<float*>(k_scales);
  c->v_scales = const_cast<float*>(v_scales);
  c->table = block_table;
  c->pages = static_cast<int>(pages);
  c->page_size = static_cast<int>(page_size);
  c->width = static_cast<int>(width);
  return TRX_OK;
}

}  // namespace trx

using namespace trx;

extern "C" int trx_paged_append(const void* q_or_null, const void* k, const void* v, void* q_out, void* k_pages,
                                void* v_pages, float* k_scales_or_null, float* v_scales_or_null,
                                const int32_t* block_table, const int32_t* lengths, const int32_t* cu_or_null,
                                const void* cos_or_null, const void* sin_or_null, int64_t n_seq, int64_t S,
                                int64_t Hq, int64_t Hk, int64_t D, int64_t pages, int64_t page_size,
                                int64_t width, const int64_t strides[23], int64_t table_rows,
                                int64_t table_row_stride, int table_dtype, int dtype, void* stream) {
  if (dtype != TRX_BF16 && dtype != TRX_F16) return TRX_ERR_DTYPE;
  if (cos_or_null && table_dtype != TRX_F32 && table_dtype != dtype) return TRX_ERR_DTYPE;
  if (!strides) return TRX_ERR_NULL_POINTER;
  if (S < 0 || Hq < 0 || Hq > 65535) return TRX_ERR_SHAPE;
  AppendParams p{};
  const int rc = make_paged_cache(&p.c, k_pages, v_pages, k_scales_or_null, v_scales_or_null, block_table, n_seq, Hk,
                                  D, pages, page_size, width, strides + 12);
  if (rc != TRX_OK) return rc;
  if (!cu_or_null && n_seq > 0 && S > ((1ll << 30) - 1) / n_seq) return TRX_ERR_SHAPE;
  if (cu_or_null && S >= (1ll << 30)) return TRX_ERR_SHAPE;
  if (n_seq >= (1ll << 30)) return TRX_ERR_SHAPE;
  p.tokens = cu_or_null ? S : n_seq * S;
  if (p.tokens == 0) return TRX_OK;
  if (!q_or_null) Hq = 0;
  if (!k || !v || (n_seq > 0 && !lengths) || (Hq > 0 && !q_out) || !cos_or_null != !sin_or_null)
    return TRX_ERR_NULL_POINTER;
  if (Hq > 0 && !cos_or_null) return TRX_ERR_NULL_POINTER;  // nothing to be done with them
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(q_or_null, 16) || (Hq > 0 && !aligned_to(q_out, 16)) ||
      !aligned_to(lengths, 4) || !aligned_to(cu_or_null, 4))
    return TRX_ERR_ALIGNMENT;
  int64_t* to[4] = {p.qs, p.ks, p.vs, p.os};
  for (int t = 0; t < 4; ++t)
    for (int i = 0; i < 3; ++i) {
      const bool unused = Hq == 0 && (t == 0 || t == 3);
      to[t][i] = unused ? 0 : strides[3 * t + i];
      if (to[t][i] < 0) return TRX_ERR_STRIDE;
      if (to[t][i] % 8) return TRX_ERR_ALIGNMENT;
    }
  if (cos_or_null) {
    if (table_rows < 0) return TRX_ERR_SHAPE;
    if (table_row_stride < D / 2) return TRX_ERR_STRIDE;
    if (!aligned_to(cos_or_null, 16) || !aligned_to(sin_or_null, 16) ||
        table_row_stride % (table_dtype == TRX_F32 ? 4 : 8))
      return TRX_ERR_ALIGNMENT;
  }
  p.q = q_or_null;
  p.k = k;
  p.v = v;
  p.qo = q_out;
  p.lengths = lengths;
  p.cu = cu_or_null;
  p.cos_t = cos_or_null;
  p.sin_t = sin_or_null;
  p.table_rows = table_rows;
  p.angle_stride = table_row_stride;
  p.table_dtype = table_dtype;
  p.S = S;
  p.n_seq = static_cast<int>(n_seq);
  p.Hq = static_cast<int>(Hq);
  p.Hk = static_cast<int>(Hk);
  p.D = static_cast<int>(D);
  if (p.cu && n_seq == 0) return Hq == 0 ? TRX_OK : TRX_ERR_SHAPE;  // rows of no sequence
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TRX_F16) return D == 128 ? launch_append<__half, 8>(p, s) : launch_append<__half, 4>(p, s);
  return D == 128 ? launch_append<__nv_bfloat16, 8>(p, s) : launch_append<__nv_bfloat16, 4>(p, s);
}

extern "C" int trx_paged_gather(const void* k_pages, const void* v_pages, const float* k_scales_or_null,
                                const float* v_scales_or_null, const int32_t* block_table, const int32_t* cu,
                                void* k_out, void* v_out, int64_t n_seq, int64_t rows, int64_t Hk, int64_t D,
                                int64_t pages, int64_t page_size, int64_t width, const int64_t strides[11],
                                int zero_rest, int dtype, void* stream) {
  if (dtype != TRX_BF16 && dtype != TRX_F16) return TRX_ERR_DTYPE;
  if (rows < 0 || rows >= (1ll << 30) || n_seq >= (1ll << 30)) return TRX_ERR_SHAPE;
  GatherParams p{};
  const int rc = make_paged_cache(&p.c, k_pages, v_pages, k_scales_or_null, v_scales_or_null, block_table, n_seq, Hk,
                                  D, pages, page_size, width, strides);
  if (rc != TRX_OK) return rc;
  if (rows == 0) return TRX_OK;
  if (!k_out || !v_out || !cu) return TRX_ERR_NULL_POINTER;
  if (!aligned_to(k_out, 16) || !aligned_to(v_out, 16) || !aligned_to(cu, 4)) return TRX_ERR_ALIGNMENT;
  p.ko = k_out;
  p.vo = v_out;
  p.cu = cu;
  p.rows = rows;
  p.n_seq = static_cast<int>(n_seq);
  p.Hk = static_cast<int>(Hk);
  p.zero_rest = zero_rest;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TRX_F16) return D == 128 ? launch_gather<__half, 8>(p, s) : launch_gather<__half, 4>(p, s);
  return D == 128 ? launch_gather<__nv_bfloat16, 8>(p, s) : launch_gather<__nv_bfloat16, 4>(p, s);
}
