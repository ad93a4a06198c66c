// Attention over packed sequences of different lengths: launches and C entry. The kernels are those of
// attention_plain.cuh and, for few rows, attention_decode.cuh in their packed form.
#include "attention_decode.cuh"
#include "attention_plain.cuh"

namespace trx {

using PackedParams = RaggedParamsOf<ATT_PACKED>;

template <int D, bool BF16, int BIAS, bool SINGLE, class P>
static int launch_packed(const P& p, dim3 grid, cudaStream_t stream) {
  const int rc = configure_plain<D, BF16, BIAS, SINGLE, P>();
  if (rc != TRX_OK) return rc;
  attn_plain_kernel<D, BF16, BIAS, SINGLE, P>
      <<<grid, AP_THREADS, plain_smem_bytes<D, SINGLE, P>(), stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

template <int D, bool BF16, bool SINGLE, class P>
static int launch_packed_bias(const P& p, dim3 grid, cudaStream_t stream) {
  // a score carries the ramp divided by the scale: not of one that is negative, or next to nothing
  if (!(p.scale_log2 > 1e-30f)) return launch_packed<D, BF16, AP_GENERAL, SINGLE>(p, grid, stream);
  if (!p.slopes) return launch_packed<D, BF16, AP_NONE, SINGLE>(p, grid, stream);
  // under a causal mask, or a window that ends at the query, every visible key is at or before it
  return p.causal || p.win_right == 0 ? launch_packed<D, BF16, AP_RAMP, SINGLE>(p, grid, stream)
                                      : launch_packed<D, BF16, AP_GENERAL, SINGLE>(p, grid, stream);
}

template <int D, bool BF16>
static int launch_packed_items(PackedParams& p, cudaStream_t stream) {
  // slots: see RaggedCursor
  const int64_t slots = p.rows / (ATT_NQ * p.tile_tokens) + static_cast<int64_t>(p.n_seq);
  p.slots_first = slots > 65535 ? 1 : 0;
  const unsigned heads = p.head_tiles, n = static_cast<unsigned>(slots);
  const dim3 grid = p.slots_first ? dim3(n, heads) : dim3(heads, n);
  if (slots * heads <= sm_count_of_current_device()) return launch_packed_bias<D, BF16, true>(p, grid, stream);
  if (p.n_seq > RAGGED_TABLE) return launch_packed_bias<D, BF16, false>(p, grid, stream);
  if (slots * heads >= (1ll << 31)) return TRX_ERR_SHAPE;
  // sequences that fit one Q tile take two tiles of heads at a time, where they are most of the sequences
  if (heads % 2 == 0 && static_cast<int64_t>(p.n_cu) * p.tile_tokens >= p.rows) {
    RaggedParamsOf<ATT_PACKED, true> alt;
    static_cast<RaggedParams&>(alt) = p;
    return launch_packed_bias<D, BF16, false>(alt, dim3(n * heads), stream);
  }
  return launch_packed_bias<D, BF16, false>(p, dim3(n * heads), stream);
}

}  // namespace trx

using namespace trx;

extern "C" int trx_attn_fwd_packed(const void* q, const void* k, const void* v, void* out,
                                   float* lse_or_null, const float* slopes_or_null, const int32_t* cu_q,
                                   const int32_t* cu_k, int64_t n_seq, int64_t Tq, int64_t Tk, int64_t Hq,
                                   int64_t Hk, int64_t D, const int64_t q_strides[2],
                                   const int64_t k_strides[2], const int64_t v_strides[2],
                                   const int64_t o_strides[2], float scale, int causal,
                                   int64_t window_left, int64_t window_right, int64_t max_sq, int zero_rest,
                                   int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != TRX_BF16 && dtype != TRX_F16) return TRX_ERR_DTYPE;
  if (n_seq < 0 || Tq < 0 || Tk < 0 || Hq <= 0 || Hk <= 0 || D <= 0 || max_sq < 0) return TRX_ERR_SHAPE;
  if (Hq % Hk != 0) return TRX_ERR_SHAPE;
  if (D != 64 && D != 128) return TRX_ERR_UNSUPPORTED;
  if ((window_left < 0) != (window_right < 0)) return TRX_ERR_SHAPE;
  if (Tq == 0 || (n_seq == 0 && !zero_rest)) return TRX_OK;
  if (!q || !out || !cu_q || !cu_k || !q_strides || !k_strides || !v_strides || !o_strides)
    return TRX_ERR_NULL_POINTER;
  if (Tk > 0 && (!k || !v)) return TRX_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < trx_attn_workspace_bytes() || !aligned_to(workspace, 16))
    return TRX_ERR_WORKSPACE;
  if (Tq >= (1ll << 30) || Tk >= (1ll << 30) || n_seq >= (1ll << 24) || Hq > 65535) return TRX_ERR_SHAPE;
  if (!aligned_to(cu_q, 4) || !aligned_to(cu_k, 4)) return TRX_ERR_ALIGNMENT;
  // (a dim of size 1 may carry any stride)
  if (!aligned_to(out, 16) || (Tq > 1 && o_strides[0] % 8) || (Hq > 1 && o_strides[1] % 8)) return TRX_ERR_ALIGNMENT;
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] < 0 || k_strides[i] < 0 || v_strides[i] < 0 || o_strides[i] < 0) return TRX_ERR_STRIDE;

  PackedParams p{};
  const int is_bf16 = dtype == TRX_BF16;
  p.Hq = static_cast<int>(Hq);
  p.group = static_cast<int>(Hq / Hk);
  choose_tile(p, 0);  // blocks of rows may run along the grid's other dimension
  int rc = make_ragged_q_map(&p.tm_q, q, is_bf16, D, Tq, Hq, 1, 0, q_strides[0], q_strides[1], p.tile_heads,
                             p.tile_tokens);
  if (rc != TRX_OK) return rc;
  // few rows: see use_decode in attention_decode.cuh
  const int64_t row_tiles = (p.group * max_sq + 15) / 16;
  const bool decode = max_sq > 0 && max_sq <= 16 && n_seq > 0 && n_seq < 65535 && Hk * row_tiles <= 65535;
  const int box = decode ? DEC_KEYS : ATT_BN;
  rc = make_ragged_kv_map(&p.tm_k, k, q, is_bf16, D, Tk, Hk, 1, 0, k_strides[0], k_strides[1], box);
  if (rc != TRX_OK) return rc;
  rc = make_ragged_kv_map(&p.tm_v, v, q, is_bf16, D, Tk, Hk, 1, 0, v_strides[0], v_strides[1], box);
  if (rc != TRX_OK) return rc;
  p.out = out;
  p.lse = lse_or_null;
  p.slopes = slopes_or_null;
  p.status = reinterpret_cast<unsigned int*>(workspace);
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.n_cu = static_cast<int>(n_seq);
  p.n_seq = p.n_cu + (zero_rest ? 1 : 0);
  p.rows = static_cast<int>(Tq);
  p.keys = static_cast<int>(Tk);
  p.o_stride_s = o_strides[0];
  p.o_stride_h = o_strides[1];
  p.lse_stride_h = Tq;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = causal ? 1 : 0;
  p.win_left = window_left < 0 ? -1 : static_cast<int>(window_left > (1ll << 29) ? (1ll << 29) : window_left);
  p.win_right = window_right < 0 ? -1 : static_cast<int>(window_right > (1ll << 29) ? (1ll << 29) : window_right);
  p.is_bf16 = is_bf16;
  // ALiBi under a causal mask: backwards, see attention_plain.cuh
  p.reverse_kv = (slopes_or_null != nullptr && (causal || window_right == 0)) ? 1 : 0;

  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (decode) {
    p.q = q;
    p.q_stride_s = q_strides[0];
    p.q_stride_h = q_strides[1];
    p.k_hdiv = p.v_hdiv = p.group;
    p.B = p.n_seq;
    p.Sq = static_cast<int>(max_sq);
    p.Sk = static_cast<int>((Tk + n_seq - 1) / n_seq);
    return launch_decode_rows(p, D, s);
  }
  if (D == 128)
    return is_bf16 ? launch_packed_items<128, true>(p, s) : launch_packed_items<128, false>(p, s);
  return is_bf16 ? launch_packed_items<64, true>(p, s) : launch_packed_items<64, false>(p, s);
}
