// Attention over the pages of a cache: the C entry, and the launches of its two kernels, for a cache of 16 bits
// (attention_decode.cuh, ATT_PAGED) and of 4 (attention_paged4.cuh).
#include "attention_paged4.cuh"

namespace trx {
int make_paged_cache(PagedCache* c, const void* k_pages, const void* v_pages, const float* k_scales,
                     const float* v_scales, const int32_t* block_table, int64_t n_seq, int64_t Hk, int64_t D,
                     int64_t pages, int64_t page_size, int64_t width, const int64_t* strides);
}  // namespace trx

using namespace trx;

extern "C" int trx_attn_fwd_paged(const void* q, const void* k_pages, const void* v_pages,
                                  const float* k_scales_or_null, const float* v_scales_or_null, void* out,
                                  float* lse_or_null, const float* slopes_or_null, const int32_t* block_table,
                                  const int32_t* lengths, int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D,
                                  int64_t pages, int64_t page_size, int64_t width, const int64_t strides[17],
                                  float scale, int64_t window_left, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (dtype != TRX_BF16 && dtype != TRX_F16) return TRX_ERR_DTYPE;
  if (!strides) return TRX_ERR_NULL_POINTER;
  if (B < 0 || Sq < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk != 0) return TRX_ERR_SHAPE;
  Paged4Params p{};
  int rc = make_paged_cache(&p.c, k_pages, v_pages, k_scales_or_null, v_scales_or_null, block_table, B, Hk, D, pages,
                            page_size, width, strides + 6);
  if (rc != TRX_OK) return rc;
  if (!(scale == scale) || scale > 1e30f || scale < -1e30f) return TRX_ERR_UNSUPPORTED;
  if (B == 0 || Sq == 0) return TRX_OK;
  if (!q || !out || !lengths) return TRX_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < trx_attn_workspace_bytes() || !aligned_to(workspace, 16))
    return TRX_ERR_WORKSPACE;
  if (pages == 0 || B > 65535 || Sq >= (1ll << 28) || Hq > 65535 || Sq * (Hq / Hk) >= (1ll << 28))
    return TRX_ERR_SHAPE;
  p.group = static_cast<int>(Hq / Hk);
  // the grid's second dimension: kv heads times tiles of 8 rows at least
  if (Hk * ((Sq * p.group + 7) / 8) > 65535) return TRX_ERR_SHAPE;
  if (!aligned_to(q, 16) || !aligned_to(out, 16) || !aligned_to(lengths, 4)) return TRX_ERR_ALIGNMENT;
  for (int i = 0; i < 6; ++i) {
    if (strides[i] < 0) return TRX_ERR_STRIDE;
    if (strides[i] % 8) return TRX_ERR_ALIGNMENT;
  }
  p.q = q;
  p.q_stride_b = strides[0];
  p.q_stride_s = strides[1];
  p.q_stride_h = strides[2];
  p.out = out;
  p.o_stride_b = strides[3];
  p.o_stride_s = strides[4];
  p.o_stride_h = strides[5];
  p.lse = lse_or_null;
  p.lse_stride_b = Hq * Sq;
  p.lse_stride_h = Sq;
  p.slopes = slopes_or_null;
  p.status = reinterpret_cast<unsigned int*>(workspace);
  p.lengths = lengths;
  p.B = static_cast<int>(B);
  p.Sq = p.seq = static_cast<int>(Sq);
  p.Hq = static_cast<int>(Hq);
  p.Sk = p.keys = static_cast<int>(width * page_size);
  p.k_hdiv = p.v_hdiv = p.group;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = 1;
  p.win_left = window_left < 0 ? -1 : static_cast<int>(window_left > (1ll << 29) ? (1ll << 29) : window_left);
  p.win_right = -1;
  p.is_bf16 = dtype == TRX_BF16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.c.k_scales) return launch_paged4_rows(p, D, s);
  const PagedCache& c = p.c;
  rc = make_map(&p.tm_k, k_pages, p.is_bf16, D, page_size, Hk, pages, c.kp[0], c.kp[2], c.kp[1], DEC_KEYS);
  if (rc != TRX_OK) return rc;
  rc = make_map(&p.tm_v, v_pages, p.is_bf16, D, page_size, Hk, pages, c.vp[0], c.vp[2], c.vp[1], DEC_KEYS);
  if (rc != TRX_OK) return rc;
  return launch_decode_rows(static_cast<const PagedAttnParams&>(p), D, s);
}
