// Host side of attention without a dense mask or dropout over one batch (the kernel: attention_plain.cuh).
#include "attention_plain.cuh"

namespace trx {

template <int D, bool BF16, int BIAS, bool SINGLE>
static int launch_plain(const AttnParams& p, cudaStream_t stream) {
  const int rc = configure_plain<D, BF16, BIAS, SINGLE, AttnParams>();
  if (rc != TRX_OK) return rc;
  const int rows = p.pair_heads ? ATT_BM : ATT_NQ * ATT_BM;
  const unsigned m = (p.Sq + rows - 1) / rows, h = p.pair_heads ? p.Hq / 2 : p.Hq, b = p.B;
  const dim3 grid = p.order == AP_MHB ? dim3(m, h, b) : p.order == AP_HMB ? dim3(h, m, b) : dim3(h, b, m);
  attn_plain_kernel<D, BF16, BIAS, SINGLE, AttnParams><<<grid, AP_THREADS, PlainSmem<D>::DYN_BYTES, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

template <int D, bool BF16, bool SINGLE>
static int launch_plain_bias(const AttnParams& p, cudaStream_t stream) {
  if (!(p.scale_log2 > 0.0f)) return launch_plain<D, BF16, AP_GENERAL, SINGLE>(p, stream);
  if (!p.slopes) return launch_plain<D, BF16, AP_NONE, SINGLE>(p, stream);
  // under a causal mask, or a window that ends at the query, every visible key is at or before it
  return p.causal || p.win_right == 0 ? launch_plain<D, BF16, AP_RAMP, SINGLE>(p, stream)
                                      : launch_plain<D, BF16, AP_GENERAL, SINGLE>(p, stream);
}

template <int D, bool BF16>
static int launch_plain_items(const AttnParams& p, bool single, cudaStream_t stream) {
  return single ? launch_plain_bias<D, BF16, true>(p, stream)
                : launch_plain_bias<D, BF16, false>(p, stream);
}

int launch_attn_plain(AttnParams& p, int64_t D, cudaStream_t stream) {
  const int rows = p.pair_heads ? ATT_BM : ATT_NQ * ATT_BM;
  const int64_t m = (p.Sq + rows - 1) / rows, h = p.pair_heads ? p.Hq / 2 : p.Hq;
  const bool single = m * h * p.B <= sm_count_of_current_device();
  p.order = AP_MHB;
  if (p.causal && m <= 65535) {
    // Heaviest row blocks first: over all heads of all batches while their keys and values are a third
    // of L2, over those of one batch up to 100 MB. One head after the other / one batch / all, us:
    // 4 x 2048, 32 / 8 heads x 128 (34 MB) 158 / 147 / 144, 2 x 4096 (34 MB) 269 / 248 / 248, 8 x 2048
    // (67 MB) 292 / 286 / 288, 16 x 4096 (268 MB, 17 of a batch) 2174 / 2166 / 2374. The upper line is
    // not fitted: 1 x 8192, 32 / 32 heads (134 MB) takes 546 / 490 / 489, 1 x 6144 (101 MB) 334 / 286 / 285.
    const double kv = 4.0 * p.Sk * static_cast<double>(D) * p.Hq / p.group;  // bytes of a batch
    if (kv * p.B <= 40e6) p.order = AP_HBM;
    else if (kv <= 100e6) p.order = AP_HMB;
  }
  if (D == 128)
    return p.is_bf16 ? launch_plain_items<128, true>(p, single, stream)
                     : launch_plain_items<128, false>(p, single, stream);
  return p.is_bf16 ? launch_plain_items<64, true>(p, single, stream)
                   : launch_plain_items<64, false>(p, single, stream);
}

}  // namespace trx
