// Attention for a batch whose sequences share a prefix: launches and C entries. Two ways, of which a cost
// picks one (shared_plan):
//
//   in parts   the rows of the whole batch are one run of query rows against the prefix, whose keys are split
//              over the CTAs (attention_plain.cuh, ATT_PREFIX): the prefix is read and multiplied once for
//              all, at 128 rows to a tile where a sequence alone would fill a few. The decode kernel then
//              does the sequences' own keys and merges. For few rows to a sequence, or a long prefix.
//   one pass   over the prefix's tiles and the sequence's own (ATT_SHARED): its own rows fill the tiles, and
//              the prefix comes from L2. For many rows, or a short prefix.
#include "attention_decode.cuh"
#include "attention_plain.cuh"

namespace trx {

using SharedParams = RaggedParamsOf<ATT_SHARED>;
using PrefixParams = RaggedParamsOf<ATT_PREFIX>;
using HalvesParams = RaggedParamsOf<ATT_PREFIX, true>;

template <int D, bool BF16, int BIAS, bool SINGLE, class P>
static int launch_form(const P& p, dim3 grid, cudaStream_t stream) {
  const int rc = configure_plain<D, BF16, BIAS, SINGLE, P>();
  if (rc != TRX_OK) return rc;
  attn_plain_kernel<D, BF16, BIAS, SINGLE, P><<<grid, AP_THREADS, PlainSmem<D>::DYN_BYTES, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}
template <int D, bool BF16, class P>
static int launch_form_items(const P& p, dim3 grid, cudaStream_t s) {
  // every visible key is at or before its query, the scale is positive
  if (static_cast<int64_t>(grid.x) * grid.y * grid.z <= sm_count_of_current_device())
    return p.slopes ? launch_form<D, BF16, AP_RAMP, true>(p, grid, s)
                    : launch_form<D, BF16, AP_NONE, true>(p, grid, s);
  return p.slopes ? launch_form<D, BF16, AP_RAMP, false>(p, grid, s)
                  : launch_form<D, BF16, AP_NONE, false>(p, grid, s);
}
template <class P>
static int launch_form_rows(const P& p, int64_t D, dim3 grid, cudaStream_t s) {
  if (D == 128)
    return p.is_bf16 ? launch_form_items<128, true>(p, grid, s) : launch_form_items<128, false>(p, grid, s);
  return p.is_bf16 ? launch_form_items<64, true>(p, grid, s) : launch_form_items<64, false>(p, grid, s);
}

struct SharedPlan {
  RaggedParams tile;  // tile_heads, tile_tokens, head_tiles
  bool in_parts;
  int splits, split_tiles;  // of the prefix
  bool halves;              // one Q tile holds all rows, and the two have halves of a split's keys
  int parts;                // results of the splits, or halves
};
// The cost, in us: a launch of attention_plain.cuh starts and ends in 6, an item in 4.5, a KV tile takes 1.95
// with both Q tiles at work on it, 1.5 with one, 0.95 with every second one each; the decode kernel by its
// own cost (decode_cost), more with two row tiles to a warp, 0.15 for each part that it merges. Fitted to
// 1 to 32 sequences of 4 to 160 rows behind 500 to 30000 keys with 16 / 16 heads x 64, 32 / 4 and 32 / 8 x 128.
// Over 84 shapes of six head configurations, 1 to 300 own keys, with and without ALiBi, the way that it picks is
// slower than the better one by 1 % in the mean and 27 % at worst behind 1024 and more keys (4 x 48 rows, 32 / 8
// heads x 128, behind 1024: 33.6 / 26.4 us in parts / one pass); by 21 % in the mean and 72 % at worst behind 300 and
// 500, where it takes one pass too often (8 x 1 behind 300, 16 / 16 heads x 64: 10.1 / 17.4). In parts / one pass,
// 32 / 8 heads x 128: 32 x 4 rows behind 8192 keys 38 / 202 us, 32 x 48 351 / 268, 4 x 48 53 / 113, 16 x 8 behind 1024
// 37 / 26. One pass for more than 16 rows and only then: up to 4 times as long (4 x 24 behind 8192 42 / 104).
static SharedPlan shared_plan(int64_t B, int64_t Sq, int64_t P, int64_t S, int64_t Hq, int64_t Hk) {
  SharedPlan s{};
  s.tile.Hq = static_cast<int>(Hq);
  s.tile.group = static_cast<int>(Hq / Hk);
  choose_tile(s.tile, Sq);
  const int64_t sms = sm_count_of_current_device(), tokens = s.tile.tile_tokens, step = ATT_NQ * tokens;
  const bool wide = s.tile.group * Sq > 16;
  const int64_t row_tiles = (s.tile.group * Sq + (wide ? 31 : 15)) / (wide ? 32 : 16);
  auto up = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
  if (Hk * row_tiles > 65535) return s;
  if (P == 0) {  // the sequences' own keys alone
    s.in_parts = Sq <= 16;
    return s;
  }
  const int64_t rows = B * Sq, tiles = up(P, ATT_BN), items = s.tile.head_tiles * up(rows, step);
  if (up(rows, step) > 65535) return s;  // more blocks of rows than the prefix's grid holds
  int64_t splits = sms / items;
  splits = splits < 1 ? 1 : splits > tiles ? tiles : splits;
  s.split_tiles = static_cast<int>(up(tiles, splits));
  s.splits = static_cast<int>(up(tiles, s.split_tiles));
  s.halves = rows <= tokens && s.split_tiles > 1;
  s.parts = s.halves ? 2 * s.splits : s.splits;
  const double visit = s.halves ? 0.95 : rows <= tokens ? 1.5 : 1.95;
  const int64_t units = Hk * row_tiles * B;
  const double in_parts = 6.0 + up(items * s.splits, sms) * (4.5 + visit * s.split_tiles) +
                          (wide ? 0.286 : 0.22) * decode_cost(decode_splits(S, units, wide), S, units, wide) +
                          0.15 * s.parts + 2.0;
  const double one_pass = 6.0 + up(s.tile.head_tiles * up(Sq, step) * B, sms) *
                                    (4.5 + (Sq <= tokens ? 1.5 : 1.95) * (tiles + up(S, ATT_BN)));
  s.in_parts = in_parts < one_pass;
  if (!s.in_parts) s.parts = 0;
  return s;
}

}  // namespace trx

using namespace trx;

static size_t shared_bytes(const SharedPlan& s, int64_t B, int64_t Sq, int64_t Hq, int64_t D) {
  return static_cast<size_t>(s.parts) * B * Sq * Hq * (D + 1) * sizeof(float);
}

extern "C" size_t trx_attn_shared_bytes(int64_t B, int64_t Sq, int64_t P, int64_t S, int64_t Hq, int64_t Hk,
                                        int64_t D) {
  if (B <= 0 || Sq <= 0 || P < 0 || S < 0 || Hq <= 0 || Hk <= 0 || D <= 0 || Hq % Hk || B > 65535 ||
      Sq >= (1ll << 30) || B * Sq >= (1ll << 30) || P >= (1ll << 29) || S >= (1ll << 29) || Hq > 65535)
    return 0;
  return shared_bytes(shared_plan(B, Sq, P, S, Hq, Hk), B, Sq, Hq, D);
}

extern "C" int trx_attn_fwd_shared(const void* q, const void* prefix_k, const void* prefix_v, const void* k,
                                   const void* v, void* out, float* lse_or_null, const float* slopes_or_null,
                                   const int32_t* lengths_or_null, int64_t B, int64_t Sq, int64_t P, int64_t S,
                                   int64_t Hq, int64_t Hk, int64_t D, const int64_t q_strides[3],
                                   const int64_t pk_strides[2], const int64_t pv_strides[2],
                                   const int64_t k_strides[3], const int64_t v_strides[3],
                                   const int64_t o_strides[3], float scale, int dtype, void* parts,
                                   size_t parts_bytes, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (dtype != TRX_BF16 && dtype != TRX_F16) return TRX_ERR_DTYPE;
  if (B < 0 || Sq < 0 || P < 0 || S < 0 || Hq <= 0 || Hk <= 0 || D <= 0 || Hq % Hk != 0) return TRX_ERR_SHAPE;
  if (D != 64 && D != 128) return TRX_ERR_UNSUPPORTED;
  if (!(scale >= 1e-30f)) return TRX_ERR_UNSUPPORTED;  // scores carry ALiBi's ramp divided by it
  if (B == 0 || Sq == 0) return TRX_OK;
  if (!q || !out || !q_strides || !pk_strides || !pv_strides || !k_strides || !v_strides || !o_strides)
    return TRX_ERR_NULL_POINTER;
  if ((P > 0 && (!prefix_k || !prefix_v)) || (S > 0 && (!k || !v))) return TRX_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < trx_attn_workspace_bytes() || !aligned_to(workspace, 16))
    return TRX_ERR_WORKSPACE;
  if (B > 65535 || Sq >= (1ll << 30) || B * Sq >= (1ll << 30) || P >= (1ll << 29) || S >= (1ll << 29) ||
      Hq > 65535)
    return TRX_ERR_SHAPE;
  if (lengths_or_null && !aligned_to(lengths_or_null, 4)) return TRX_ERR_ALIGNMENT;
  if (!aligned_to(out, 16) || o_strides[0] % 8 || o_strides[1] % 8 || o_strides[2] % 8)
    return TRX_ERR_ALIGNMENT;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || k_strides[i] < 0 || v_strides[i] < 0 || o_strides[i] < 0 ||
        (i < 2 && (pk_strides[i] < 0 || pv_strides[i] < 0)))
      return TRX_ERR_STRIDE;
  int64_t qb = q_strides[0], qs = q_strides[1], qh = q_strides[2];
  int rc = check_ragged_q(q, D, Sq, Hq, B, qb, qs, qh);  // whichever way is taken: one of them makes no map of q
  if (rc != TRX_OK) return rc;

  SharedPlan plan = shared_plan(B, Sq, P, S, Hq, Hk);
  // the rows of the batch as one run: what the prefix's launch wants
  const int64_t row_stride = Sq == 1 ? q_strides[0] : q_strides[1];
  if (plan.parts > 0 && B > 1 && Sq > 1 && q_strides[0] != Sq * q_strides[1]) {
    plan.in_parts = false;
    plan.parts = 0;
  }
  if (plan.parts > 0 &&
      (!parts || !aligned_to(parts, 16) || parts_bytes < shared_bytes(plan, B, Sq, Hq, D)))
    return TRX_ERR_WORKSPACE;

  SharedParams p{};
  const int is_bf16 = dtype == TRX_BF16, tokens = plan.tile.tile_tokens, heads = plan.tile.tile_heads;
  const int box = plan.in_parts ? DEC_KEYS : ATT_BN;
  rc = make_ragged_kv_map(&p.tm_k, k, q, is_bf16, D, S, Hk, B, k_strides[0], k_strides[1], k_strides[2], box);
  if (rc != TRX_OK) return rc;
  rc = make_ragged_kv_map(&p.tm_v, v, q, is_bf16, D, S, Hk, B, v_strides[0], v_strides[1], v_strides[2], box);
  if (rc != TRX_OK) return rc;
  rc = make_ragged_kv_map(&p.tm_pk, prefix_k, q, is_bf16, D, P, Hk, 1, 0, pk_strides[0], pk_strides[1], ATT_BN);
  if (rc != TRX_OK) return rc;
  rc = make_ragged_kv_map(&p.tm_pv, prefix_v, q, is_bf16, D, P, Hk, 1, 0, pv_strides[0], pv_strides[1], ATT_BN);
  if (rc != TRX_OK) return rc;
  p.tile_heads = heads;
  p.tile_tokens = tokens;
  p.per_head = plan.tile.per_head;
  p.head_tiles = plan.tile.head_tiles;
  p.group = plan.tile.group;
  p.k_hdiv = p.v_hdiv = p.group;
  p.k_bmul = p.v_bmul = 1;
  p.slopes = slopes_or_null;
  p.status = reinterpret_cast<unsigned int*>(workspace);
  p.lengths = lengths_or_null;
  p.B = static_cast<int>(B);
  p.Sq = p.seq = static_cast<int>(Sq);
  p.Sk = p.keys = static_cast<int>(S);
  p.Hq = static_cast<int>(Hq);
  p.prefix = static_cast<int>(P);
  p.prefix_tiles = static_cast<int>((P + ATT_BN - 1) / ATT_BN);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = 1;
  p.win_left = p.win_right = -1;
  p.is_bf16 = is_bf16;
  p.reverse_kv = slopes_or_null ? 1 : 0;  // ALiBi: backwards, see attention_plain.cuh
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t step = ATT_NQ * tokens, rows = plan.parts > 0 ? B * Sq : Sq;
  const int64_t blocks = (rows + step - 1) / step;
  if (blocks > 65535 && !(plan.in_parts && plan.parts == 0)) return TRX_ERR_SHAPE;
  dim3 grid(static_cast<unsigned>(Hq / heads), static_cast<unsigned>(blocks), static_cast<unsigned>(B));

  bool beside = false;
  if (plan.parts > 0) {
    PrefixParams f{};
    static_cast<RaggedParams&>(f) = p;
    rc = make_ragged_q_map(&f.tm_q, q, is_bf16, D, B * Sq, Hq, 1, 0, row_stride, q_strides[2], heads, tokens);
    if (rc != TRX_OK) return rc;
    const int64_t n = B * Sq * Hq;
    f.rows = static_cast<int>(B * Sq);
    f.split_tiles = plan.split_tiles;
    f.out = parts;
    f.o_stride_b = n * D;
    f.o_stride_s = Hq * D;
    f.o_stride_h = D;
    f.lse = static_cast<float*>(parts) + plan.parts * n * D;
    f.lse_stride_b = n;
    p.part_o = static_cast<float*>(parts);
    p.part_lse = f.lse;
    p.parts = plan.parts;
    grid.z = plan.splits;
    // the decode kernel beside the prefix's, where all of that one's CTAs are running
    beside = static_cast<int64_t>(grid.x) * grid.y * grid.z <= sm_count_of_current_device();
    if (plan.halves) {
      HalvesParams two;
      static_cast<RaggedParams&>(two) = f;
      rc = launch_form_rows(two, D, grid, s);
    } else {
      rc = launch_form_rows(f, D, grid, s);
    }
    if (rc != TRX_OK) return rc;
  }
  p.out = out;
  p.o_stride_b = o_strides[0];
  p.o_stride_s = o_strides[1];
  p.o_stride_h = o_strides[2];
  p.lse = lse_or_null;
  p.lse_stride_b = Hq * Sq;
  p.lse_stride_h = Sq;
  if (plan.in_parts) {
    p.q = q;
    p.q_stride_b = q_strides[0];
    p.q_stride_s = q_strides[1];
    p.q_stride_h = q_strides[2];
    return launch_decode_rows(p, D, s, beside);
  }
  rc = make_ragged_q_map(&p.tm_q, q, is_bf16, D, Sq, Hq, B, q_strides[0], q_strides[1], q_strides[2], heads,
                         tokens);
  if (rc != TRX_OK) return rc;
  return launch_form_rows(p, D, grid, s);
}
