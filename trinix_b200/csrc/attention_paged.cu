// Attention over the pages of a cache: the C entries, and the launches of attention_paged.cuh.
#include "attention_paged.cuh"

namespace trx {

// The shape that a call takes: f(D, 4 bits, tiles of 8 rows) as compile-time numbers.
template <class F>
static auto paged_shape(int64_t D, bool four, int64_t rows, F&& f) {
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  auto by_rows = [&](auto d, auto bits) { return rows > 8 ? f(d, bits, Two{}) : f(d, bits, One{}); };
  auto by_bits = [&](auto d) { return four ? by_rows(d, std::true_type{}) : by_rows(d, std::false_type{}); };
  return D == 128 ? by_bits(D128{}) : by_bits(D64{});
}

// What the plan of a call goes by; keys: the most that a sequence may have.
static PagedPlan plan_of(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D, int64_t keys, int64_t window_left,
                         bool four) {
  const int64_t rows = Sq * (Hq / Hk), tile = rows > 8 ? 16 : 8;
  if (window_left >= 0 && window_left < keys - Sq) keys = Sq + window_left;
  return paged_shape(D, four, rows, [&](auto d, auto bits, auto nt) {
    return paged_plan<decltype(d)::value, decltype(bits)::value, decltype(nt)::value>(
        B * Hk * ((rows + tile - 1) / tile), keys);
  });
}

}  // namespace trx

using namespace trx;

extern "C" size_t trx_attn_paged_bytes(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D, int64_t keys,
                                       int64_t window_left, int four_bits) {
  if (B <= 0 || Sq <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || (D != 64 && D != 128) || keys < 0 || B > 65535 ||
      Sq >= (1ll << 28) || Hq > 65535 || keys >= (1ll << 29))
    return 0;
  return plan_of(B, Sq, Hq, Hk, D, keys, window_left, four_bits != 0).bytes;
}

extern "C" int trx_attn_fwd_paged(const void* q, const void* k_pages, const void* v_pages,
                                  const float* k_scales_or_null, const float* v_scales_or_null, void* out,
                                  float* lse_or_null, const float* slopes_or_null, const int32_t* block_table,
                                  const int32_t* lengths, int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D,
                                  int64_t pages, int64_t page_size, int64_t width, const int64_t strides[17],
                                  float scale, int64_t window_left, int dtype, void* parts_or_null,
                                  size_t parts_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != TRX_BF16 && dtype != TRX_F16) return TRX_ERR_DTYPE;
  if (!strides) return TRX_ERR_NULL_POINTER;
  if (B < 0 || Sq < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk != 0) return TRX_ERR_SHAPE;
  PagedParams p{};
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
  const int64_t rows = Sq * p.group, tile = rows > 8 ? 16 : 8;
  p.row_tiles = static_cast<int>((rows + tile - 1) / tile);
  if (Hk * p.row_tiles > 65535 || B * Hk * p.row_tiles >= (1ll << 31) / PG_MOST_SPLITS) return TRX_ERR_SHAPE;
  if (!aligned_to(q, 16) || !aligned_to(out, 16) || !aligned_to(lengths, 4)) return TRX_ERR_ALIGNMENT;
  for (int i = 0; i < 6; ++i) {
    if (strides[i] < 0) return TRX_ERR_STRIDE;
    if (strides[i] % 8) return TRX_ERR_ALIGNMENT;
  }
  p.capacity = static_cast<int>(width * page_size);
  p.win_left = window_left < 0 ? -1 : static_cast<int>(window_left > (1ll << 29) ? (1ll << 29) : window_left);
  const bool four = p.c.k_scales != nullptr, bf16 = dtype == TRX_BF16;
  const PagedPlan plan = plan_of(B, Sq, Hq, Hk, D, p.capacity, p.win_left, four);
  if (plan.bytes > 0 && (!parts_or_null || !aligned_to(parts_or_null, 16) || parts_bytes < plan.bytes))
    return TRX_ERR_WORKSPACE;
  p.splits = plan.splits;
  p.pieces = static_cast<PagedPiece*>(parts_or_null);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(parts_or_null) + plan.pieces_bytes);
  p.q = q;
  p.q_stride_b = strides[0];
  p.q_stride_s = strides[1];
  p.q_stride_h = strides[2];
  p.out = out;
  p.o_stride_b = strides[3];
  p.o_stride_s = strides[4];
  p.o_stride_h = strides[5];
  p.lse = lse_or_null;
  p.slopes = slopes_or_null;
  p.status = reinterpret_cast<unsigned int*>(workspace);
  p.lengths = lengths;
  p.B = static_cast<int>(B);
  p.Sq = static_cast<int>(Sq);
  p.Hq = static_cast<int>(Hq);
  p.heads = static_cast<int>(Hk);
  p.units = p.heads * p.row_tiles;
  // r * magic / 2^32 is off r / group by less than r * group / 2^32 / group
  if (p.group > 1 && rows * p.group < (1ll << 32))
    p.group_magic = static_cast<unsigned>(((1ull << 32) + p.group - 1) / p.group);
  p.scale_log2 = scale * 1.4426950408889634f;
  if (!four) {
    const PagedCache& c = p.c;
    rc = make_map(&p.tm_k, k_pages, bf16, D, page_size, Hk, pages, c.kp[0], c.kp[2], c.kp[1], PG_RUN);
    if (rc != TRX_OK) return rc;
    rc = make_map(&p.tm_v, v_pages, bf16, D, page_size, Hk, pages, c.vp[0], c.vp[2], c.vp[1], PG_RUN);
    if (rc != TRX_OK) return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return paged_shape(D, four, rows, [&](auto d, auto bits, auto nt) {
    constexpr int DIM = decltype(d)::value, NT = decltype(nt)::value;
    constexpr bool FOUR = decltype(bits)::value;
    auto launch = [&](auto twice) {
      constexpr bool TWICE = decltype(twice)::value;
      return bf16 ? launch_paged<DIM, true, FOUR, NT, TWICE>(p, plan, s)
                  : launch_paged<DIM, false, FOUR, NT, TWICE>(p, plan, s);
    };
    if constexpr (NT == 1) {
      if (rows <= 4) return launch(std::true_type{});
    }
    return launch(std::false_type{});
  });
}
