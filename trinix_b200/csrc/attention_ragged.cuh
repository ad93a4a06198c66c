// Rows and keys that are not one batch of equal lengths: what attention_plain.cuh's kernel and the decode
// kernel need to know of them.
//
//   ATT_PACKED  sequences of any lengths one after the other in q and in k / v, bounded by cu_q and cu_k
//               (device memory: the host knows only the totals);
//   ATT_SHARED  a batch whose sequences all have the keys of one prefix in front of their own, which lie in
//               a cache of fixed capacity of which lengths[b] are in use;
//   ATT_PREFIX  the prefix alone, the rows of the whole batch as one run, its keys split over CTAs; fp32
//               results that the decode kernel merges with those of the sequences' own keys.
//
// Query i of a sequence of Sq queries and Sk keys stands at key position i + Sk - Sq, the last query at the
// last key: a whole prompt, a piece of one behind cached keys and a single token are the same case.
//
// Query tiles: `tile_heads` query heads of one kv head times `tile_tokens` tokens, heads running faster, at
// most 128 rows. All heads of a group share a tile, so a short sequence fills it with heads where a tile of
// one head would be padding, and a CTA's two tiles see almost the same keys.
//
// Where one Q tile holds all the rows, the CTA's two tiles take every second K and V tile each (`alt` of an
// item), so that one tile's softmax runs under the other's MMAs: a packed sequence of up to `tile_tokens`
// rows with two tiles of heads, a run of that few rows against a prefix with two halves of its keys. Such
// launches have instantiations of their own (ALT): the test in the issuing warps' loop costs the others 3 to
// 5 % (16 prompts of 32 to 2048 rows 111 us, so 114; 16 x 512, 32 / 8 heads x 128 93, so 97; of ALT, 64 x
// 128, 16 heads x 64 36.9, so 28.6; 64 x 32, 32 / 8 heads x 128 31, so 25).
//
// Key tiles are not cut to a sequence: what follows its last key in memory belongs to another one, or is
// stale, and may be NaN. Scores there are masked as any others; in V, where a probability of 0 would not
// hide it (0 * NaN), the rows behind the last key are zeroed in shared memory (attention_plain.cuh).
#pragma once

#include "attention_common.cuh"

namespace trx {

struct RaggedParams : AttnParams {
  CUtensorMap tm_pk, tm_pv;  // the shared prefix
  const int* cu_q;           // packed: [n_cu + 1] first rows; the last is the end
  const int* cu_k;
  const int* lengths;        // shared: own keys in use; null: all
  int n_cu;                  // sequences of cu_q
  int n_seq;                 // and one more, without keys, if rows behind the last are to be zeroed
  int rows, keys;            // of the whole packed q and k / v; shared: keys a sequence's cache holds
  int tile_heads, tile_tokens;
  int per_head;              // 2^16 / tile_heads, rounded up: r / tile_heads of a row r < 128 of a tile
  int head_tiles;            // query heads / tile_heads
  int slots_first;           // packed without a table: the grid's x counts slots (and not heads)
  int seq;                   // shared: queries per sequence
  int prefix, prefix_tiles;  // keys of the prefix, in KV tiles
  int split_tiles;           // KV tiles of one split of the prefix
  const float* part_o;       // shared, decode kernel: [parts][B * Sq][Hq][D] results of the prefix's splits
  const float* part_lse;     // and their row sums' log2, [parts][B * Sq][Hq]
  int parts;
};
template <int F, bool A = false>
struct RaggedParamsOf : RaggedParams {
  static constexpr int FORM = F;
  static constexpr bool ALT = A;
};

struct RaggedItem : PlainItem {
  int q0, sq, k0, sk;  // first row and rows, first key and keys of the item's sequence
  int alt;             // 1: visit v is Q tile v & 1's alone
};

__device__ __forceinline__ int ragged_tokens(const RaggedParams& p) { return p.tile_tokens; }
__device__ __forceinline__ uint32_t ragged_q_bytes(const RaggedParams& p) {  // of 64 columns of a Q tile
  return 128u * p.tile_heads * p.tile_tokens;
}
// The token of row r of a Q tile. r * per_head is off r * 2^16 / tile_heads by less than 128: r / tile_heads
// is never nearer to the next whole number than 1 / 128.
__device__ __forceinline__ int ragged_token(const RaggedParams& p, int r) { return (r * p.per_head) >> 16; }
__device__ __forceinline__ int ragged_tokens(const AttnParams&) { return 0; }
__device__ __forceinline__ uint32_t ragged_q_bytes(const AttnParams&) { return 0; }

// Bounds that are out of range or out of order are cut to what the tensors hold.
__device__ __forceinline__ int ragged_row(const RaggedParams& p, int i) {  // first row of sequence i
  return i > p.n_cu ? p.rows : min(max(p.cu_q[i], 0), p.rows);
}
__device__ __forceinline__ int ragged_key(const RaggedParams& p, int i) {
  return min(max(p.cu_k[i], 0), p.keys);
}
__device__ __forceinline__ int ragged_length(const RaggedParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.keys) : p.keys;
}
// Position, behind the prefix, of row r of the batch.
__device__ __forceinline__ int ragged_position(const RaggedParams& p, int r) {
  const int b = r / p.seq;
  return p.prefix + ragged_length(p, b) - p.seq + (r - b * p.seq);
}
__device__ __forceinline__ int ragged_position(const AttnParams&, int) { return 0; }

// Packed rows: which sequence a block works on. The host knows the rows and the number of sequences but not
// where they end, and a table of blocks would cost a launch in front. A launch of several items per CTA with
// up to RAGGED_TABLE sequences counts every sequence's items (blocks of rows times tiles of heads, or pairs
// of these) in shared memory when a CTA starts, and finds an item by bisection there. Otherwise the grid is
// tiles of heads times slots: each sequence has the slots from floor(first row / R) + its index to
// the next one's, R rows being a block's: at least as many as it has blocks, on average half a slot too
// many, which are passed over, and found by a search in cu_q alone.
constexpr int RAGGED_TABLE = 1024;
// The sequences of every 128 are taken in the order of their keys, the most first: a block of many keys
// that starts late ends the launch late.
struct RaggedTable {
  int first[RAGGED_TABLE + 1];  // items before each sequence, in that order; the last: all
  int seq[RAGGED_TABLE];        // which one it is
  int row[RAGGED_TABLE + 1], key[RAGGED_TABLE + 1];
  int warp_sum[16];
};

// Whether a sequence of sq rows has its tiles of heads (an even number of them) in pairs.
template <bool ALT>
__device__ __forceinline__ bool ragged_pairs(const RaggedParams& p, int sq) {
  return ALT && sq <= p.tile_tokens;
}

struct RaggedCursor {
  int q0, sq, k0, sk;  // of the sequence
  int block, head;     // of its blocks of rows; tile of heads
  int alt;             // and the next tile of heads

  static __device__ __forceinline__ int first_slot(const RaggedParams& p, int i) {
    return ragged_row(p, i) / (ATT_NQ * p.tile_tokens) + i;
  }
  __device__ __forceinline__ void load(const RaggedParams& p, int s, int slot) {
    q0 = ragged_row(p, s);
    sq = max(0, ragged_row(p, s + 1) - q0);
    k0 = sk = 0;
    if (s < p.n_cu) {
      k0 = ragged_key(p, s);
      sk = max(0, ragged_key(p, s + 1) - k0);
    }
    block = slot - (q0 / (ATT_NQ * p.tile_tokens) + s);
    alt = 0;
  }
  // The last sequence whose first slot is not behind `at`; a whole warp, 32 probes at a time.
  __device__ __forceinline__ void seek(const RaggedParams& p, int at, int lane) {
    int lo = 0, hi = p.n_seq;
#pragma unroll 1
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, i = lo + lane * step;
      const unsigned not_behind = __ballot_sync(0xffffffffu, i < hi && first_slot(p, i) <= at);
      const int n = __popc(not_behind);
      lo += max(0, n - 1) * step;
      hi = min(hi, lo + step);
    }
    load(p, lo, at);
  }
  // The same by one thread: 15 probes at a time, whose loads are in flight together where a bisection
  // waits for each.
  __device__ __forceinline__ void seek_alone(const RaggedParams& p, int at) {
    constexpr int N = 15;
    int lo = 0, hi = p.n_seq;
#pragma unroll 1
    while (hi - lo > 1) {
      const int step = (hi - lo + N) / (N + 1);
      int n = 0;
#pragma unroll
      for (int i = 1; i <= N; ++i) {
        const int probe = lo + i * step;
        n += probe < hi && first_slot(p, min(probe, hi - 1)) <= at ? 1 : 0;
      }
      lo += n * step;
      if (n < N) hi = min(hi, lo + step);
    }
    load(p, lo, at);
  }
  template <bool ALT>
  __device__ __forceinline__ void look_up(const RaggedParams& p, const RaggedTable& t, int at) {
    int lo = 0, hi = p.n_seq;
#pragma unroll 1
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (t.first[mid] <= at) lo = mid;
      else hi = mid;
    }
    const int s = t.seq[lo], i = at - t.first[lo];
    q0 = t.row[s];
    sq = max(0, t.row[s + 1] - q0);
    k0 = t.key[s];
    sk = s < p.n_cu ? max(0, t.key[s + 1] - k0) : 0;
    alt = ragged_pairs<ALT>(p, sq) ? 1 : 0;
    const int heads = p.head_tiles >> alt;
    block = i / heads;
    head = (i - block * heads) << alt;
  }
};
// The whole CTA, 512 threads of two sequences each.
template <bool ALT>
__device__ __forceinline__ void ragged_fill(const RaggedParams& p, RaggedTable& t) {
  static_assert(RAGGED_TABLE == 2 * 512, "two sequences per thread");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = 2 * threadIdx.x;
  const int step = ATT_NQ * p.tile_tokens;
  for (int e = threadIdx.x; e <= p.n_seq; e += 512) {
    t.row[e] = ragged_row(p, e);
    t.key[e] = ragged_key(p, min(e, p.n_cu));
  }
  __syncthreads();
  auto keys_of = [&](int s) { return t.key[s + 1] - t.key[s]; };
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int s = i + e;
    if (s < p.n_seq) {
      const int own = keys_of(s), from = s - s % 128, to = min(p.n_seq, from + 128);
      int more = from;  // sequences in front of this one
#pragma unroll 4
      for (int o = from; o < to; ++o) {
        const int k = keys_of(o);
        more += k > own || (k == own && o < s) ? 1 : 0;
      }
      t.seq[more] = s;
    }
  }
  __syncthreads();
  int blocks[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    blocks[e] = 0;
    if (i + e < p.n_seq) {
      const int s = t.seq[i + e];
      const int rows = max(0, t.row[s + 1] - t.row[s]);
      blocks[e] = (rows + step - 1) / step * (ragged_pairs<ALT>(p, rows) ? p.head_tiles / 2 : p.head_tiles);
    }
  }
  const int own = blocks[0] + blocks[1];
  int sum = own;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int below = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += below;
  }
  if (lane == 31) t.warp_sum[warp] = sum;
  __syncthreads();
  int before = sum - own;
  for (int w = 0; w < warp; ++w) before += t.warp_sum[w];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (i + e < p.n_seq) t.first[i + e] = before;
    before += blocks[e];
    if (i + e == p.n_seq - 1) t.first[p.n_seq] = before;
  }
  __syncthreads();
}

// The cursor of a block of the grid without a table.
__device__ __forceinline__ int ragged_slot(const RaggedParams& p, int x, int y) {
  return p.slots_first ? x : y;
}
__device__ __forceinline__ int ragged_head(const RaggedParams& p, int x, int y) {
  return p.slots_first ? y : x;
}
__device__ __forceinline__ bool ragged_has_rows(const RaggedItem& w) { return w.sq > 0; }
__device__ __forceinline__ bool ragged_has_rows(const PlainItem&) { return true; }

// KV tiles that the rows of a Q tile see, the first of them `row0` of its sequence. Shared form: the tiles
// of the prefix, then those of the sequence's own keys.
template <int FORM>
__device__ __forceinline__ TileRange ragged_range(const RaggedParams& p, const RaggedItem& w, int row0) {
  TileRange r{0, 0};
  if (row0 >= w.sq) return r;
  const int last = min(w.sq, row0 + p.tile_tokens) - 1;
  if constexpr (FORM == ATT_PREFIX) {
    r.jlo = w.b * p.split_tiles;
    r.jhi = min(p.prefix_tiles, r.jlo + p.split_tiles);
  } else if constexpr (FORM == ATT_SHARED) {
    const int hi = last + w.sk - w.sq;  // of its own keys
    if (hi >= 0) r.jhi = p.prefix_tiles + hi / ATT_BN + 1;
    else if (p.prefix + hi >= 0) r.jhi = (p.prefix + hi) / ATT_BN + 1;
  } else {
    const int shift = w.sk - w.sq;
    int hi = w.sk - 1, lo = 0;
    if (p.causal) hi = min(hi, last + shift);
    if (p.win_right >= 0) hi = min(hi, last + shift + p.win_right);
    if (p.win_left >= 0) lo = max(0, row0 + shift - p.win_left);
    if (hi < lo) return r;
    r.jlo = lo / ATT_BN;
    r.jhi = hi / ATT_BN + 1;
  }
  return r;
}

template <int FORM, bool ALT>
__device__ __forceinline__ RaggedItem ragged_item(const RaggedParamsOf<FORM, ALT>& p, const RaggedCursor& c,
                                                  int x, int y, int z) {
  RaggedItem w;
  const int step = ATT_NQ * p.tile_tokens;
  w.valid = 1;
  if constexpr (FORM == ATT_PACKED) {
    w.b = 0;
    w.h = c.head * p.tile_heads;
    w.q0 = c.q0;
    w.sq = c.sq;
    w.k0 = c.k0;
    w.sk = c.sk;
    w.alt = ALT ? c.alt : 0;
    const int blocks = (c.sq + step - 1) / step;
    if (c.block < 0 || c.block >= blocks) {  // the slot holds no rows
      w.sq = w.m0 = 0;
    } else {
      w.m0 = (p.causal ? blocks - 1 - c.block : c.block) * step;  // heaviest first
    }
  } else {
    w.b = z;  // sequence, or split of the prefix
    w.h = x * p.tile_heads;
    w.q0 = w.k0 = 0;
    w.sq = FORM == ATT_SHARED ? p.seq : p.rows;
    w.sk = FORM == ATT_SHARED ? ragged_length(p, z) : 0;
    w.alt = ALT ? 1 : 0;
    w.m0 = static_cast<int>(gridDim.y - 1 - y) * step;
  }
  TileRange r[ATT_NQ];
  int jlo = 1 << 30, jhi = 0;
#pragma unroll
  for (int t = 0; t < ATT_NQ; ++t) {
    r[t] = ragged_range<FORM>(p, w, w.m0 + (w.alt ? 0 : t * p.tile_tokens));
    if (r[t].jhi > r[t].jlo) {
      jlo = min(jlo, r[t].jlo);
      jhi = max(jhi, r[t].jhi);
    }
  }
  w.n = max(0, jhi - jlo);
  w.first = p.reverse_kv ? jhi - 1 : jlo;
#pragma unroll
  for (int t = 0; t < ATT_NQ; ++t) {
    const bool any = r[t].jhi > r[t].jlo;
    w.lo[t] = !any ? 0 : p.reverse_kv ? jhi - r[t].jhi : r[t].jlo - jlo;
    w.hi[t] = !any ? 0 : w.lo[t] + r[t].jhi - r[t].jlo;
  }
  if (ALT && w.alt) {  // both have the same range: every second visit each
    if (FORM == ATT_PACKED) w.n *= 2;  // (of two heads)
#pragma unroll
    for (int t = 0; t < ATT_NQ; ++t) {
      const int own = (w.n - t + 1) / 2;
      w.lo[t] = own > 0 ? t : 0;
      w.hi[t] = own > 0 ? t + 2 * own - 1 : 0;
    }
  }
  return w;
}

// Where KV tile j of an item starts, and how many of its rows are the sequence's; `edge`: the others are
// inside the tensor (behind its end the copy fills with zeros).
struct RaggedTile {
  int row, b, rows;
  bool prefix, edge;
};
template <int BN, int FORM, bool ALT>
__device__ __forceinline__ RaggedTile ragged_tile(const RaggedParamsOf<FORM, ALT>& p, const RaggedItem& w, int j) {
  RaggedTile r;
  r.prefix = FORM == ATT_PREFIX || (FORM == ATT_SHARED && j < p.prefix_tiles);
  const int first = (FORM == ATT_SHARED && !r.prefix ? j - p.prefix_tiles : j) * BN;
  const int keys = r.prefix ? p.prefix : w.sk;
  r.row = w.k0 + first;
  r.b = FORM == ATT_SHARED && !r.prefix ? w.b : 0;
  r.rows = keys - first;
  r.edge = r.rows < BN && w.k0 + keys < (r.prefix ? p.prefix : p.keys);
  return r;
}

// ------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------
// What base and element strides of (B, rows, H, D) queries have to be, for their tensor map and for the decode
// kernel's 4-byte loads. Dims of size 1 may carry any stride: they are given a legal one.
inline int check_ragged_q(const void* base, int64_t D, int64_t rows, int64_t H, int64_t B, int64_t& sb, int64_t& ss,
                          int64_t& sh) {
  if (!aligned_to(base, 16)) return TRX_ERR_ALIGNMENT;
  if (rows == 1) ss = D;
  if (H == 1) sh = D;
  if (B == 1) sb = D;
  if (ss < D || sh < D || sb < D) return TRX_ERR_STRIDE;
  if (ss % 8 || sh % 8 || sb % 8) return TRX_ERR_ALIGNMENT;
  if (ss >= (1ll << 38) || sh >= (1ll << 30) || sb >= (1ll << 38)) return TRX_ERR_STRIDE;
  return TRX_OK;
}

// Keys or values (B, rows, H, D). Without rows nothing is loaded: any legal map, whatever strides a tensor
// without elements carries; `other` is memory for it.
inline int make_ragged_kv_map(CUtensorMap* tm, const void* base, const void* other, int is_bf16, int64_t D,
                              int64_t rows, int64_t H, int64_t B, int64_t sb, int64_t ss, int64_t sh, int box_rows) {
  if (rows == 0) return make_map(tm, other, is_bf16, D, 1, 1, 1, D, D, D, box_rows);
  return make_map(tm, base, is_bf16, D, rows, H, B, sb, ss, sh, box_rows);
}

// Queries for tiles of `heads` heads x `tokens` rows: dims D, head in tile, row, tile of heads, B.
inline int make_ragged_q_map(CUtensorMap* tm, const void* base, int is_bf16, int64_t D, int64_t rows, int64_t H,
                             int64_t B, int64_t sb, int64_t ss, int64_t sh, int heads, int tokens) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return TRX_ERR_CUDA;
  const int rc = check_ragged_q(base, D, rows, H, B, sb, ss, sh);
  if (rc != TRX_OK) return rc;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(H / heads),
                              static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(ss) * 2,
                                 static_cast<cuuint64_t>(sh) * heads * 2, static_cast<cuuint64_t>(sb) * 2};
  const cuuint32_t tile[5] = {64, static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(tokens), 1, 1},
                   step[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(tm, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                         const_cast<void*>(base), dims, strides, tile, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TRX_OK : TRX_ERR_CUDA;
}

// Query heads of one tile, and tokens: as many heads of the group as leave at most a tenth of a tile's 128
// rows unused, and a run of `rows` no more blocks than a grid's dimension holds. (A group of 71 heads is none
// but 1 and 71, and 71 would leave 57 rows.)
inline void choose_tile(RaggedParams& p, int64_t rows) {  // from its Hq and group
  p.tile_heads = 1;
  for (int h = 2; h <= p.group && h <= ATT_BM; ++h)
    if (p.group % h == 0 && ATT_BM / h * h * 10 >= ATT_BM * 9 && rows <= 65535ll * ATT_NQ * (ATT_BM / h))
      p.tile_heads = h;
  p.tile_tokens = ATT_BM / p.tile_heads;
  p.per_head = (65536 + p.tile_heads - 1) / p.tile_heads;
  p.head_tiles = p.Hq / p.tile_heads;
}

}  // namespace trx
