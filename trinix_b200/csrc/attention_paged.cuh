// Attention forward for few query rows against the keys in the pages of a cache (paged_cache.cuh), of 16 bits or
// of 4.
//
// Reading the keys is the work, and sequences of one batch may have a hundred times the keys of others. So the
// tiles of keys of the whole batch, (sequence, kv head, tile of rows) one after the other, are one line that is
// cut into as many equal pieces as there are CTAs: a CTA works on the end of one such unit, some whole ones and
// the beginning of another. What it has of a unit that is not whole goes to memory, unnormalised, and a second
// launch, prepared beside the first one's end, adds the parts up. The cuts follow from the lengths, which only the
// device knows: every CTA adds them up when it starts. The sums' order is fixed by the lengths and the SM count.
// All that costs a call 5 to 7 us. (Parts added up by the CTA that finds them all there, told by flags, so that
// there is one launch: 2 x 131072 keys of 4 bits 48 us, so 44; 48 sequences of up to 8192 of 16 bits 73, so 71.)
// Where the cache holds few keys to a sequence a unit has a CTA, or, where there are
// few units, a cluster, whose CTAs share its keys alike and add up over distributed shared memory.
//
//   * Both products are transposed: S^T = K Q^T and O^T = V^T P^T, so that a tile's 16 is keys, or columns of V,
//     and its 8 is query rows: a group of four heads fills half of the tile where it would be a quarter. The
//     scores' fragment becomes the operand of the second product by one movmatrix per 8 keys.
//   * Each warp has a ring of tiles of its own, and its own running maximum, sum and O; the next unit's first tiles
//     are on their way while the CTA's warps' results meet in shared memory.
//   * The reference maximum of a row follows only when it is far behind (by ATT_LAZY_RESCALE), and until a lane
//     sees that, the rows' maxima, three shuffles each, are not asked for.
//
// 4 bits. A key costs D + 16 bytes (codes, step and lowest of K and of V) where 16 bits cost 4 D, so of the same
// bandwidth four times the keys come by, and what is done to each has to be that much cheaper:
//   * The codes enter the matrix instructions as they are: a code c in the low bits of a 16-bit half is the
//     subnormal fp16 number c * 2^-24, one in the next four bits 16 times that, and mma.sync takes subnormal
//     operands. A word of eight codes becomes four operand registers by one shift and four ANDs; nothing is
//     converted, and nothing is multiplied, since with one step and lowest to a row
//         score = step_k (q . c_k) + lowest_k sum(q),    O = sum(p step_v c_v) + sum(p lowest_v).
//     The powers of two are put into Q and taken out of the results, exactly.
//   * Which column of the row a fragment's element is does not matter as long as both sides agree: a lane reads 16
//     (K) and 8 (V) bytes of a row in one piece. Of 8 keys the fragment's rows are in the order 0, 4, 1, 5, ...:
//     then the four V rows that a load reads are neighbours.
//   * fp16 operands serve both activation types: Q's rows are scaled by a power of two to below 2^14 (what is
//     2^-28 of the row's largest value or more stays exact; a row with values of 2^114 and more is not a number).
//     Probabilities are weighed with step_v before they become fp16, two numbers each, and the running
//     maximum is that of the weighed ones, so that the largest weight of a row is of the order of 1 whatever the steps
//     are.
// Scores, sums and O are fp32.
//
// Measured (32 / 8 heads x 128, one token to a sequence): 48 sequences of 128 to 8192 keys, 16 bits, 385 MB: 72 us,
// 5.3 TB/s; 64 of 4 bits, 143 MB: 44.7 us; 2 x 131072 and fewer keys of 4 bits, 155 MB: 44.2 us, 3.5 TB/s. What bounds
// it: 16 bits, the memory (without the arithmetic 67.7 us). 4 bits, both: loads alone would take 36 us, arithmetic
// alone 37 (500 instructions to 32 keys of a warp, 176 of them the shifts, ANDs and permutes that make operands of
// codes; three CTAs of 168 registers issue 46 % of the time), 8 of either the call's start, the cuts and the parts.
// Tried: 16 keys at a time as in attention_decode.cuh and clusters of fixed splits, 4 bits 100 and 109 us; tiles of
// 32 keys 48 and 47 us; four CTAs to an SM 64 to 67 (registers); two sums for a run's products, or two steps of 32
// keys unrolled: nothing.
#pragma once

#include "attention_decode.cuh"
#include "paged_cache.cuh"

namespace trx {

constexpr int PG_WARPS = 4;
constexpr int PG_THREADS = PG_WARPS * 32;
constexpr int PG_RUN = 16;  // keys that lie in one page
constexpr int PG_MOST_SPLITS = 8;
constexpr int PG_MOST_CTAS = 1024;  // of a launch that cuts units
// The steps of V that are 0, of rows of one value, are weighed as this; the others are larger (paged_cache.cuh). A
// weight over this and the keys of a sequence times 2^20 stay within fp32.
constexpr float PG_LEAST_STEP = 0x1p-80f;
// The reference maximum of a row that has seen nothing: finite, so that no difference of it is not a number.
constexpr float PG_NOTHING = -1e30f;
// fp16 weights are 2^7 times what the reference maximum makes of them, so that those of 2^-31 of it and more are not
// lost; with ATT_LAZY_RESCALE they stay below 2^15.
constexpr float PG_FP16_UP = 7.0f, PG_FP16_SCALE = 0x1p7f;

// What a CTA of the first launch leaves for the second one: the unit that it found begun, if there is one.
struct PagedPiece {
  long long lo;          // the CTA's first place on the line
  long long unit, end;   // where the unit begins, and its last tile ends; unit < 0: none
  int b, head, r0, pad;
};

struct PagedParams {
  CUtensorMap tm_k, tm_v;  // 16 bits
  PagedCache c;
  const void* q;
  void* out;
  float* lse;
  const float* slopes;
  const int* lengths;
  unsigned int* status;
  long long q_stride_b, q_stride_s, q_stride_h;
  long long o_stride_b, o_stride_s, o_stride_h;
  int B, Sq, Hq, group, row_tiles;
  int heads, units;        // kv heads; units of a sequence: these * row tiles
  unsigned group_magic;    // 2^32 / group, rounded up, where that divides every row; or 0
  int capacity;            // keys that a row of the block table holds
  int win_left;            // < 0: no window
  int splits;              // CTAs of a unit's cluster; 0: the batch is one line
  float scale_log2;
  PagedPiece* pieces;      // [CTAs]
  float* part;             // [CTAs][2]: of the unit found begun, of the one left unfinished: O, m, l
};

template <int D, bool FOUR, int NT>
struct PgShape {
  static constexpr int KEYS = FOUR ? 64 : 16;  // of a tile
  static constexpr int RUNS = KEYS / PG_RUN;
  static constexpr int STEP = FOUR ? 32 : 16;  // keys that a warp works on at a time
  static constexpr int STAGES = FOUR ? 2 : 3;
  static constexpr int CTAS_PER_SM = FOUR && (NT == 1 || D == 64) ? 3 : 2;
  static constexpr int CODES = PG_RUN * D / 2, SCALES = PG_RUN * 8;  // bytes of 16 keys
  // a tile's K codes, V codes, K scales, V scales
  static constexpr int V_OFF = RUNS * CODES, KS_OFF = 2 * V_OFF, VS_OFF = KS_OFF + RUNS * SCALES;
  static constexpr int CHUNKS = D / 64, CHUNK_BYTES = 16 * 128, HALF_BYTES = CHUNKS * CHUNK_BYTES;  // 16 bits
  static constexpr int STAGE_BYTES = FOUR ? VS_OFF + RUNS * SCALES : 2 * HALF_BYTES;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int ROWS = 8 * NT;
  // a warp's partial O takes the place of this many stages, the next unit's tiles the others
  static constexpr int O_BYTES = 8 * D * 4;  // of 8 rows
  static constexpr int O_STAGES = NT * O_BYTES <= STAGE_BYTES ? 1 : NT;
  static_assert(O_BYTES <= STAGE_BYTES && O_STAGES < STAGES, "partial O");
  static constexpr int BAR_OFF = PG_WARPS * RING_BYTES;
  static constexpr int ML_OFF = BAR_OFF + PG_WARPS * STAGES * 8;      // max, sum per warp and row
  static constexpr int CTA_ML_OFF = ML_OFF + 2 * PG_WARPS * ROWS * 4;
  static constexpr int AT_OFF = CTA_ML_OFF + 2 * ROWS * 4;            // where each warp's O is
  static constexpr int FLAG_OFF = AT_OFF + PG_WARPS * NT * 4;         // a flag per warp: it has no result
  static constexpr int TOTAL = FLAG_OFF + (PG_WARPS + 1) * 4;
  static constexpr int ALIGN = FOUR ? 128 : 1024;
  static constexpr int DYN_BYTES = TOTAL + ALIGN;
  static constexpr int PART_FLOATS = ROWS * (D + 2);  // of one part in memory
  // What a unit costs beside its tiles, in tiles. 4 bits 2, 3, 4, 6, 8, 12: 64 sequences of 128 to 8192 keys 54.0, 49.5,
  // 47.4, 44.5, 45.8, 47.6 us, 256 of up to 600 46.7, 43.2, 43.5, 39.9, 39.7, 41.4; 16 bits 4, 6, 8, 12, 16, 24: 48
  // sequences 80.9, 73.6, 71.6, 71.8, 71.3, 72.9, 256 of up to 600 60.2, 53.4, 50.5, 45.1, 45.1, 48.4.
  // What a piece of the line has at least, so that a CTA that has one works longer than it takes to start and to hand
  // its part over. It matters to lines of few tiles alone: 4 bits, 2 to 8 alike, 16: 24 x 5 rows of up to 3001 keys 29.3
  // instead of 26.0 us, 16 sequences of up to 8000 23.1 instead of 21.9, one of 32768 21.2 instead of 23.3; 16 bits, 4 to
  // 32 alike.
  static constexpr int UNIT_COST = FOUR ? 6 : 12;
  static constexpr int LEAST_PIECE = FOUR ? 8 : 16;
  static_assert(RING_BYTES >= PG_THREADS * 8, "the sums of the lengths");
};

// What is read where no page is.
__device__ uint4 pg_zeros[64 * 128 / 2 / 16];

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
// (lo, hi) as 16-bit numbers that are not larger, for those that are not negative.
template <bool BF16>
__device__ __forceinline__ uint32_t pack16_below(float lo, float hi) {
  if constexpr (BF16) return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
  uint32_t d;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
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

// The keys that some query of sequence b sees, in tiles.
struct PagedKeys {
  int sk, first, tiles;
};
template <int KEYS>
__device__ __forceinline__ PagedKeys paged_keys(const PagedParams& p, int b) {
  PagedKeys k;
  k.sk = min(max(__ldg(p.lengths + b), 0), p.capacity);
  int lo = 0;
  if (p.win_left >= 0) lo = max(0, k.sk - p.Sq - p.win_left);
  k.first = lo / KEYS;
  k.tiles = k.sk > 0 ? (k.sk - 1) / KEYS + 1 - k.first : 0;
  return k;
}

// Where partial result `which` of CTA `cta` is: O [ROWS][D], then the rows' maxima, then their sums.
template <int D, bool FOUR, int NT>
__device__ __forceinline__ float* paged_part(const PagedParams& p, int cta, int which) {
  return p.part + (2ll * cta + which) * PgShape<D, FOUR, NT>::PART_FLOATS;
}

// r / group of a row r of a sequence.
__device__ __forceinline__ int paged_token(const PagedParams& p, int r) {
  return p.group == 1 ? r : p.group_magic ? static_cast<int>(__umulhi(r, p.group_magic)) : r / p.group;
}

// Four columns of a row of the result, and the row's LSE: acc / l. A row without keys has l == 0.
template <int D, bool BF16>
__device__ __forceinline__ void paged_emit(const PagedParams& p, int b, int head, int row, int c4, float4 acc, float mx,
                                           float l) {
  const int s = paged_token(p, row), h = head * p.group + row - s * p.group;
  const float inv = l > 0.0f ? __fdividef(1.0f, l) : l == l ? 0.0f : l;
  uint2 v;
  v.x = pack16<BF16>(acc.x * inv, acc.y * inv);
  v.y = pack16<BF16>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + b * p.o_stride_b + s * p.o_stride_s +
                            h * p.o_stride_h + 4 * c4) = v;
  if (p.lse && c4 == 0)
    p.lse[(static_cast<long long>(b) * p.Hq + h) * p.Sq + s] =
        l == 0.0f ? -INFINITY : (mx + log2f(l)) * 0.6931471805599453f;
}

// TWICE: at most four rows, which have two of the tile's eight columns each (see the weights below).
template <int D, bool BF16, bool FOUR, int NT, bool TWICE>
__global__ void __launch_bounds__(PG_THREADS, PgShape<D, FOUR, NT>::CTAS_PER_SM)
    attn_paged_kernel(const __grid_constant__ PagedParams p) {
  using L = PgShape<D, FOUR, NT>;
  constexpr int KEYS = L::KEYS, RUNS = L::RUNS, STAGES = L::STAGES;
  constexpr int KW = D / 32;       // 4 bits: words of a K row to a thread
  constexpr int VW = D / 64;       // of a V row
  constexpr int MTILES = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + L::ALIGN - 1) &
                                             ~static_cast<uintptr_t>(L::ALIGN - 1));
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t4 = lane & 3, g8 = lane >> 2;
  const uint32_t ring = sbase + warp * L::RING_BYTES;
  const uint32_t bars = sbase + L::BAR_OFF + warp * STAGES * 8;
  float* ml = reinterpret_cast<float*>(smem + L::ML_OFF);          // [2][PG_WARPS][ROWS]
  float* cta_ml = reinterpret_cast<float*>(smem + L::CTA_ML_OFF);  // [2][ROWS]
  int* o_at = reinterpret_cast<int*>(smem + L::AT_OFF);    // [PG_WARPS][NT]
  volatile int* no_result = reinterpret_cast<int*>(smem + L::FLAG_OFF);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(bars + 8 * s, 1);
    no_result[warp] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (threadIdx.x == 0) no_result[PG_WARPS] = *reinterpret_cast<volatile unsigned int*>(p.status) != 0u;

  // ---- this CTA's piece [at, stop) of the line, and the sequence that it begins in --------------
  long long at = 0, stop = 0, seq_at = 0;  // seq_at: where that sequence's units begin
  int b = 0;
  PagedKeys keys{};
  int split = 0;
  if (p.splits) {
    const int i = blockIdx.x / p.splits;
    split = blockIdx.x - i * p.splits;
    b = i / p.units;
    keys = paged_keys<KEYS>(p, b);
    at = static_cast<long long>(i - b * p.units) * (keys.tiles + L::UNIT_COST);
    stop = at + keys.tiles + L::UNIT_COST;
    __syncthreads();
  } else {
    long long* sums = reinterpret_cast<long long*>(smem);  // [PG_THREADS]
    auto cost = [&](int i) -> long long { return i < p.B ? paged_keys<KEYS>(p, i).tiles + L::UNIT_COST : 0; };
    const long long first_cost = cost(threadIdx.x);
    long long mine = first_cost;
    for (int i = threadIdx.x + PG_THREADS; i < p.B; i += PG_THREADS) mine += cost(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int w = 0; w < PG_WARPS; ++w) all += sums[w];
    all *= p.units;
    const long long most = all / L::LEAST_PIECE;
    const long long ctas = most < 1 ? 1 : most < gridDim.x ? most : gridDim.x;
    at = static_cast<long long>(blockIdx.x) < ctas ? blockIdx.x * all / ctas : all;
    stop = static_cast<long long>(blockIdx.x) < ctas ? (blockIdx.x + 1) * all / ctas : all;
    if (threadIdx.x == 0) {
      PagedPiece piece{at, -1, -1, 0, 0, 0, 0};
      p.pieces[blockIdx.x] = piece;  // until it is known better
    }
    if (at >= stop) return;
    // the sequence of `at`: sums over 128 of them at a time
    for (int i0 = 0; i0 < p.B; i0 += PG_THREADS) {
      long long v = i0 == 0 ? first_cost : cost(i0 + threadIdx.x);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
      }
      __syncthreads();
      sums[threadIdx.x] = v;  // within the warp
      __syncthreads();
      long long before = seq_at;
      int found = -1;
      for (int w = 0; w < PG_WARPS && found < 0; ++w) {
        const long long in_warp = sums[32 * w + 31] * p.units;
        if (at < before + in_warp) {
          const unsigned behind = __ballot_sync(0xffffffffu, before + sums[32 * w + lane] * p.units > at);
          const int i = __ffs(behind) - 1;
          found = i0 + 32 * w + i;
          seq_at = before + (i > 0 ? sums[32 * w + i - 1] * p.units : 0);
        }
        before += in_warp;
      }
      if (found >= 0) {
        b = found;
        break;
      }
      seq_at = before;
    }
    keys = paged_keys<KEYS>(p, b);
    __syncthreads();  // the sums have been read: the ring is there
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // A launch that follows a recorded failure writes nothing. The word may turn non-zero at any time, so that CTAs of
  // a cluster may see it differently: they all stay to the end.
  const bool skip = no_result[PG_WARPS] != 0;
  if (skip) {
    if (threadIdx.x == 0) report_status(p.status);
    if (p.splits < 2) return;
  }

  // every CTA runs: the second launch may take its place beside this one
  if (!p.splits) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- units ---------------------------------------------------------------------------------
  struct Unit {
    int valid, b, head, r0;
    int sk, t0, t1;      // its tiles that this CTA has
    int which;           // 0, 1: the part of it that this CTA leaves, -1: all of it
    int tiles;           // of the whole unit
    int hi, hi_min, lo_max;
  };
  const int rows = p.group * p.Sq;
  // where the next one begins, which it is
  int unit_head, unit_tile;
  long long unit_at;
  {
    const int cost = keys.tiles + L::UNIT_COST, m = static_cast<int>((at - seq_at) / cost);
    unit_at = seq_at + static_cast<long long>(m) * cost;
    unit_head = m / p.row_tiles;
    unit_tile = m - unit_head * p.row_tiles;
  }
  auto next_unit = [&](Unit& u) {
    u.valid = 0;
    while (at < stop && !u.valid) {
      const long long end = unit_at + keys.tiles + L::UNIT_COST;
      const int t0 = static_cast<int>(at - unit_at);
      const int t1 = static_cast<int>(stop - unit_at < keys.tiles ? stop - unit_at : keys.tiles);
      if (t0 < t1 || (keys.tiles == 0 && t0 == 0)) {
        const int shift = keys.sk - p.Sq;
        u.valid = 1;
        u.b = b;
        u.head = unit_head;
        u.r0 = unit_tile * L::ROWS;
        u.sk = keys.sk;
        u.t0 = keys.first + t0;
        u.t1 = keys.first + t1;
        u.which = t0 > 0 ? 0 : t1 < keys.tiles ? 1 : -1;
        u.tiles = keys.tiles;
        const int s_min = paged_token(p, u.r0), s_max = paged_token(p, min(rows - 1, u.r0 + L::ROWS - 1));
        u.hi = s_max + shift;
        u.hi_min = s_min + shift;
        u.lo_max = p.win_left >= 0 ? s_max + shift - p.win_left : 0;
        if (t0 > 0 && threadIdx.x == 0) {
          PagedPiece piece{at, unit_at, unit_at + keys.tiles, b, unit_head, u.r0, 0};
          p.pieces[blockIdx.x] = piece;
        }
      }
      at = end < stop ? end : stop;
      if (at < stop) {
        unit_at = end;
        if (++unit_tile == p.row_tiles) {
          unit_tile = 0;
          if (++unit_head == p.heads) {
            unit_head = 0;
            if (++b < p.B) keys = paged_keys<KEYS>(p, b);
            else stop = at;  // lengths that another stream has changed meanwhile
          }
        }
      }
    }
  };

  // ---- the warp's ring: fills and reads count on over all units -----------------------------------
  int filled = 0, read = 0;  // tiles since the start
  int run_page = -1, run_row = 0;  // of one of the 16 keys' runs of the unit's next tiles, a lane's each
  constexpr int AHEAD = 32 / RUNS;
  // A lane's copy: of K codes, V codes, K scales or V scales, run lane % RUNS, or, where pages hold whole tiles, both.
  const bool whole_tiles = p.c.page_size % KEYS == 0;
  const int copy_run = whole_tiles ? 0 : lane % RUNS, copy_of = whole_tiles ? lane : lane / RUNS;
  const bool of_codes = copy_of < 2, of_k = (copy_of & 1) == 0;
  const int64_t copy_page = of_codes ? (of_k ? p.c.kp : p.c.vp)[0] : 4 * (of_k ? p.c.ksp : p.c.vsp)[0];
  const int64_t copy_head = of_codes ? (of_k ? p.c.kp : p.c.vp)[1] : 4 * (of_k ? p.c.ksp : p.c.vsp)[1];
  const uint8_t* copy_base = of_codes ? static_cast<const uint8_t*>(of_k ? p.c.k : p.c.v)
                                      : reinterpret_cast<const uint8_t*>(of_k ? p.c.k_scales : p.c.v_scales);
  const int copy_unit = of_codes ? L::CODES : L::SCALES, copy_bytes = whole_tiles ? RUNS * copy_unit : copy_unit;
  const uint32_t copy_dst = copy_run * copy_unit + (of_codes ? (of_k ? 0 : L::V_OFF) : of_k ? L::KS_OFF : L::VS_OFF);
  // The runs' pages are looked up a batch of AHEAD tiles before they are needed: `soon` is this unit's next batch,
  // or, in its last one, the next unit's first.
  Unit u, next;
  int n_it, next_n = 0;  // the warp's tiles of the two
  int soon_page = -1, soon_row = 0;
  auto look_up = [&](const Unit& u, int i, int n) {
    const int j = i + lane / RUNS, key = (u.t0 + warp + j * PG_WARPS) * KEYS + (lane % RUNS) * PG_RUN;
    soon_page = -1;
    if (j < n && key < u.sk) {  // a run behind the last key is on a page of nobody's, perhaps
      soon_page = page_of(p.c, u.b, key);
      soon_row = key % p.c.page_size;
    }
  };
  auto fill = [&](const Unit& u, int i, int n) {  // the i-th of the warp's n tiles of a unit; the whole warp
    if (i % AHEAD == 0) {
      run_page = soon_page;
      run_row = soon_row;
      if (i + AHEAD < n) look_up(u, i + AHEAD, n);
      else if (i > 0) look_up(next, 0, next_n);
    }
    const int from = (i % AHEAD) * RUNS + (FOUR ? copy_run : 0);
    const int page = __shfl_sync(0xffffffffu, run_page, from), row = __shfl_sync(0xffffffffu, run_row, from);
    const int s = filled % STAGES;
    const uint32_t bar = bars + 8 * s, to = ring + s * L::STAGE_BYTES;
    ++filled;
    if (lane == 0) mbar_expect_tx(bar, L::STAGE_BYTES);
    if constexpr (FOUR) {
      __syncwarp();
      if (lane < (whole_tiles ? 4 : 4 * RUNS)) {
        const uint8_t* src =
            copy_base + page * copy_page + u.head * copy_head + row * (of_codes ? D / 2 : 8);
        bulk_load(to + copy_dst, page < 0 ? reinterpret_cast<const uint8_t*>(pg_zeros) : src,
                  copy_bytes, bar);
      }
    } else if (lane == 0) {
      const int head = u.head, from_page = page < 0 ? p.c.pages : page;  // none: zeros, behind the tensor
#pragma unroll
      for (int c = 0; c < L::CHUNKS; ++c) {
        tma_load_4d(to + c * L::CHUNK_BYTES, &p.tm_k, bar, c * 64, row, head, from_page);
        tma_load_4d(to + L::HALF_BYTES + c * L::CHUNK_BYTES, &p.tm_v, bar, c * 64, row, head, from_page);
      }
    }
  };
  auto tiles_of = [&](const Unit& u) { return u.valid ? max(0, (u.t1 - u.t0 - warp + PG_WARPS - 1) / PG_WARPS) : 0; };

  // (the sum of 4 bits goes by 1 / step_v, which has the factor)
  constexpr bool FP16_WEIGHTS = FOUR || !BF16;
  constexpr float O_DOWN = FP16_WEIGHTS ? 1.0f / PG_FP16_SCALE : 1.0f, L_DOWN = FOUR ? 1.0f : O_DOWN;
  const float sl2 = p.scale_log2;
  const bool has_alibi = p.slopes != nullptr;
  const int key_of_row = FOUR ? (g8 >> 1) + ((g8 & 1) << 2) : g8;  // 4 bits: 0, 4, 1, 5, 2, 6, 3, 7
  next_unit(u);
  if (p.splits > 1) {  // the unit's tiles alike
    const int share = (u.tiles + p.splits - 1) / p.splits, first = u.t0;
    u.t1 = first + min(u.tiles, (split + 1) * share);
    u.t0 = first + min(u.tiles, split * share);
  }
  n_it = skip ? 0 : tiles_of(u);
  look_up(u, 0, n_it);
  for (int i = 0; i < min(n_it, STAGES); ++i) fill(u, i, n_it);
  bool ok = true;

#pragma unroll 1
  while (u.valid) {
    next_unit(next);
    next_n = tiles_of(next);
    if (n_it <= AHEAD) look_up(next, 0, next_n);
    if (next.valid) {  // its queries, a 32nd of a row to a lane
      const int r = next.r0 + lane / 4, token = paged_token(p, r);
      if (r < rows)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint16_t*>(p.q) + next.b * p.q_stride_b +
                                                      token * p.q_stride_s +
                                                      ((next.head - token) * p.group + r) * p.q_stride_h +
                                                      t4 * (D / 4)));
    }
    float o[MTILES][NT][4];
    float m_run[NT][2], l_run[NT][2], low_run[NT][2];
    // Q: row 8 n + g8 of the tile is the operand's column g8. 4 bits: word w of a thread has the row's columns
    // t4 * D / 4 + 8 w .. + 7, which the ANDs below take as (0, 4), (1, 5), (2, 6), (3, 7), the second and the
    // fourth pair 16 times too large.
    uint32_t qf[NT][MTILES][2];
    float factor[NT][2], q_sum[NT][2], slope2[NT][2];  // of rows 8 n + 2 t4, + 1, the scores' columns
    int row_at[NT][2];                                 // their positions
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = u.r0 + 8 * n + (TWICE ? g8 & 3 : g8);
      const bool live = r < rows;
      const int rr = live ? r : rows - 1, token = paged_token(p, rr);
      const int h = u.head * p.group + rr - token * p.group;
      const uint16_t* qrow = reinterpret_cast<const uint16_t*>(p.q) + u.b * p.q_stride_b + token * p.q_stride_s +
                             h * p.q_stride_h;
      float down = sl2;
      if constexpr (FOUR) {
        using P = std::conditional_t<BF16, Pack<__nv_bfloat16>, Pack<__half>>;
        uint4 v[KW];
        auto top2 = P::absacc_init();
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          v[w] = live ? __ldg(reinterpret_cast<const uint4*>(qrow + t4 * (D / 4)) + w) : make_uint4(0u, 0u, 0u, 0u);
          P::absacc(v[w], top2);
        }
        float top = P::absacc_final(top2);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // the power of two that brings the row's largest value to 2^13 .. 2^14, and what takes it out again
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 16), 240);
        const float up = __uint_as_float(static_cast<unsigned>(267 - e) << 23);
        down = __uint_as_float(static_cast<unsigned>(e - 13) << 23) * 0x1p24f * sl2;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          float x[8];
          P::unpack(v[w], x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = i & 1 ? up * 0.0625f : up;
            qf[n][2 * w + i / 2][i & 1] = Pack<__half>::pack2(x[i] * f, x[i + 4] * f);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < MTILES; ++ks)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            qf[n][ks][c] = live ? __ldg(reinterpret_cast<const uint32_t*>(qrow + 16 * ks + 8 * c + 2 * t4)) : 0u;
      }
      const float slope = has_alibi ? p.slopes[h] * 1.4426950408889634f : 0.0f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * t4 + c);
        if constexpr (FOUR) {
          factor[n][c] = __shfl_sync(0xffffffffu, down, from);
        }
        slope2[n][c] = __shfl_sync(0xffffffffu, slope, from);
        row_at[n][c] = __shfl_sync(0xffffffffu, token, from) + u.sk - p.Sq;
      }
      if constexpr (FOUR) {
        // sum(q): the product with ones, and 16 where Q has a 16th
        const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x4C004C00u, 0x4C004C00u};
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < MTILES; ++ks) mma_16816<false>(sum, ones, qf[n][ks][0], qf[n][ks][1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) q_sum[n][c] = sum[c] * factor[n][c] * 0x1p-24f;
      }
    }

#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m_run[n][c] = PG_NOTHING;
        l_run[n][c] = low_run[n][c] = 0.0f;
      }
#pragma unroll
      for (int m = 0; m < MTILES; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[m][n][i] = 0.0f;
    }

    int next_fill = min(n_it, STAGES);
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
      const int st = read % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, (read / STAGES) & 1, no_result + warp, p.status,
                                             ATT_ST_SOFTMAX));
      if (!ok) break;
      ++read;
      constexpr int SUBS = L::STEP / PG_RUN;
#pragma unroll 1
      for (int step = 0; step < KEYS / L::STEP; ++step) {
        const uint32_t tile = ring + st * L::STAGE_BYTES + step * SUBS * L::CODES;
        const uint32_t scales = tile + L::KS_OFF + step * SUBS * (L::SCALES - L::CODES);
        const int c0 = (u.t0 + warp + it * PG_WARPS) * KEYS + step * L::STEP;
        if (c0 > u.hi) break;
        const bool need_mask = c0 + L::STEP - 1 > u.hi_min || c0 < u.lo_max;

        // scores of keys key_of_row (+ 8) of each run; 4 bits: weighed with V's step, x + log2 step_v
        float x[SUBS][NT][4];
        float v_low[SUBS][2], v_inv[SUBS][2];  // 4 bits
#pragma unroll
        for (int k = 0; k < SUBS; ++k) {
          float s[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
          if constexpr (FOUR) {
            uint32_t ka[KW], kb[KW];
            const uint32_t sub = tile + k * L::CODES + key_of_row * (D / 2) + t4 * (D / 8);
            lds_words<KW>(sub, ka);
            lds_words<KW>(sub + 8 * (D / 2), kb);
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
          } else {
            const int key = lane & 15, half = lane >> 4;  // ldmatrix rows: keys 0-15 by column halves
#pragma unroll
            for (int ks = 0; ks < MTILES; ++ks) {
              uint32_t f[4];
              const int col = (ks % 4) * 2 + half;
              ldsm_x4(tile + (ks / 4) * L::CHUNK_BYTES + key * 128 + ((col ^ (lane & 7)) << 4), f);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_16816<BF16>(s[n], f, qf[n][ks][0], qf[n][ks][1]);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key_of_row + 8 * e;
            if constexpr (FOUR) {
              const float2 ks = lds_float2(scales + k * L::SCALES + 8 * key);
              const float2 vs = lds_float2(scales + L::VS_OFF - L::KS_OFF + k * L::SCALES + 8 * key);
              // (of a row that is not a number `lowest` says so)
              const float v_step = fmaxf(vs.x, PG_LEAST_STEP);
              float log_step;
              asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(log_step) : "f"(v_step));
              asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(v_inv[k][e]) : "f"(v_step * PG_FP16_SCALE));
              v_low[k][e] = vs.y;
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  x[k][n][2 * e + c] =
                      fmaf(s[n][2 * e + c] * factor[n][c], ks.x, fmaf(q_sum[n][c], ks.y, log_step));
            } else {
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) x[k][n][2 * e + c] = s[n][2 * e + c] * sl2;
            }
          }
        }
        if (has_alibi) {
#pragma unroll
          for (int k = 0; k < SUBS; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int j = c0 + PG_RUN * k + key_of_row + 8 * (i >> 1);
                x[k][n][i] = fmaf(-slope2[n][i & 1], static_cast<float>(row_at[n][i & 1] - j), x[k][n][i]);
              }
        }
        if (need_mask) {
#pragma unroll
          for (int k = 0; k < SUBS; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int away = row_at[n][i & 1] - (c0 + PG_RUN * k + key_of_row + 8 * (i >> 1));
                if (away < 0 || (p.win_left >= 0 && away > p.win_left)) x[k][n][i] = -INFINITY;
              }
        }
        bool behind = false;
        float mx[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            mx[n][c] = fmaxf(x[0][n][c], x[0][n][2 + c]);
#pragma unroll
            for (int k = 1; k < SUBS; ++k) mx[n][c] = max3(mx[n][c], x[k][n][c], x[k][n][2 + c]);
            behind = behind || mx[n][c] > m_run[n][c] + ATT_LAZY_RESCALE;
          }
        if (__any_sync(0xffffffffu, behind)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float m = mx[n][c];
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
              if (m > m_run[n][c] + ATT_LAZY_RESCALE) {
                const float f = fast_exp2(m_run[n][c] - m);  // 0 where nothing was seen
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
        // The weights of the second product, and what their rounding takes off them, in a product of its own, or, where
        // a row has two columns, in the second one: the two together are within 2^-16 (fp16: 2^-22) of the fp32
        // weight, which the sum has whole. (64 sequences, 4 bits: 44.7 us with two columns to a row, 47.3 with a second
        // product, 44.4 with rounded weights alone; 48 sequences of 16 bits 71.8, 71.2, 70.6. Rounded weights alone are
        // up to a third farther off the definition than the output's own type.)
        // 16 bits: both are above 0, so that an infinite value stays infinite (down to weights of 2^-10, in fp16, where
        // the second one may be 0).
        // 4 bits: a key that a row does not see may be anything, behind the last one there is what was there.
        uint32_t pf[SUBS][NT][2], pr[SUBS][NT][2];
        auto weigh = [&](auto masked) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < SUBS; ++k)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float w[2], r[2];
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  w[c] = fast_exp2(x[k][n][2 * e + c] - (FP16_WEIGHTS ? m_run[n][c] - PG_FP16_UP : m_run[n][c]));
                const uint32_t first = FOUR ? pack16<false>(w[0], w[1]) : pack16_below<BF16>(w[0], w[1]);
                if constexpr (FP16_WEIGHTS) {
                  Pack<__half>::unpack2(first, r[0], r[1]);
                } else {
                  r[0] = __uint_as_float(first << 16);
                  r[1] = __uint_as_float(first & 0xffff0000u);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) r[c] = FOUR ? w[c] - r[c] : fmaxf(w[c] - r[c], w[c] * 0x1p-22f);
                const uint32_t rest = pack16<!FP16_WEIGHTS>(r[0], r[1]);
                pf[k][n][e] = transpose_8x8(TWICE && t4 >= 2 ? rest : first);
                if constexpr (!TWICE) pr[k][n][e] = transpose_8x8(rest);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  if constexpr (FOUR) {
                    const float prob = w[c] * v_inv[k][e];
                    float low = v_low[k][e];
                    if constexpr (decltype(masked)::value)
                      if (x[k][n][2 * e + c] == -INFINITY) low = 0.0f;
                    l_run[n][c] += prob;
                    low_run[n][c] = fmaf(prob, low, low_run[n][c]);
                  } else {
                    l_run[n][c] += w[c];
                  }
                }
              }
        };
        if (FOUR && need_mask) weigh(std::true_type{});
        else weigh(std::false_type{});
        if constexpr (FOUR) {
#pragma unroll
          for (int k = 0; k < SUBS; ++k) {
            const uint32_t sub = tile + L::V_OFF + k * L::CODES + t4 * (D / 2) + g8 * (D / 16);
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
                  for (int n = 0; n < NT; ++n) {
                    mma_16816<false>(o[4 * w + 2 * half + i][n], f, pf[k][n][0], pf[k][n][1]);
                    if constexpr (!TWICE) mma_16816<false>(o[4 * w + 2 * half + i][n], f, pr[k][n][0], pr[k][n][1]);
                  }
                  a >>= 8;
                  c >>= 8;
                }
              }
          }
        } else {
          // V of keys that no row sees may be anything: of keys 2 t4, 2 t4 + 1 of either half, those that `first` to
          // `last` has
          auto seen = [&](int first, int last, uint32_t (&keep)[2]) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = c0 + 8 * e + 2 * t4;
              keep[e] = (j >= first && j <= last ? 0xffffu : 0u) | (j + 1 >= first && j < last ? 0xffff0000u : 0u);
            }
          };
          const int key = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
          auto values = [&](int m, const uint32_t (&keep)[2], uint32_t (&f)[4]) {
            const int col = (m % 4) * 2 + half;
            ldsm_x4_trans(tile + L::HALF_BYTES + (m / 4) * L::CHUNK_BYTES + key * 128 + ((col ^ (lane & 7)) << 4), f);
            if (need_mask)
#pragma unroll
              for (int i = 0; i < 4; ++i) f[i] &= keep[i >> 1];
          };
          uint32_t keep[2];
          if (need_mask) seen(p.win_left >= 0 ? u.hi_min - p.win_left : 0, u.hi, keep);
          // where rows see different keys, a value that is not finite would reach those that do not see it, as 0 times it
          bool odd = false;
          if (need_mask && u.hi != u.hi_min) {
#pragma unroll
            for (int m = 0; m < MTILES; ++m) {
              constexpr uint32_t EXPONENT = BF16 ? 0x7F80u : 0x7C00u;
              uint32_t f[4];
              values(m, keep, f);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                odd = odd || (f[i] & EXPONENT) == EXPONENT || (f[i] >> 16 & EXPONENT) == EXPONENT;
            }
            odd = __any_sync(0xffffffffu, odd);
          }
          if (!odd) {
#pragma unroll
            for (int m = 0; m < MTILES; ++m) {
              uint32_t f[4];
              values(m, keep, f);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma_16816<BF16>(o[m][n], f, pf[0][n][0], pf[0][n][1]);
                if constexpr (!TWICE) mma_16816<BF16>(o[m][n], f, pr[0][n][0], pr[0][n][1]);
              }
            }
          } else {  // a row at a time, with the values that it sees
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll 1
              for (int r = 0; r < 8; ++r) {
                const int at = __shfl_sync(0xffffffffu, r & 1 ? row_at[n][1] : row_at[n][0], r >> 1);
                seen(p.win_left >= 0 ? at - p.win_left : 0, at, keep);
                const bool mine = t4 == r >> 1;
#pragma unroll
                for (int m = 0; m < MTILES; ++m) {
                  uint32_t f[4];
                  float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  values(m, keep, f);
                  mma_16816<BF16>(d, f, pf[0][n][0], pf[0][n][1]);
                  if constexpr (!TWICE) mma_16816<BF16>(d, f, pr[0][n][0], pr[0][n][1]);
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    if (mine && (i & 1) == (r & 1)) o[m][n][i] += d[i];
                }
              }
          }
        }
      }
      __syncwarp();  // every lane has read the tile
      if (next_fill < n_it) fill(u, next_fill++, n_it);
    }

    // ---- the next unit's first tiles, then this warp's partial result where the ring has room --------------
    if (ok) {
      for (int i = 0; i < min(next_n, STAGES - L::O_STAGES); ++i) fill(next, i, next_n);
    } else if (lane == 0) {
      no_result[warp] = 1;
      report_status(p.status);
    }
    // (a warp that gave up may still have copies on the way into its ring: it leaves no result)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int off = warp * L::RING_BYTES +
                      (L::O_STAGES > 1 ? ((filled + n) % STAGES) * L::STAGE_BYTES
                                       : (filled % STAGES) * L::STAGE_BYTES + n * L::O_BYTES);
      float* ow = reinterpret_cast<float*>(smem + off);
      if (lane == 0) o_at[warp * NT + n] = off;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 2 * t4 + c, swap = t4 << 3;  // a row's columns are 8 t4 apart from where they would be
        float l = l_run[n][c], low = low_run[n][c];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) {
          l += __shfl_xor_sync(0xffffffffu, l, w);
          if constexpr (FOUR) low += __shfl_xor_sync(0xffffffffu, low, w);
        }
        if (TWICE && t4 >= 2) low = 0.0f;  // the row's other column has it
        if (g8 == 0) {
          ml[warp * L::ROWS + 8 * n + r] = m_run[n][c];
          ml[(PG_WARPS + warp) * L::ROWS + 8 * n + r] = l * L_DOWN;
        }
        if (ok)
#pragma unroll
          for (int m = 0; m < MTILES; ++m) {
            if constexpr (FOUR) {  // columns 2 m, 2 m + 1 of this lane's D / 8
              *reinterpret_cast<float2*>(ow + r * D + ((g8 * (D / 8) + 2 * m) ^ swap)) =
                  make_float2(fmaf(o[m][n][c], 0x1p24f * O_DOWN, low), fmaf(o[m][n][2 + c], 0x1p20f * O_DOWN, low));
            } else {
              ow[r * D + ((16 * m + g8) ^ swap)] = o[m][n][c] * O_DOWN;
              ow[r * D + ((16 * m + 8 + g8) ^ swap)] = o[m][n][2 + c] * O_DOWN;
            }
          }
      }
    }
    __syncthreads();
    bool complete = true;  // every warp has a result; else nothing is written
#pragma unroll
    for (int w = 0; w < PG_WARPS; ++w) complete = complete && no_result[w] == 0;
    complete = complete && !skip;
    if (!complete && p.splits < 2) break;

    // the sum of the warps' results: weights 2^(m_i - max m), 0 for an empty part
    const int live_rows = min(L::ROWS, rows - u.r0);
    float* part = u.which < 0 || p.splits ? nullptr : paged_part<D, FOUR, NT>(p, blockIdx.x, u.which);
    for (int idx = threadIdx.x; idx < live_rows * (D / 4); idx += PG_THREADS) {
      const int r = idx / (D / 4), c4 = idx % (D / 4);
      float top = PG_NOTHING, l = 0.0f;
#pragma unroll
      for (int w = 0; w < PG_WARPS; ++w) top = fmaxf(top, ml[w * L::ROWS + r]);
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < PG_WARPS; ++w) {
        const float f = fast_exp2(ml[w * L::ROWS + r] - top);
        const float* from = reinterpret_cast<const float*>(smem + o_at[w * NT + (r >> 3)]);
        float4 v = *reinterpret_cast<const float4*>(from + (r & 7) * D + ((4 * c4) ^ (((r & 7) >> 1) << 3)));
        if constexpr (TWICE) {
          const float4 rest = *reinterpret_cast<const float4*>(from + (r + 4) * D + ((4 * c4) ^ (((r + 4) >> 1) << 3)));
          v = make_float4(v.x + rest.x, v.y + rest.y, v.z + rest.z, v.w + rest.w);
        }
        l = fmaf(f, ml[(PG_WARPS + w) * L::ROWS + r], l);
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
      if (p.splits > 1) {  // this thread's own elements
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(smem + o_at[r >> 3]) + (r & 7) * D +
                                   ((4 * c4) ^ (((r & 7) >> 1) << 3))) = acc;
        if (c4 == 0) {
          cta_ml[r] = top;
          cta_ml[L::ROWS + r] = l;
        }
      } else if (part) {
        *reinterpret_cast<float4*>(part + r * D + 4 * c4) = acc;
        if (c4 == 0) {
          part[L::ROWS * D + r] = top;
          part[L::ROWS * (D + 1) + r] = l;
        }
      } else {
        paged_emit<D, BF16>(p, u.b, u.head, u.r0 + r, c4, acc, top, l);
      }
    }
    if (p.splits > 1) {
      namespace cg = cooperative_groups;
      cg::cluster_group cluster = cg::this_cluster();
      if (threadIdx.x == 0) no_result[PG_WARPS] = complete ? 0 : 1;
      cluster.sync();
      int* flags = reinterpret_cast<int*>(smem + L::FLAG_OFF);
      static_assert(PG_MOST_SPLITS <= 32, "one lane per CTA");
      complete = __all_sync(0xffffffffu, lane >= p.splits || cluster.map_shared_rank(flags, lane)[PG_WARPS] == 0);
      for (int idx = split * PG_THREADS + threadIdx.x; complete && idx < live_rows * (D / 4);
           idx += p.splits * PG_THREADS) {
        const int r = idx / (D / 4), c4 = idx % (D / 4);
        float top = PG_NOTHING, l = 0.0f;
        for (int k = 0; k < p.splits; ++k) top = fmaxf(top, cluster.map_shared_rank(cta_ml, k)[r]);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < p.splits; ++k) {
          const float* kml = cluster.map_shared_rank(cta_ml, k);
          const float f = fast_exp2(kml[r] - top);
          const int off = cluster.map_shared_rank(o_at, k)[r >> 3];
          const float4 v = *reinterpret_cast<const float4*>(
              reinterpret_cast<const float*>(cluster.map_shared_rank(smem, k) + off) + (r & 7) * D +
              ((4 * c4) ^ (((r & 7) >> 1) << 3)));
          l = fmaf(f, kml[L::ROWS + r], l);
          acc.x = fmaf(f, v.x, acc.x);
          acc.y = fmaf(f, v.y, acc.y);
          acc.z = fmaf(f, v.z, acc.z);
          acc.w = fmaf(f, v.w, acc.w);
        }
        paged_emit<D, BF16>(p, u.b, u.head, u.r0 + r, c4, acc, top, l);
      }
      cluster.sync();  // no CTA leaves while another one reads its shared memory
      break;
    }
    __syncthreads();  // all of it has been read: the ring has its room back
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    u = next;
    n_it = next_n;
    for (int i = min(n_it, STAGES - L::O_STAGES); i < min(n_it, STAGES); ++i) fill(u, i, n_it);
  }
  // Copies on their way, where a warp of this CTA gave up: wait for them (bounded) before the CTA ends.
  for (; read < filled; ++read) {
    const uint64_t t0 = global_ns();
    bool done = false;
    while (!done && global_ns() - t0 < ATT_WAIT_NS) {
      done = mbar_try_wait(bars + 8 * (read % STAGES), (read / STAGES) & 1);
    }
    if (!done) atomicOr(p.status, ATT_ST_DRAIN);
  }
}

// The units that CTAs of the first launch share: block (c, y) has two rows of the one that CTA c + 1 found begun, if
// CTA c began it. A unit may have as many parts as there are CTAs: the rows' weights are made first, by as many
// threads as there are parts, then groups of threads add up every PG_GROUPS-th part, eight loads in flight (one
// after the other, 2 x 131072 keys, 56 parts to a unit, took 27 us).
constexpr int PG_MERGE_ROWS = 2, PG_MERGE_THREADS = 256;
template <int D, bool BF16, bool FOUR, int NT>
__global__ void __launch_bounds__(PG_MERGE_THREADS) attn_paged_merge_kernel(const __grid_constant__ PagedParams p) {
  using L = PgShape<D, FOUR, NT>;
  constexpr int ITEMS = PG_MERGE_ROWS * D / 4, GROUPS = PG_MERGE_THREADS / ITEMS;  // float4 of the rows
  __shared__ float weight[PG_MOST_CTAS][PG_MERGE_ROWS], sum[PG_MOST_CTAS][PG_MERGE_ROWS];
  __shared__ float red[2][PG_MERGE_THREADS / 32][PG_MERGE_ROWS];
  __shared__ float4 sums[GROUPS][ITEMS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x + 1, ctas = gridDim.x + 1;
  const PagedPiece piece = p.pieces[c];
  const long long began = p.pieces[c - 1].lo;
  const bool failed = *reinterpret_cast<volatile unsigned int*>(p.status) != 0u;
  // the first of the CTAs that may have tiles of the unit: `lo` ascends
  long long lo = p.pieces[min(c + static_cast<int>(threadIdx.x), ctas - 1)].lo;
  if (piece.unit < 0 || piece.unit < began) return;
  const int rows = p.group * p.Sq, r0 = piece.r0, row0 = PG_MERGE_ROWS * blockIdx.y;
  if (r0 + row0 >= rows || failed) return;
  int parts = 1;  // CTAs c - 1 .. c - 2 + parts
  for (int k = c;;) {
    const int n = __syncthreads_count(k + static_cast<int>(threadIdx.x) < ctas && lo < piece.end);
    parts += n;
    if (n < PG_MERGE_THREADS) break;
    k += PG_MERGE_THREADS;
    lo = p.pieces[min(k + static_cast<int>(threadIdx.x), ctas - 1)].lo;
  }
  auto part = [&](int k) { return paged_part<D, FOUR, NT>(p, c - 1 + k, k > 0 ? 0 : 1); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = threadIdx.x / ITEMS, item = threadIdx.x % ITEMS, r = item / (D / 4), c4 = item % (D / 4);
  // a thread's first parts of O, on their way with the rows' maxima and sums
  constexpr int EARLY = 8;
  float4 o[EARLY];
#pragma unroll
  for (int i = 0; i < EARLY; ++i) {
    const int k = group + i * GROUPS;
    o[i] = k < parts ? *reinterpret_cast<const float4*>(part(k) + (row0 + r) * D + 4 * c4)
                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  float top[PG_MERGE_ROWS], l[PG_MERGE_ROWS];
#pragma unroll
  for (int r = 0; r < PG_MERGE_ROWS; ++r) {
    top[r] = PG_NOTHING;
    for (int k = threadIdx.x; k < parts; k += PG_MERGE_THREADS) {
      const float m = part(k)[L::ROWS * D + row0 + r];
      weight[k][r] = m;
      sum[k][r] = part(k)[L::ROWS * (D + 1) + row0 + r];
      top[r] = fmaxf(top[r], m);
    }
  }
#pragma unroll
  for (int r = 0; r < PG_MERGE_ROWS; ++r) {
    top[r] = warp_reduce<true>(top[r]);
    if (lane == 0) red[0][warp][r] = top[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < PG_MERGE_ROWS; ++r) {
#pragma unroll
    for (int w = 0; w < PG_MERGE_THREADS / 32; ++w) top[r] = fmaxf(top[r], red[0][w][r]);
    l[r] = 0.0f;
    for (int k = threadIdx.x; k < parts; k += PG_MERGE_THREADS) {
      const float f = fast_exp2(weight[k][r] - top[r]);
      weight[k][r] = f;
      l[r] = fmaf(f, sum[k][r], l[r]);
    }
    l[r] = warp_reduce<false>(l[r]);
    if (lane == 0) red[1][warp][r] = l[r];
  }
  __syncthreads();
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](int k, const float4& v) {
    const float f = weight[k][r];
    acc.x = fmaf(f, v.x, acc.x);
    acc.y = fmaf(f, v.y, acc.y);
    acc.z = fmaf(f, v.z, acc.z);
    acc.w = fmaf(f, v.w, acc.w);
  };
#pragma unroll
  for (int i = 0; i < EARLY; ++i)
    if (group + i * GROUPS < parts) add(group + i * GROUPS, o[i]);
#pragma unroll 8
  for (int k = group + EARLY * GROUPS; k < parts; k += GROUPS)
    add(k, *reinterpret_cast<const float4*>(part(k) + (row0 + r) * D + 4 * c4));
  sums[group][item] = acc;
  __syncthreads();
  if (group == 0 && r0 + row0 + r < rows) {
    float total = 0.0f, most = PG_NOTHING;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
      const float4 v = sums[g][item];
      acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
    }
#pragma unroll
    for (int w = 0; w < PG_MERGE_THREADS / 32; ++w) {
      total += red[1][w][r];
      most = fmaxf(most, red[0][w][r]);
    }
    paged_emit<D, BF16>(p, piece.b, piece.head, r0 + row0 + r, c4, acc, most, total);
  }
}

// How a call is cut: CTAs, and bytes of the parts.
struct PagedPlan {
  int64_t ctas;
  int splits;  // 0: one line
  size_t pieces_bytes, bytes;
};
template <int D, bool FOUR, int NT>
static PagedPlan paged_plan(int64_t units, int64_t keys) {
  using L = PgShape<D, FOUR, NT>;
  PagedPlan plan{};
  const int64_t tiles = (keys + L::KEYS - 1) / L::KEYS;
  const int64_t slots = static_cast<int64_t>(sm_count_of_current_device()) * L::CTAS_PER_SM;
  // clusters of as many CTAs as leave a warp two tiles (4 bits: one), within one wave
  int n = 1;
  while (n < PG_MOST_SPLITS && units * 2 * n <= slots && tiles >= 2 * n * PG_WARPS * (FOUR ? 1 : 2)) n *= 2;
  const int64_t chain = (tiles + n * PG_WARPS - 1) / (n * PG_WARPS);
  // More than a few tiles to a warp, or units that do not all run at once: the line. Line / clusters, us, 16 bits and 4,
  // 32 / 8 heads x 128, sequences of up to so many keys; first units that run at once (so many tiles to a warp):
  //   16 bits: 1 of 600 (3) 11.7 / 8.9, 16 of 500 (4) 12.6 / 9.6, 1 of 4096 (8) 12.3 / 13.0, 16 of 2000 (16) 15.2 / 19.9, 1
  //   of 32768 (64) 32.1 / 55.3. 4 bits: 1 of 600 (2) 13.0 / 10.4, 16 of 500 (1) 15.1 / 9.7, 16 of 2000 (4) 16.4 / 15.3,
  //   16 of 8000 (16) 21.9 / 38.8.
  // and the others: 16 bits: 64 of 100 (2) 14.4 / 11.2, 64 of 500 (8) 17.8 / 15.8, 256 of 250 (4) 36.0 / 40.5, 64 of 1000
  //   (16) 22.5 / 23.2. 4 bits: 64 of 250 (1) 16.6 / 13.5, 64 of 500 (2) 17.6 / 15.1, 64 of 1000 (4) 19.7 / 18.1, 256 of
  //   600 (3) 40.3 / 39.8, 64 of 2048 (8) 25.3 / 27.1.
  // `keys` is what the block table has room for: the lengths are the device's.
  const bool line = chain > (units * n <= slots ? (FOUR ? 5 : 16) : (FOUR ? 2 : 3));
  plan.splits = line ? 0 : n;
  plan.ctas = !line ? units * n : slots < PG_MOST_CTAS ? slots : PG_MOST_CTAS;
  if (line) {
    plan.pieces_bytes = plan.ctas * sizeof(PagedPiece);
    plan.bytes = plan.pieces_bytes + plan.ctas * 2 * L::PART_FLOATS * sizeof(float);
  }
  return plan;
}

template <int D, bool BF16, bool FOUR, int NT, bool TWICE>
static int launch_paged(PagedParams& p, const PagedPlan& plan, cudaStream_t stream) {
  using L = PgShape<D, FOUR, NT>;
  auto kernel = attn_paged_kernel<D, BF16, FOUR, NT, TWICE>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TRX_ERR_CUDA;
  const bool cacheable = dev >= 0 && dev < 64;
  if (!cacheable || !configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN_BYTES) != cudaSuccess)
      return TRX_ERR_CUDA;
    if (cacheable) configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = plan.splits > 1 ? plan.splits : 1;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(plan.ctas));
  cfg.blockDim = dim3(PG_THREADS);
  cfg.dynamicSmemBytes = L::DYN_BYTES;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return TRX_ERR_CUDA;
  if (plan.splits || plan.ctas < 2) return TRX_OK;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(plan.ctas - 1), L::ROWS / PG_MERGE_ROWS);
  cfg.blockDim = dim3(PG_MERGE_THREADS);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attn_paged_merge_kernel<D, BF16, FOUR, NT>, p) == cudaSuccess ? TRX_OK : TRX_ERR_CUDA;
}

}  // namespace trx
