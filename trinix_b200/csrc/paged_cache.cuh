// A cache of keys and values in pages: what append_paged, gather_paged and attention_paged share.
//
// Pages are (pages, kv heads, page size, head_dim), of 16 bits or of 4; a sequence's row `block_table[b]` names
// its pages in order. Position p of a sequence is row p % size of page block_table[b][p / size]. A page number
// outside the cache (unused entries are -1) names no memory: nothing is written there, and zeros are read.
//
// 4 bits: a row x of head_dim values is held as codes 0 .. 15 and two fp32 numbers,
//   lowest = min x,  step = (max x - lowest) fp32(1/15),  code = rint(15 (x - lowest) / (max x - lowest)),
//   value = lowest + code * step
// (step 0 and codes 0 where the values are within 2^-76 of each other, both numbers NaN where a value is not finite
// or they are more than 2^120 apart); byte j of the codes is column 2 j in its low bits and 2 j + 1 in its high ones.
// A row (and not a group of its columns) has one step, because then the step comes out of both of attention's
// products: it scales a key's score and a value's probability, and the matrix instructions see the codes themselves.
#pragma once

#include "common.cuh"

namespace trx {

struct PagedCache {
  void* k;
  void* v;
  float* k_scales;  // (pages, kv heads, page size, 2): step, lowest; null: 16 bits
  float* v_scales;
  int64_t kp[3], vp[3];  // (page, head, row) strides: elements, of 4 bits bytes
  int64_t ksp[2], vsp[2];  // (page, head) strides of the scales
  const int* table;
  int64_t table_stride;
  int pages, page_size, width;  // width: entries of a table's row
};

// A C entry's arguments, checked: n_seq rows of the block table; strides as in the public header.
int make_paged_cache(PagedCache* c, const void* k_pages, const void* v_pages, const float* k_scales,
                     const float* v_scales, const int32_t* block_table, int64_t n_seq, int64_t Hk, int64_t D,
                     int64_t pages, int64_t page_size, int64_t width, const int64_t* strides);

// The page of position `pos`, or -1.
__device__ __forceinline__ int page_of(const PagedCache& c, int64_t b, int pos) {
  const int i = pos / c.page_size;
  if (pos < 0 || i >= c.width) return -1;
  const int page = __ldg(c.table + b * c.table_stride + i);
  return page >= 0 && page < c.pages ? page : -1;
}

// The sequence of a packed row: the last of n whose first row is not behind it. Bounds as they are.
__device__ __forceinline__ int sequence_of(const int* cu, int n, int row) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace trx
