// What the operators over a paged KV cache share: number types, division by a launch constant, and the
// batch a step runs on (include/q4llm.h, q4_paged_kv).
#pragma once

#include "q4_common.h"

namespace q4 {

// n / d and n % d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and m = floor(2^(31 + s) / d) + 1 the
// product n m / 2^(31 + s) lies in [n / d, n / d + n / 2^(31 + s)), and the second term is below 1 / d.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    uint32_t l = 0;
    while ((uint64_t{1} << l) < div) ++l;
    s = l;
    m = static_cast<uint32_t>((uint64_t{1} << (31 + l)) / div + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * m) >> (31 + s));
  }
};

// 16-bit storage <-> fp32, round to nearest even.
template <int DT>
struct Num;
template <>
struct Num<Q4_F32> {
  typedef float type;
};
template <>
struct Num<Q4_F16> {
  typedef _Float16 type;
};
template <>
struct Num<Q4_BF16> {
  typedef __bf16 type;
};

// The batch of a step, checked on the host; see q4_paged_kv.
struct PagedBatch {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  int64_t stride;
  int num_pages, page_size, max_pages, batch;
  int rows;  // tokens of each sequence where cu is null
  FastDiv by_rows, by_page;

  // Row of the cache that entry `page` of a page list gives at offset `off`, -1 for no page of the pool.
  __device__ __forceinline__ int slot(int page, int off) const {
    return page >= 0 && page < num_pages ? page * page_size + off : -1;
  }
};

// Checks of the cache and the batch for T tokens of dtype; fills `b`.
inline int paged_batch(const q4_paged_kv* kv, int dtype, int64_t T, PagedBatch* b) {
  if (!kv || !kv->k_cache || !kv->v_cache || !kv->page_table || !kv->seq_lens) return Q4_ERR_NULL;
  if (kv->dtype != Q4_F16 && kv->dtype != Q4_BF16) return Q4_ERR_DTYPE;
  if (kv->dtype == Q4_BF16 ? dtype != Q4_BF16 : (dtype != Q4_F32 && dtype != Q4_F16)) return Q4_ERR_DTYPE;
  if (kv->batch <= 0 || kv->n_kv <= 0 || kv->head_dim <= 0 || kv->page_size <= 0 || kv->max_pages <= 0 ||
      kv->num_pages <= 0 || T < 0 || T > INT32_MAX)
    return Q4_ERR_SHAPE;
  if (kv->num_pages > INT32_MAX / kv->page_size || kv->table_stride < kv->max_pages) return Q4_ERR_SHAPE;
  if (!kv->cu_q && T % kv->batch) return Q4_ERR_SHAPE;
  if (!aligned(kv->page_table, 4) || !aligned(kv->seq_lens, 4) || !aligned(kv->cu_q, 4)) return Q4_ERR_ALIGN;
  b->table = kv->page_table;
  b->lens = kv->seq_lens;
  b->cu = kv->cu_q;
  b->stride = kv->table_stride;
  b->num_pages = static_cast<int>(kv->num_pages);
  b->page_size = kv->page_size;
  b->max_pages = kv->max_pages;
  b->batch = kv->batch;
  b->rows = kv->cu_q ? 0 : static_cast<int>(T / kv->batch);
  b->by_rows = FastDiv(static_cast<uint32_t>(b->rows > 0 ? b->rows : 1));
  b->by_page = FastDiv(static_cast<uint32_t>(kv->page_size));
  return Q4_OK;
}

}  // namespace q4
