// Device-side view of a paged cache: what the append and the attention kernels share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged.h"

namespace ti {

struct PagedView {
  int8_t* k_pages;
  int8_t* v_pages;
  const int* table;
  const int* query_starts;
  const int* kv_lens;
  long long table_ld;
  int table_width;  // pages a row of the block table holds
  int num_pages, kv_heads, page_shift;
  int batch, tokens, max_query_len;
  int* status;
};

inline PagedView make_paged_view(const PagedBatch& b, int* status) {
  PagedView v;
  v.k_pages = b.k_pages;
  v.v_pages = b.v_pages;
  v.table = b.block_table;
  v.query_starts = b.query_starts;
  v.kv_lens = b.kv_lens;
  v.table_ld = b.table_ld;
  v.table_width = static_cast<int>(b.table_width);
  v.num_pages = static_cast<int>(b.num_pages);
  v.kv_heads = static_cast<int>(b.kv_heads);
  v.page_shift = 0;
  while ((1ll << v.page_shift) < b.page_size) ++v.page_shift;
  v.batch = static_cast<int>(b.batch);
  v.tokens = static_cast<int>(b.tokens);
  v.max_query_len = static_cast<int>(b.max_query_len < b.tokens ? b.max_query_len : b.tokens);
  v.status = status;
  return v;
}

struct PagedSeq {
  int q0;  // first new token
  int T;   // new tokens
  int L;   // keys, new ones included
};

// The lengths of sequence b.  false (and status 211) where they disagree with the number of tokens, the
// caller's bounds or the block table: nothing of such a sequence is read or written.
__device__ __forceinline__ bool paged_sequence(const PagedView& v, int b, int max_kv_len, PagedSeq* s) {
  const int q0 = v.query_starts[b], q1 = v.query_starts[b + 1], L = v.kv_lens[b];
  s->q0 = q0;
  s->T = q1 - q0;
  s->L = L;
  const bool ok = q0 >= 0 && q1 >= q0 && q1 <= v.tokens && q1 - q0 <= v.max_query_len && L >= 0 && L <= max_kv_len &&
                  ((static_cast<long long>(L) + (1 << v.page_shift) - 1) >> v.page_shift) <= v.table_width;
  if (!ok) atomicCAS(v.status, 0, static_cast<int>(TI_ERR_PAGED_LENGTHS));
  return ok;
}

// A block table entry that is in use.  One outside the pool sets status 212 and gives -1.
__device__ __forceinline__ int paged_checked(const PagedView& v, int page) {
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(v.num_pages)) {
    atomicCAS(v.status, 0, static_cast<int>(TI_ERR_PAGED_PAGE));
    return -1;
  }
  return page;
}
// Page of block table entry `i` of sequence b.
__device__ __forceinline__ int paged_page(const PagedView& v, int b, int i) {
  return paged_checked(v, v.table[b * v.table_ld + i]);
}

}  // namespace ti
