// Host-side description of a ragged batch over a paged int8 key/value cache, shared by the append
// (paged_append.cu) and attention (paged_attention.cu) launchers and their kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ti {

// Sequence b brings the new tokens [query_starts[b], query_starts[b + 1]) and holds kv_lens[b] keys, the
// new ones included.  Position p of it lies in page block_table[b * table_ld + (p >> page_shift)], row
// p & (page_size - 1); both pools are [num_pages][kv_heads][page_size][head_dim] int8.  All three index
// arrays are device memory: a step has no host parameters that change with the lengths.
struct PagedBatch {
  int8_t* k_pages = nullptr;
  int8_t* v_pages = nullptr;
  const int32_t* block_table = nullptr;
  const int32_t* query_starts = nullptr;
  const int32_t* kv_lens = nullptr;
  int64_t num_pages = 0, kv_heads = 0, page_size = 0, head_dim = 0;
  int64_t table_ld = 0, table_width = 0;
  int64_t batch = 0, tokens = 0;
  int64_t max_query_len = 0;  // upper bound of a sequence's new tokens
};

struct PagedAppend {
  const void* q = nullptr;  // optional
  const void* k = nullptr;
  const void* v = nullptr;
  int dtype = 0;                            // 0 fp32, 1 fp16, 2 bf16, 3 int8
  int64_t ld_q = 0, ld_k = 0, ld_v = 0;     // elements between tokens; heads and columns packed
  int64_t q_heads = 0;
  float q_alpha = 1.f, k_alpha = 1.f, v_alpha = 1.f;
  const float* rotary = nullptr;            // [rotary_rows][rotary_dim]: cosines, then sines
  int64_t rotary_rows = 0, rotary_dim = 0;
  int interleaved = 0;
  int8_t* q_out = nullptr;                  // [tokens][q_heads][head_dim]
};

struct PagedAttention {
  const int8_t* q = nullptr;                // [tokens][q_heads][head_dim], tokens ld_q apart
  int64_t ld_q = 0, q_heads = 0;
  int64_t max_kv_len = 0;                   // upper bound of kv_lens
  float alpha_qk = 1.f, alpha_pv = 1.f;
  void* out = nullptr;                      // [tokens][q_heads][head_dim]
  int out_kind = 0;                         // 1 fp16, 2 bf16, 3 int8
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

// Status codes of the device status word (0 = ok).
enum : int {
  TI_ERR_PAGED_LENGTHS = 211,  // query_starts / kv_lens disagree with the tokens, the bounds or the block table
  TI_ERR_PAGED_PAGE = 212,     // a block table entry is outside the pool
};

// Common argument checks; name = the entry point for the message.  0 or TI_E_INVALID.
int check_paged_batch(const PagedBatch& b, const char* name);
int paged_append(const PagedBatch& b, const PagedAppend& a, cudaStream_t stream);
int paged_attention(const PagedBatch& b, const PagedAttention& a, cudaStream_t stream);
int64_t paged_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t max_query_len, int64_t max_kv_len);

}  // namespace ti
