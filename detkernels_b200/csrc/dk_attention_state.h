// Interface between the attention translation units.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace dk {
namespace host {

// Paged KV description (null: a contiguous [n_seq, heads, capacity, d] cache).
struct PagedKV {
  const int32_t* table;
  int64_t table_stride;
  int32_t page;
  int32_t blocks_per_seq;
  int64_t n_blocks;
};

// Softmax states of every row over its own KV tokens (arguments as dk_attention_batch_invariant /
// _paged_ without the output): st_o [n_rows][n_q_heads][head_dim], st_ml [n_rows][n_q_heads][2].  Must
// follow, on the same stream, a kernel of the same call that waits for its own predecessors.
int attention_state(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k, const void* v,
                    int64_t kv_stride_seq, int64_t kv_stride_head, int64_t kv_stride_tok, int64_t kv_n_seq,
                    int64_t kv_capacity, const int32_t* kv_lens, const int32_t* row_tiles, int32_t n_tiles,
                    int32_t n_rows, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len,
                    float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream, const PagedKV* pg,
                    const char* what, float* st_o, float* st_ml);

}  // namespace host
}  // namespace dk
