// The decode attention kernel's state instances: every (row, query head)'s softmax state (m, l, O)
// over its own KV tokens, for attention over a shared prefix (dk_serving.cu) to merge.
#include "dk_attention_host.cuh"
#include "dk_attention_state.h"

namespace dk {
namespace host {

cudaError_t attention_state_status(int clear, int* code, int* detail) { return unit_status(clear, code, detail); }

int attention_state(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k, const void* v,
                    int64_t kv_stride_seq, int64_t kv_stride_head, int64_t kv_stride_tok, int64_t kv_n_seq,
                    int64_t kv_capacity, const int32_t* kv_lens, const int32_t* row_tiles, int32_t n_tiles,
                    int32_t n_rows, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len,
                    float scale, int dtype, void* workspace, size_t workspace_bytes, void* stream, const PagedKV* pg,
                    const char* what, float* st_o, float* st_ml) {
  return attention_invariant_impl<true>(q, q_stride_row, q_stride_head, k, v, kv_stride_seq, kv_stride_head,
                                        kv_stride_tok, kv_n_seq, kv_capacity, nullptr, 0, 0, kv_lens, 0, row_tiles,
                                        n_tiles, n_rows, n_q_heads, n_kv_heads, head_dim, max_kv_len, scale, dtype,
                                        workspace, workspace_bytes, stream, pg, what, st_o, st_ml);
}

}  // namespace host
}  // namespace dk
