/*
 * detkernels_b200 -- C ABI of the batch-invariant kernel library for NVIDIA B200 (sm_100a).
 *
 * Every entry point takes raw device pointers, element strides, sizes, a CUDA
 * stream (passed as void*, i.e. a cudaStream_t) and, where the kernel needs
 * scratch space, a caller-provided device workspace.  The library never
 * allocates device memory.  Launches are asynchronous on the given stream; the
 * return value reports argument validation and launch errors only.  Errors
 * detected on the device (a bounded wait that expired, an index outside the
 * caller's buffers) are recorded in a per-device status word that
 * dk_device_status() reads and clears.
 *
 * Each compute entry point names the reference interface it replaces
 * (AdityaShome/DetKernels, Python + Triton):
 *   kernels/rmsnorm.py, kernels/matmul.py, kernels/attention.py.
 *
 * Batch invariance contract: for every entry point marked "invariant", the
 * bits written for one output row depend only on that row's inputs (and, for
 * attention, that row's own KV sequence and length) -- never on how many other
 * rows are in the call, what they contain, or which work schedule the library
 * picked for the call.
 */
#ifndef DETKERNELS_B200_H
#define DETKERNELS_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---- */
#define DK_OK 0
#define DK_ERR_INVALID_ARGUMENT 1 /* shape, stride, pointer or alignment rejected */
#define DK_ERR_UNSUPPORTED 2      /* dtype / head_dim / size combination not built */
#define DK_ERR_WORKSPACE 3        /* workspace missing or smaller than *_workspace_size() */
#define DK_ERR_CUDA 4             /* a CUDA runtime or driver call failed */
#define DK_ERR_DEVICE_TIMEOUT 5   /* a bounded device-side wait expired (see detail) */
#define DK_ERR_DEVICE_CHECK 6     /* a device-side index check failed (see detail) */

/* ---- workspaces ----
 * Every workspace starts with DK_WORKSPACE_COUNTER_BYTES of arrival counters shared by all entry
 * points.  Zero that area once when the workspace is created; every call leaves it zero again (after
 * a device-side error, zero it again).  Scratch data always lives after it.  Calls that may overlap
 * on the GPU (different streams) need different workspaces. */
#define DK_WORKSPACE_COUNTER_BYTES (1u << 20)

/* ---- dtype codes ---- */
#define DK_F32 0
#define DK_F16 1
#define DK_BF16 2

/* ---- fixed numerics of the invariant kernels (part of the output definition) ---- */
#define DK_MATMUL_K_SLICES 8        /* K is reduced as 8 fixed slices, summed along a fixed f32 tree */
#define DK_ATTN_KV_SPLIT 256        /* decode attention reduces KV in fixed splits of 256 tokens */
#define DK_RMSNORM_THREADS 256      /* one CTA of 256 threads per row */

/* ---- library / device queries ---- */
/* Layout version of this header's structs and signatures; dk_abi_version() of a library built from it
 * returns the same number.  2: dk_matmul_epilogue gained the DK_EPI_RESIDUAL_RMSNORM fields.
 * 3: dk_matmul_epilogue gained the paged-KV fields (block_table ... n_blocks). */
#define DK_ABI_VERSION 3
int dk_abi_version(void);
/* Message for the last non-zero return code on the calling host thread. */
const char* dk_last_error(void);
/* Reads the device status word of `device` (synchronises that device).  If
 * `clear` is non-zero the word is reset to DK_OK afterwards. */
int dk_device_status(int device, int clear, int* code, int* detail);
int dk_num_sms(int device, int* out);
/* Introspection of the compiled kernels on the current device (registers per thread, the
 * launch-time thread limit, local-memory bytes, dynamic shared-memory limit).  which: 0 = bf16
 * GEMM, 1 = bf16 decode attention d128, 2 = bf16 decode attention d64, 3 = f32 RMSNorm. */
int dk_kernel_attributes(int which, int* num_regs, int* max_threads, int* local_bytes, int* max_dynamic_smem);
/* Self-test of the device-side bounded wait that every kernel of this library uses: one CTA waits on
 * a shared-memory barrier for at most limit_ns (0 < limit_ns <= 100 ms).  A second warp arrives on it
 * unless skip_arrive is non-zero; then the wait runs out, the kernel records DK_ERR_DEVICE_TIMEOUT
 * (detail 0x7E57) in the device status word and returns -- the context stays usable.  No counterpart
 * in the reference (its Triton kernels have no bounded waits). */
int dk_test_bounded_wait(int skip_arrive, int64_t limit_ns, void* stream);

/* ---- RMSNorm: y = x * rsqrt(mean(x^2) + eps) * w, f32 math, y in x's dtype ----
 * x, out: [n_rows, n_cols] with unit column stride and the given row strides
 * (elements).  dtype: DK_F32 / DK_F16 / DK_BF16 for x and out; weight_dtype
 * for w (any of the three). */

/* replaces kernels/rmsnorm.py:155-177 rmsnorm_batch_invariant (+ _single_block_kernel 63-89) */
int dk_rmsnorm_batch_invariant(const void* x, int64_t x_row_stride, const void* weight, void* out,
                               int64_t out_row_stride, int64_t n_rows, int64_t n_cols, int dtype,
                               int weight_dtype, float eps, void* stream);

/* Embedding lookup + invariant RMSNorm: x_out[r, :] = table[row_index[r], :] and out[r, :] =
 * dk_rmsnorm_batch_invariant(x_out[r, :]), the same bits as the lookup followed by that call, in one
 * launch.  row_index: device int64[n_rows]; an index outside [0, table_rows) sets the device status
 * (DK_ERR_DEVICE_CHECK) and leaves its row unwritten.  Any row alignment and n_cols (16-byte aligned rows
 * with n_cols a multiple of 16 bytes take the vector path).  No counterpart in the reference: it fuses the decoder's
 * `self.embed[token_ids]` (kernels/tiny_model.py:110) into the first block's input norm. */
int dk_rmsnorm_gather_batch_invariant(const void* table, int64_t table_row_stride, int64_t table_rows,
                                      const int64_t* row_index, const void* weight, void* x_out, int64_t x_row_stride,
                                      void* out, int64_t out_row_stride, int64_t n_rows, int64_t n_cols, int dtype,
                                      int wdtype, float eps, void* stream);

/* Scratch bytes dk_rmsnorm_batch_variant needs for n_rows rows. */
size_t dk_rmsnorm_variant_workspace_size(int64_t n_rows);
/* replaces kernels/rmsnorm.py:180-218 rmsnorm_batch_variant: when n_rows < split_threshold each row's
 * sum of squares is split into n_splits chunks combined with f32 atomics (order decided by the
 * scheduler: deliberately NOT batch invariant); otherwise identical to the invariant kernel. */
int dk_rmsnorm_batch_variant(const void* x, int64_t x_row_stride, const void* weight, void* out,
                             int64_t out_row_stride, int64_t n_rows, int64_t n_cols, int dtype,
                             int weight_dtype, float eps, int split_threshold, int n_splits,
                             void* workspace, size_t workspace_bytes, void* stream);

/* ---- Matmul: C[M,N] = A[M,K] @ B[K,N] (row-major, unit inner stride), f32 accumulate ----
 * dtype: DK_BF16 or DK_F16 (A, B and C share it).  Row strides (lda, ldb, ldc)
 * in elements; lda and ldb must be multiples of 8 and A, B 16-byte aligned
 * (TMA).  The invariant kernel reduces K as DK_MATMUL_K_SLICES fixed slices of
 * ceil16(K/8) elements, each accumulated by tcgen05 in ascending 16-wide K
 * steps into its own f32 TMEM accumulator (partial p_s), then summed along the
 * fixed tree ((p0+p1)+(p2+p3))+((p4+p5)+(p6+p7)) and rounded to the dtype. */

/* Scratch bytes the invariant / variant matmul may need for this shape: f32 subtree sums when
 * the schedule splits K over CTAs, and for large token counts (the CTA-pair kernel) a 128 KB
 * stash per resident CTA for the left half of the slice tree.  0 means no workspace is needed. */
size_t dk_matmul_workspace_size(int64_t M, int64_t N, int64_t K);
/* replaces kernels/matmul.py:161-186 matmul_batch_invariant (+ _matmul_kernel 64-100) */
int dk_matmul_batch_invariant(const void* a, int64_t lda, const void* b, int64_t ldb, void* c, int64_t ldc,
                              int64_t M, int64_t N, int64_t K, int dtype, void* workspace,
                              size_t workspace_bytes, void* stream);
/* Same numerics for one aligned group of slices [slice_begin, slice_end) (1, 2, 4 or 8 slices,
 * slice_begin a multiple of the group size): writes that group's subtree sum to partial[m * N + n]
 * (f32).  Row-parallel tensor parallelism: rank r of a TP-way split computes group r. */
int dk_matmul_slice_partials(const void* a, int64_t lda, const void* b, int64_t ldb, float* partial,
                             int64_t M, int64_t N, int64_t K, int slice_begin, int slice_end, int dtype,
                             void* stream);
/* Row-parallel tensor parallelism on K shards.  dk_matmul_shard_range gives the K range [k_begin,
 * k_end) of the full K that an aligned slice group [slice_begin, slice_end) covers; a rank holding only
 * that range -- a: [M, k_end - k_begin] (its columns of A), b: [k_end - k_begin, N] (its rows of B) --
 * calls dk_matmul_shard_partials with the FULL K to get the group's f32 subtree sum, bit-identical to
 * dk_matmul_slice_partials on the unsharded operands.  No counterpart in the reference (its matmul has
 * no tensor parallelism, kernels/matmul.py:161-186). */
void dk_matmul_shard_range(int64_t K, int slice_begin, int slice_end, int64_t* k_begin, int64_t* k_end);
int dk_matmul_shard_partials(const void* a, int64_t lda, const void* b, int64_t ldb, float* partial, int64_t M,
                             int64_t N, int64_t K, int slice_begin, int slice_end, int dtype, void* stream);
/* out[m,n] = the upper tree levels over n_parts (1, 2, 4 or 8) subtree sums in group order,
 * partials[j * M * N + m * N + n], rounded to dtype: reproduces dk_matmul_batch_invariant bit for bit. */
int dk_matmul_fold_slices(const float* partials, int n_parts, void* c, int64_t ldc, int64_t M, int64_t N,
                          int dtype, void* stream);
/* Scratch bytes dk_matmul_batch_variant needs on its split-K path. */
size_t dk_matmul_variant_workspace_size(int64_t M, int64_t N);
/* replaces kernels/matmul.py:189-228 matmul_batch_variant: when M < split_m_threshold, K is split
 * into split_k chunks whose f32 partials are combined with atomics (deliberately NOT batch
 * invariant); otherwise the invariant kernel runs. */
int dk_matmul_batch_variant(const void* a, int64_t lda, const void* b, int64_t ldb, void* c, int64_t ldc,
                            int64_t M, int64_t N, int64_t K, int dtype, int split_m_threshold, int split_k,
                            void* workspace, size_t workspace_bytes, void* stream);

/* ---- Matmul with a fused epilogue ----
 * What happens to each output element's f32 tree sum v(m, n) before it is stored.  Every step rounds
 * exactly where the unfused torch ops of a decoder block round (matmul output, residual add, SiLU,
 * product), so a fused call returns the bits of the unfused sequence. */
#define DK_EPI_STORE 0     /* C[m,n] = round(v) */
#define DK_EPI_RESIDUAL 1  /* C[m,n] = round(R[m,n] + round(v)); R may be C itself */
#define DK_EPI_SILU 2      /* C[m,n] = round(silu(round(v))), silu(x) = x / (1 + exp(-x)) */
#define DK_EPI_SILU_MUL 3  /* B's columns hold gate/up pairs (2j, 2j+1); C is [M, N/2]:
                              C[m,j] = round(round(silu(round(v(m,2j)))) * round(v(m,2j+1))) */
#define DK_EPI_QKV_CACHE 4 /* columns [0, q_cols) -> C[m, n]; the next kv_cols -> K cache, the next kv_cols ->
                              V cache, at (row_seq[m], n' / head_dim, row_pos[m], n' % head_dim) */
#define DK_EPI_ARGMAX 5    /* per row, the first column holding the largest round(v) (NaN above all, -0 == +0),
                              torch.argmax's answer, folded into argmax_keys[m] with 64-bit atomicMax of
                              (ordered value << 32 | ~n): order-free, so deterministic.  C is optional
                              (NULL: logits are not stored).  argmax_keys must be 0 before the call;
                              dk_argmax_finish reads and re-zeroes them. */
#define DK_EPI_RESIDUAL_RMSNORM 6 /* C = round(R + round(v)) as DK_EPI_RESIDUAL, then norm_out[m, :] =
                                 * dk_rmsnorm_batch_invariant(C[m, :], norm_w, eps): the same bits as the two
                                 * calls, with the norm computed while C is folded (one launch fewer) */
typedef struct dk_matmul_epilogue {
  int mode;
  const void* resid;       /* DK_EPI_RESIDUAL: R, same dtype as C */
  int64_t ld_resid;
  int32_t q_cols, kv_cols, head_dim;  /* DK_EPI_QKV_CACHE */
  void* k_cache;
  void* v_cache;
  int64_t cache_stride_seq, cache_stride_head, cache_stride_tok;  /* elements; unit stride along d */
  const int32_t* row_seq;  /* device int32[M]; NULL: row m writes cache sequence m */
  const int32_t* row_pos;  /* device int32[M]: token position written by row m */
  unsigned long long* argmax_keys;  /* DK_EPI_ARGMAX: device uint64[M] */
  const void* norm_w;      /* DK_EPI_RESIDUAL_RMSNORM: weight [N] of norm_w_dtype */
  int norm_w_dtype;
  void* norm_out;          /* [M, N] rows norm_ld apart, dtype of C */
  int64_t norm_ld;
  float norm_eps;
  /* DK_EPI_QKV_CACHE into a paged cache (block_table non-NULL): k_cache / v_cache are block pools
   * [n_blocks, heads, page_size, head_dim] (cache_stride_seq = the block stride), and position pos of
   * sequence s goes to block block_table[s * block_table_stride + pos / page_size], token pos %
   * page_size.  A position past blocks_per_seq blocks or an entry outside [0, n_blocks) is recorded as
   * DK_ERR_DEVICE_CHECK and not stored. */
  const int32_t* block_table;
  int64_t block_table_stride;
  int32_t page_size;
  int32_t blocks_per_seq;
  int64_t n_blocks;
} dk_matmul_epilogue;

/* dk_matmul_batch_invariant followed by the epilogue `epi` (same K numerics; NULL epi = DK_EPI_STORE).
 * No counterpart in the reference: it fuses the reference decoder's element-wise torch ops
 * (tiny_model.py:110-139) into the matmul that produces their input. */
int dk_matmul_batch_invariant_ex(const void* a, int64_t lda, const void* b, int64_t ldb, void* c, int64_t ldc,
                                 int64_t M, int64_t N, int64_t K, int dtype, const dk_matmul_epilogue* epi,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* End of a greedy decode step after a DK_EPI_ARGMAX matmul, one thread per row: tokens[r] = the row's
 * argmax column (also into tokens_copy[r] when non-NULL), keys[r] = 0, and lens_a[r] += 1,
 * lens_b[r] += 1 for the non-NULL ones.  No counterpart in the reference: it replaces the
 * `logits.argmax(-1)` and cache-length bookkeeping of tiny_model.py:150-157. */
int dk_argmax_finish(unsigned long long* keys, int64_t n_rows, int64_t* tokens, int64_t* tokens_copy,
                     int32_t* lens_a, int32_t* lens_b, void* stream);

/* ---- Tensor-parallel decoder layers (no counterpart in the reference: its TinyModel runs on one
 * device, kernels/tiny_model.py:99-140) ---- */
/* Row-parallel layer output: the fold of dk_matmul_fold_slices (n_parts = 1, 2, 4 or 8 subtree sums in
 * group order, partials[j * M * N + m * N + n]) followed by the epilogue `epi` exactly as
 * dk_matmul_batch_invariant_ex applies it (DK_EPI_STORE, _RESIDUAL, _RESIDUAL_RMSNORM, _SILU, _SILU_MUL
 * or _ARGMAX; NULL = DK_EPI_STORE), so a layer split over ranks returns the one-GPU fused bits. */
int dk_matmul_fold_slices_ex(const float* partials, int n_parts, void* c, int64_t ldc, int64_t M, int64_t N,
                             int dtype, const dk_matmul_epilogue* epi, void* stream);
/* Greedy step end for a column-parallel LM head: keys[p * part_stride + r] (p < n_parts <= 8) are part
 * p's DK_EPI_ARGMAX keys over its own columns, which start at column col_offsets[p] (host array) of the
 * full vocabulary.  tokens[r] = the global argmax (largest value, then smallest column: the one-GPU
 * answer); then as dk_argmax_finish, with reset_keys[r] = 0 for the caller's local key buffer (optional). */
int dk_argmax_finish_parts(const unsigned long long* keys, int n_parts, int64_t part_stride,
                           const int64_t* col_offsets, int64_t n_rows, int64_t* tokens, int64_t* tokens_copy,
                           int32_t* lens_a, int32_t* lens_b, unsigned long long* reset_keys, void* stream);

/* ---- Decode attention (one query per row, split-KV with a fixed split size) ----
 * q:   [n_rows, n_q_heads, head_dim], strides (q_stride_row, q_stride_head), unit d stride.
 * k,v: KV cache viewed as [kv_n_seq, n_kv_heads, kv_capacity, head_dim] with element strides
 *      (kv_stride_seq, kv_stride_head, kv_stride_tok), unit d stride; k and v share strides.
 * out: [n_rows, n_q_heads, head_dim], strides (out_stride_row, out_stride_head).
 * Row r attends to tokens [0, kv_len_r) of KV sequence seq_r, q head h uses kv head
 * h / (n_q_heads / n_kv_heads).  kv_lens (device int32[n_rows]) may be NULL, then every row
 * uses uniform_kv_len.  row_tiles (device int32[3 * n_tiles]: first row, row count, seq) groups
 * consecutive rows that read the same KV sequence (at most 16 / group rows per tile; a tile of 0 rows is
 * skipped, and rows that no tile covers are left as they were in out); when NULL,
 * row r is its own tile reading sequence r.  max_kv_len bounds every kv_len_r (sizes the grid).
 * head_dim in {32, 64, 128}; dtype DK_BF16 or DK_F16; scale multiplies q.k. */
/* Scratch bytes for a call with n_tiles tiles (n_rows when row_tiles is NULL) of up to rows_per_tile rows
 * (1 without row_tiles); 0 when no row needs more than one split. */
size_t dk_attention_workspace_size(int32_t n_tiles, int32_t rows_per_tile, int32_t n_q_heads, int32_t n_kv_heads,
                                   int32_t head_dim, int32_t max_kv_len);
/* replaces kernels/attention.py:289-298 attention_batch_invariant (+ _attn_direct_kernel 86-143,
 * _run_direct 266-286), extended with GQA, per-row KV lengths and row tiles */
int dk_attention_batch_invariant(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k,
                                 const void* v, int64_t kv_stride_seq, int64_t kv_stride_head,
                                 int64_t kv_stride_tok, int64_t kv_n_seq, int64_t kv_capacity, void* out,
                                 int64_t out_stride_row, int64_t out_stride_head, const int32_t* kv_lens,
                                 int32_t uniform_kv_len, const int32_t* row_tiles, int32_t n_tiles,
                                 int32_t n_rows, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                 int32_t max_kv_len, float scale, int dtype, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* Decode attention over a paged KV cache: the arithmetic, arguments and bits of
 * dk_attention_batch_invariant, with the K/V cache given as block pools k_pool / v_pool
 * [n_blocks, n_kv_heads, page_size, head_dim] (element strides pool_stride_block, pool_stride_head,
 * pool_stride_tok; unit d stride) and a block table: token t of KV sequence s is token t % page_size
 * of block block_table[s * block_table_stride + t / page_size] (device int32 [kv_n_seq][...], at least
 * blocks_per_seq entries per row).  page_size must be a multiple of 64; kv lengths may reach
 * blocks_per_seq * page_size.  A table entry outside [0, n_blocks) is recorded as DK_ERR_DEVICE_CHECK
 * (detail 0x212).  Workspace as dk_attention_workspace_size.  No counterpart in the reference: its
 * cache is one contiguous tensor grown by torch.cat (kernels/tiny_model.py:119-125) and it lists
 * paging as a simplification (kernels/attention.py:35-40). */
int dk_attention_paged_batch_invariant(const void* q, int64_t q_stride_row, int64_t q_stride_head,
                                       const void* k_pool, const void* v_pool, int64_t pool_stride_block,
                                       int64_t pool_stride_head, int64_t pool_stride_tok, int64_t n_blocks,
                                       int32_t page_size, const int32_t* block_table, int64_t block_table_stride,
                                       int64_t kv_n_seq, int32_t blocks_per_seq, void* out, int64_t out_stride_row,
                                       int64_t out_stride_head, const int32_t* kv_lens, int32_t uniform_kv_len,
                                       const int32_t* row_tiles, int32_t n_tiles, int32_t n_rows,
                                       int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len,
                                       float scale, int dtype, void* workspace, size_t workspace_bytes,
                                       void* stream);

/* Scratch bytes dk_attention_batch_variant needs. */
size_t dk_attention_variant_workspace_size(int32_t batch, int32_t n_heads, int32_t head_dim);
/* replaces kernels/attention.py:145-249 (_attn_split_max_kernel, _attn_split_sumacc_kernel) as dispatched by
 * attention_batch_variant (attention.py:301-348): q [batch, n_heads, head_dim], k/v [batch, n_heads, seq_len,
 * head_dim] (unit d stride), KV cut into split_s chunks combined with f32 atomics -- deliberately NOT
 * batch invariant.  dtype DK_F32 / DK_F16 / DK_BF16. */
int dk_attention_batch_variant(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k, const void* v,
                               int64_t kv_stride_b, int64_t kv_stride_h, int64_t kv_stride_s, void* out,
                               int64_t out_stride_b, int64_t out_stride_h, int32_t batch, int32_t n_heads,
                               int32_t seq_len, int32_t head_dim, float scale, int32_t split_s, int dtype,
                               void* workspace, size_t workspace_bytes, void* stream);

/* ---- decode attention for callers that cannot allocate device memory ----
 * No counterpart in the reference.  Some callers cannot hand this library a workspace: code that
 * runs inside another runtime's allocator or memory-pool callbacks, plugins whose host owns every
 * device allocation, or paths where a cudaMalloc would synchronise the device at the wrong time.
 * This entry point takes the same arguments as dk_attention_batch_invariant minus the workspace,
 * and produces the same bits.  Its scratch is a 32 MiB array in device memory that belongs to the
 * library (dk_attention_noalloc_scratch_limit() returns the size): every GPU that loads the library
 * keeps it until the process exits.  Calls whose multi-split scratch would exceed it are rejected
 * with DK_ERR_WORKSPACE.  It never allocates: the first call on a device looks up the array's
 * device address with that device current (cudaGetSymbolAddress) and caches it, so make that first
 * call before any stream capture on the device.  Each call clears the arrival counters it uses on
 * `stream`.  All calls share the one array, so calls on one device that may overlap on the GPU (for
 * example on different streams without ordering) race and give wrong results; order them. */
size_t dk_attention_noalloc_scratch_limit(void);
int dk_attention_batch_invariant_noalloc(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k,
                                         const void* v, int64_t kv_stride_seq, int64_t kv_stride_head,
                                         int64_t kv_stride_tok, int64_t kv_n_seq, int64_t kv_capacity, void* out,
                                         int64_t out_stride_row, int64_t out_stride_head, const int32_t* kv_lens,
                                         int32_t uniform_kv_len, const int32_t* row_tiles, int32_t n_tiles,
                                         int32_t n_rows, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                         int32_t max_kv_len, float scale, int dtype, void* stream);

/* ---- Gated delta rule (Gated DeltaNet linear attention), forward ----
 * replaces the FLA `chunk_gated_delta_rule` / `fused_recurrent_gated_delta_rule` calls of the
 * reference's gdn/repro.py:76,161-162,293-294 (fla 0.5.1 API, [B, T, heads, dim] layout).
 * q, k: [tokens, n_heads, head_dim_k]; v: [tokens, n_v_heads, head_dim_v]; g (log decay), beta:
 * [tokens, n_v_heads]; o: [tokens, n_v_heads, head_dim_v] in q's dtype, all contiguous, q/k/v
 * starting on a 16-byte boundary.  Value head j
 * uses query/key head j / (n_v_heads / n_heads).  Sequences: cu_seqlens (device int64[n_seqs + 1])
 * with seq_len = the packed length T of q/k/v/g/beta/o (a sequence whose pair falls outside [0, T] or
 * decreases is skipped and recorded as DK_ERR_DEVICE_CHECK, detail 0x500), or, when cu_seqlens is
 * NULL, n_seqs rows of seq_len tokens each.  initial_state / final_state: [n_seqs,
 * n_v_heads, head_dim_k, head_dim_v] (final in f32), either may be NULL.  chunk_size 64 computes
 * 64-token chunks from each sequence's start (chunked form); 1 steps token by token in the order of
 * the recurrence (decode path; FLA's fused_recurrent_gated_delta_rule).  A sequence's
 * result never depends on the other sequences of the call.  Head dims: 32/32, 64/64, 128/128. */
int dk_gdn_forward(const void* q, const void* k, const void* v, const void* g, const void* beta, void* o,
                   const int64_t* cu_seqlens, int64_t n_seqs, int64_t seq_len, int n_heads, int n_v_heads,
                   int head_dim_k, int head_dim_v, int dtype, int gb_dtype, float scale, const void* initial_state,
                   int state_dtype, float* final_state, int chunk_size, void* stream);

/* ---- Serving steps: page plan, head norm + rotation into the cache, shared-prefix attention ----
 * No counterparts in the reference (its cache is one tensor grown by torch.cat, its decoder has no
 * rotation, and every row reads its whole KV sequence: kernels/tiny_model.py:99-140). */

/* Scratch bytes of dk_paged_plan (uninitialised memory will do). */
size_t dk_paged_plan_workspace_size(int64_t n_seqs);
/* Plans one step of n_seqs sequences on the device.  Sequence b holds kv_lens[b] tokens and gets
 * new_lens[b] more (device int32[n_seqs], >= 0).
 *  - free_blocks (device int32[n_free], may be NULL: the table is only read): the table entries
 *    [ceil(kv / page_size), ceil((kv + new) / page_size)) of row b of block_table [n_seqs][blocks_per_seq]
 *    become the next free blocks from position *cursor on, in sequence order; *cursor_out = *cursor + the
 *    number taken (cursor_out may be cursor).  The other entries stay as they are.
 *  - cu_rows: int32[n_seqs + 1], the exclusive sums of new_lens.
 *  - row_seq, row_pos, slots, q_lens (all or none; n_rows entries each): row cu_rows[b] + i is token
 *    pos = kv_lens[b] + i of sequence b, at slot table[b][pos / page_size] * page_size + pos % page_size,
 *    and attends to q_lens = pos + 1 tokens.  Entries past cu_rows[n_seqs] stay as they are.
 *  - row_tiles (may be NULL; int32[n_tiles][3]): (first row, rows, sequence) of up to rows_per_tile rows
 *    of one sequence, the row_tiles of the attention entry points.  Tiles past the last stay as they are.
 * A negative length or a sequence beyond blocks_per_seq pages (detail 0x600), too few free blocks (0x601)
 * or more rows or tiles than the outputs hold (0x602) is recorded as DK_ERR_DEVICE_CHECK; then only cu_rows
 * and the workspace are written and *cursor_out = *cursor.  The operators below take an earlier plan's slots and
 * tiles for this step's: where the sizes are bounds, or a refused plan may go unseen, use dk_paged_plan_padded. */
int dk_paged_plan(int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq, const int32_t* kv_lens,
                  const int32_t* new_lens, int32_t n_seqs, int32_t page_size, const int32_t* free_blocks,
                  int64_t n_free, const int32_t* cursor, int32_t* cursor_out, int32_t* cu_rows, int32_t* row_seq,
                  int32_t* row_pos, int64_t* slots, int32_t* q_lens, int64_t n_rows, int32_t* row_tiles,
                  int32_t rows_per_tile, int64_t n_tiles, void* workspace, size_t workspace_bytes, void* stream);

/* The same plan for outputs whose sizes are bounds (a captured step that serves smaller ones): the entries past its
 * totals, and all of them when the plan is refused, become neutral for the operators below: row_seq, row_pos and
 * q_lens 0, slots -1 (nothing is stored there), tiles of 0 rows (attention skips them).  dk_matmul_epilogue's store into
 * the cache goes by row_seq and row_pos and knows no such rows: it needs exact sizes.  n_seqs = 0 writes nothing. */
int dk_paged_plan_padded(int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq,
                         const int32_t* kv_lens, const int32_t* new_lens, int32_t n_seqs, int32_t page_size,
                         const int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out,
                         int32_t* cu_rows, int32_t* row_seq, int32_t* row_pos, int64_t* slots, int32_t* q_lens,
                         int64_t n_rows, int32_t* row_tiles, int32_t rows_per_tile, int64_t n_tiles, void* workspace,
                         size_t workspace_bytes, void* stream);

/* RMSNorm of every query and key head followed by the rotation of its first rotary_dim elements, f32
 * math, one rounding at the store.  q [n_rows, n_q_heads, head_dim], k and v [n_rows, n_kv_heads,
 * head_dim]: element strides by row and head, unit stride along head_dim.  Pairs are (i, i +
 * rotary_dim / 2), or (2i, 2i + 1) when interleaved; row r's angles are row positions[r] (device int32, or
 * int64 when positions_64) of rope_table: f32 [max_pos, rotary_dim] = cos[rotary_dim / 2], sin[...].
 * q_out may be q and k_out may be k (same strides).  With k_cache / v_cache [cache_slabs, n_kv_heads,
 * cache_capacity, head_dim] (slab = sequence or block), slots (device int64[n_rows]) and v, the rotated
 * key and the value of row r go to slab slots[r] / cache_capacity, token slots[r] % cache_capacity; a
 * negative slot stores nothing, one beyond the cache is recorded (DK_ERR_DEVICE_CHECK, detail 0x611) and
 * stores nothing; rows must not share a slot.  k_out may be NULL with a cache.  A position outside the table is recorded (0x610) and
 * its row not written.  head_dim <= 512; any dtype of the three for q/k/v/caches, and for the weights
 * [head_dim].  Calls whose every tensor has rows and heads on 16 bytes, and whose rotated half is a half or a quarter
 * of the head in whole 16-byte vectors (neighbouring pairs: any rotary_dim of whole vectors, an even number of
 * vectors a head), take the vector path; it and the other are each batch invariant, but sum squares in another order. */
int dk_qk_norm_rope(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k, int64_t k_stride_row,
                    int64_t k_stride_head, const void* v, int64_t v_stride_row, int64_t v_stride_head, void* q_out,
                    int64_t q_out_stride_row, int64_t q_out_stride_head, void* k_out, int64_t k_out_stride_row,
                    int64_t k_out_stride_head, void* k_cache, void* v_cache, int64_t cache_stride_slab,
                    int64_t cache_stride_head, int64_t cache_stride_tok, int64_t cache_slabs, int64_t cache_capacity,
                    const int64_t* slots, const void* positions, int positions_64, const void* q_weight,
                    const void* k_weight, int weight_dtype, const float* rope_table, int64_t max_pos, int64_t n_rows,
                    int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t rotary_dim, int interleaved,
                    float eps, int dtype, void* stream);

/* Workspace bytes of dk_attention_shared_prefix (uninitialised memory will do; no counters).  n_tiles =
 * n_rows without row_tiles. */
size_t dk_attention_shared_prefix_workspace_size(int32_t n_rows, int32_t n_tiles, int32_t n_q_heads, int32_t n_kv_heads,
                                      int32_t head_dim, int32_t prefix_len, int32_t max_kv_len);
/* Decode attention of rows that share a prefix: row r attends to the prefix_len prefix tokens and then
 * to tokens [0, kv_len_r) of its own KV sequence, the prefix part computed once for all rows.
 * The prefix: k_prefix / v_prefix [n_kv_heads, prefix_len, head_dim] (prefix_stride_head / _tok), or,
 * with prefix_blocks (device int32[ceil(prefix_len / prefix_page)]), block pools [prefix_pool_blocks,
 * n_kv_heads, prefix_page, head_dim] whose block prefix_blocks[t / prefix_page] holds token t (a block id
 * outside the pool: DK_ERR_DEVICE_CHECK, detail 0x62a).  prefix_page is a multiple of 64.
 * The rows' own tokens: q, k, v, kv_lens, row_tiles, max_kv_len, scale as in
 * dk_attention_batch_invariant, or with block_table as in dk_attention_paged_batch_invariant
 * (kv_stride_seq is then the block stride); max_kv_len = 0: no row has any, and k, v and kv_lens are not
 * read.  A length beyond max_kv_len or the cache (detail 0x210), a malformed tile (0x211) or a block id outside
 * the pool (0x212) is recorded as DK_ERR_DEVICE_CHECK; the rows of a tile that is malformed or holds such a
 * length are left as they were in out, and so is a row that no tile covers.  Nothing beyond a row's own length
 * reaches it, whatever the cache holds there.  q must be 16-byte aligned with strides that are multiples
 * of 8 elements.
 * Batch invariant: a row's bits follow from its q, the prefix and its own tokens. */
int dk_attention_shared_prefix(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k_prefix,
                               const void* v_prefix, int64_t prefix_stride_block, int64_t prefix_stride_head,
                               int64_t prefix_stride_tok, int32_t prefix_len, const int32_t* prefix_blocks,
                               int64_t prefix_pool_blocks, int32_t prefix_page, const void* k, const void* v,
                               int64_t kv_stride_seq, int64_t kv_stride_head, int64_t kv_stride_tok, int64_t kv_n_seq,
                               int64_t kv_capacity, const int32_t* block_table, int64_t block_table_stride,
                               int32_t blocks_per_seq, int64_t n_blocks, int32_t page_size, void* out,
                               int64_t out_stride_row, int64_t out_stride_head, const int32_t* kv_lens,
                               const int32_t* row_tiles, int32_t n_tiles, int32_t n_rows, int32_t n_q_heads,
                               int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len, float scale, int dtype,
                               void* workspace, size_t workspace_bytes, void* stream);

/* ---- Drafted tokens: their attention, log probabilities, the accepted path of a tree, pages forked, compacted and freed ----
 * No counterparts in the reference (its decoder takes one token a step, greedily, into a cache that only grows:
 * kernels/tiny_model.py:119-157). */

/* Workspace bytes of dk_attention_tree (uninitialised memory will do; 0: none is needed).  max_rows and max_kv_len bound
 * the rows and the tokens (drafts included) of a sequence. */
size_t dk_attention_tree_workspace_size(int32_t n_seqs, int32_t n_rows, int32_t max_rows, int32_t n_q_heads,
                                        int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len);
/* Attention of drafted tokens over a cache that holds them: sequence b has kv_lens[b] tokens and, behind them, its
 * drafts, whose queries are the rows [cu_rows[b], cu_rows[b + 1]) of q [n_rows, n_q_heads, head_dim] (cu_rows: device
 * int32[n_seqs + 1]).  Row cu_rows[b] + i attends to tokens [0, kv_lens[b]) and to token kv_lens[b] + j where bit j of its
 * mask is set (mask: device int64[n_rows][mask_words], 64 drafts a word from the lowest bit, row stride mask_stride;
 * bits from the sequence's row count on are ignored, drafts past the words are not seen).  A row that sees nothing is 0.
 * The caches k, v are [kv_n_seq, n_kv_heads, kv_capacity, head_dim], or with block_table block pools as in
 * dk_attention_paged_batch_invariant; strides, scale, head_dim and dtypes as there, at most 128 query heads a KV head.
 * Rows behind cu_rows[n_seqs] are left as they were in out.  Offsets that do not ascend inside the rows, more than
 * max_rows rows a sequence, a negative length or more than max_kv_len tokens (detail 0x67d: the sequence's rows are left
 * as they were) and a block id outside the pool (0x67a: read as block 0) are recorded as DK_ERR_DEVICE_CHECK.  Nothing
 * that a row does not see reaches it, whatever the cache holds there.
 * Batch invariant: a row's bits follow from its q and the tokens that it sees at their positions. */
int dk_attention_tree(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k, const void* v,
                      int64_t kv_stride_seq, int64_t kv_stride_head, int64_t kv_stride_tok, int64_t kv_n_seq,
                      int64_t kv_capacity, const int32_t* block_table, int64_t block_table_stride,
                      int32_t blocks_per_seq, int64_t n_blocks, int32_t page_size, void* out, int64_t out_stride_row,
                      int64_t out_stride_head, const int32_t* kv_lens, const int32_t* cu_rows, const int64_t* mask,
                      int64_t mask_stride, int32_t mask_words, int32_t n_seqs, int32_t n_rows, int32_t max_rows,
                      int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len, float scale,
                      int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* Log probabilities of rows of logits [n_rows, n_vocab] (any of the three dtypes, element stride stride_row, unit
 * stride along the vocabulary; rows need no alignment but their elements').
 *  - tokens (device int64[n_rows], may be NULL): logprobs[r] = log softmax(row r)[tokens[r]]; a token of -1 asks for
 *    nothing and gives 0, any other outside the vocabulary is recorded (DK_ERR_DEVICE_CHECK, detail 0x650) and gives NaN.
 *  - entropy (may be NULL): -sum p log p in nats (a logit of -infinity has p = 0 and adds nothing).
 *  - top_k <= 32 alternatives: top_ids [n_rows, top_k] int64 and their log probabilities, the largest logit first,
 *    equal ones by their index (NaN is above all, -0 equals 0).
 * f32 arithmetic.  A row with a NaN, +infinity or nothing but -infinity has NaN log probabilities and entropy.
 * Batch invariant: a row's bits follow from its logits alone. */
int dk_token_logprobs(const void* logits, int64_t stride_row, int64_t n_rows, int32_t n_vocab, int dtype,
                      const int64_t* tokens, float* logprobs, float* entropy, int32_t top_k, int64_t* top_ids,
                      float* top_logprobs, void* stream);

/* The accepted path of each sequence's tree of drafted tokens.  Sequence b's nodes are the rows [cu_rows[b],
 * cu_rows[b + 1]) of parents (index of the parent among the sequence's nodes, smaller than the node's own; -1: none),
 * tokens and picked (the model's token after the node).  From node 0 the path goes to the first child whose token is
 * the pick after the current node, at most max_keep nodes.  keep [n_seqs, max_keep]: its nodes in ascending order, -1
 * behind them; n_keep [n_seqs]; next_tokens [n_seqs]: the pick after its last node.  A sequence without nodes has
 * n_keep 0 and next_tokens -1, and so has one whose offsets do not ascend inside [0, n_rows], which is recorded
 * (DK_ERR_DEVICE_CHECK, detail 0x660). */
int dk_tree_accept(const int32_t* parents, const int64_t* tokens, const int64_t* picked, const int32_t* cu_rows,
                   int32_t n_seqs, int32_t n_rows, int32_t max_keep, int32_t* keep, int32_t* n_keep,
                   int64_t* next_tokens, void* stream);

/* The pools of the next two calls: n_pools device pointers (an array on the host) to tensors [n_blocks, n_heads, page_size,
 * head_dim] of elements of element_size bytes (1, 2, 4 or 8), all with the same element strides by block, head and token
 * (positive, where there is more than one) and unit stride along head_dim; no two of them overlap.  shares (device
 * int32[n_blocks]): how many further sequences hold a block beyond the first.
 * The free list: free_blocks[0, *cursor) are handed out, as for dk_paged_plan; cursor_out may be cursor. */
size_t dk_paged_fork_workspace_size(int32_t table_rows);   /* uninitialised memory will do */
/* Row dst[i] of block_table [table_rows][blocks_per_seq] becomes a copy of row src[i], kv_lens[dst[i]] =
 * kv_lens[src[i]].  With shares, whole pages are shared (shares[block] += 1) and the last, open page gets the next
 * free block; without, every page does.  The tokens of new blocks are copied in all pools.  The blocks that row dst
 * held are not given back, its entries past the copied ones stay.  A source may be named several times; a destination
 * once, and not as a source.  Recorded as DK_ERR_DEVICE_CHECK: rows outside the table or so misnamed (detail 0x640), a
 * length outside its row (0x641), a block id outside [0, n_blocks) (0x642), too few free blocks (0x643); then nothing
 * changes but the workspace, and *cursor_out = *cursor. */
int dk_paged_fork(int32_t* block_table, int64_t block_table_stride, int32_t table_rows, int32_t blocks_per_seq,
                  int32_t* kv_lens, const int32_t* src, const int32_t* dst, int32_t n_forks, int32_t page_size,
                  const int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out,
                  int32_t* shares, int64_t n_blocks, void* const* pools, int32_t n_pools, int64_t pool_stride_block,
                  int64_t pool_stride_head, int64_t pool_stride_tok, int32_t n_heads, int32_t head_dim,
                  int32_t element_size, void* workspace, size_t workspace_bytes, void* stream);

size_t dk_paged_compact_workspace_size(void);              /* uninitialised memory will do */
/* Sequence b holds kv_lens[b] tokens and new_lens[b] behind them, of which n_keep[b] stay: those at kv_lens[b] +
 * keep[b][j], ascending (keep [n_seqs][keep_width], row stride keep_stride; NULL: the first n_keep[b]).  They are moved to
 * kv_lens[b] + j in all pools, lens_out[b] = kv_lens[b] + n_keep[b] (lens_out is none of the inputs), and with
 * free_blocks the pages [ceil(lens_out / page), ceil((kv + new) / page)) are given up: a page with shares loses one, any
 * other goes back, free_blocks[*cursor_out, *cursor) in the order of (sequence, page), a page given up by all its
 * holders in this call at the last of them.  Without shares a page is one sequence's alone; with them n_seqs *
 * blocks_per_seq must be below 2^30.  Table entries stay.  kv_lens = 0 and n_keep = 0 free a whole sequence.
 * Tokens are not moved into a page that another sequence shares, were it to give the page up in the same call: from the
 * first token that moves on, the pages are the sequence's own, as dk_paged_fork leaves the open one.  A sequence that then
 * ends inside a shared page must not take new tokens there: dk_paged_fork gives its copy a page of its own.  Recorded as
 * DK_ERR_DEVICE_CHECK: bad lengths (detail 0x644), a bad row of keep (0x645), a block id outside [0, n_blocks) among those
 * that moved tokens or given-up pages name (0x642), more pages than were handed out (0x643), a page given up by more
 * sequences than hold it (0x646), a token to move into a page that has shares (0x647); then lens_out = kv_lens, *cursor_out =
 * *cursor, and nothing else changes. */
int dk_paged_compact(const int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq,
                     const int32_t* kv_lens, const int32_t* new_lens, const int32_t* n_keep, const int32_t* keep,
                     int64_t keep_stride, int32_t keep_width, int32_t n_seqs, int32_t page_size, int32_t* lens_out,
                     int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out, int32_t* shares,
                     int64_t n_blocks, void* const* pools, int32_t n_pools, int64_t pool_stride_block,
                     int64_t pool_stride_head, int64_t pool_stride_tok, int32_t n_heads, int32_t head_dim,
                     int32_t element_size, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DETKERNELS_B200_H */
