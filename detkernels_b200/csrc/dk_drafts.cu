// C ABI of the operators around drafted tokens (see include/detkernels_b200.h): log probabilities of given tokens, the
// accepted path of a tree, and forking, compacting and freeing the pages of a cache.  (dk_tree.cu: their attention.)
#include <algorithm>

#include "dk_accept.cuh"
#include "dk_common.cuh"
#include "dk_host.cuh"
#include "dk_logprobs.cuh"
#include "dk_pages.cuh"

namespace dk {
namespace host {
cudaError_t drafts_status(int clear, int* code, int* detail) { return unit_status(clear, code, detail); }
}  // namespace host
}  // namespace dk

using namespace dk::host;

namespace {

constexpr int64_t kI32Max = 0x7fffffffLL;

// ============================ log probabilities ============================
template <typename T, bool TOPK, bool ALIGNED>
int logprobs_launch(dk::logprobs::Params p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  auto fn = dk::logprobs::logprobs_kernel<T, TOPK, ALIGNED>;
  // the CTAs that fit at once, each walking rows
  using C = dk::logprobs::Cfg<T, TOPK>;
  static bool done[kMaxDevices] = {false};
  constexpr int kShared = 226 * 1024;   // an SM's, without what the system takes of it for a few CTAs
  int rc = ensure_smem(fn, C::STAGES * C::STAGE + C::STATES, done);
  if (rc) return rc;
  const int sms = sm_count(current_device());
  const int64_t ctas = std::min<int64_t>(p.split ? p.n_rows * p.parts : p.n_rows, static_cast<int64_t>(C::CTAS) * sms);
  // A ring as deep as the CTAs of an SM leave room for: at four, three stages (of 2 and 3 no difference: 93 and 94 us for
  // 4096 rows of 50,001 bf16 logits; the other CTAs' passes are in flight too); one alone needs more to cover a copy's latency.
  const int share = kShared / static_cast<int>(ceil_div(ctas, sms)) - C::STATIC - 1024 - (p.split ? C::STATES : 0);
  p.stages = std::max(2, std::min<int>(C::STAGES, share / C::STAGE));
  const int64_t resident = static_cast<int64_t>(C::CTAS) * sms;
  cfg.gridDim = dim3(static_cast<unsigned>(p.split ? p.n_rows * p.parts : std::min(p.n_rows, resident)));
  cfg.blockDim = dim3(dk::logprobs::kThreads);
  cfg.dynamicSmemBytes = p.stages * C::STAGE + (p.split ? C::STATES : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.parts);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "token_logprobs: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

template <typename T>
int logprobs_for(const dk::logprobs::Params& p, cudaStream_t st) {
  const bool aligned = aligned16(p.x) && (p.n_rows == 1 || p.stride * sizeof(T) % 16 == 0);
  if (p.k > 0) return aligned ? logprobs_launch<T, true, true>(p, st) : logprobs_launch<T, true, false>(p, st);
  return aligned ? logprobs_launch<T, false, true>(p, st) : logprobs_launch<T, false, false>(p, st);
}

// ============================ pages ============================
struct Pools {
  void* const* ptr;
  int32_t n;
  int64_t s_block, s_head, s_tok, n_blocks;
  int32_t heads, dim, size;
};

int check_pools(const Pools& c, int64_t page, const char* what) {
  if (c.n < 0 || (c.n > 0 && !c.ptr)) return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (c.n_blocks <= 0 || c.n_blocks > kI32Max) return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad number of blocks", what);
  if (c.n == 0) return DK_OK;
  if (c.size != 1 && c.size != 2 && c.size != 4 && c.size != 8)
    return fail(DK_ERR_UNSUPPORTED, "%s: elements of %d bytes", what, c.size);
  if (c.heads <= 0 || c.dim <= 0 || static_cast<int64_t>(c.n) * c.heads * c.dim > kI32Max)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad pool shape", what);
  if ((c.n_blocks > 1 && c.s_block <= 0) || (c.heads > 1 && c.s_head <= 0) || (page > 1 && c.s_tok <= 0))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: the pools' elements must each have a place of their own", what);
  for (int i = 0; i < c.n; ++i)
    if (!c.ptr[i] || reinterpret_cast<uintptr_t>(c.ptr[i]) % c.size)
      return fail(DK_ERR_INVALID_ARGUMENT, "%s: a pool's address is null or not that of an element", what);
  return DK_OK;
}

template <typename V>
cudaError_t move_launch(const dk::pages::MoveParams& p, int64_t grid, bool after_another, cudaStream_t st) {
  const dim3 g(static_cast<unsigned>(grid)), t(dk::pages::kMoveThreads);
  if (p.src) return launch_pdl(dk::pages::move_kernel<V, 8, true>, g, t, 0, st, p);
  if (!after_another) return launch_pdl(dk::pages::move_kernel<V, 8, false>, g, t, 0, st, p);
  // the kernel before this one is another part of the pools' move, not release_kernel: it is waited for in whole
  dk::pages::move_kernel<V, 8, false><<<g, t, 0, st>>>(p);
  return cudaGetLastError();
}

// Moves the tokens of `n` sequences, at most `most` each, in every pool; or says beforehand whether it will.
int move(dk::pages::MoveParams& p, const Pools& c, int64_t n, int64_t most, bool launch, const char* what, cudaStream_t st) {
  if (c.n == 0 || n == 0 || most <= 0) return DK_OK;
  bool wide = c.dim * static_cast<int64_t>(c.size) % 16 == 0 && c.s_block * c.size % 16 == 0 &&
              c.s_head * c.size % 16 == 0 && c.s_tok * c.size % 16 == 0;
  for (int i = 0; i < c.n; ++i) wide = wide && aligned16(c.ptr[i]);
  const int vec = wide ? 16 / c.size : 1;   // elements a vector
  p.heads = c.heads;
  p.vecs = c.dim / vec;
  p.s_block = c.s_block / vec;
  p.s_head = c.s_head / vec;
  p.s_tok = c.s_tok / vec;
  p.n_blocks = c.n_blocks;
  // Token lanes as the tokens ask for: a few of many columns at once, or many of a head's columns.
  constexpr int U = 8;
  int lanes_log = 0;
  while (lanes_log < dk::pages::kMaxLanesLog && (static_cast<int64_t>(U) << lanes_log) < most) ++lanes_log;
  p.cols_log = 8 - lanes_log;
  // A few long caches, the longest first: 279 us for 8 of up to 16,000 tokens in any order, in their own 275 to 295.
  p.sorted = !p.src && n <= 32 && most > (int64_t{4} * U << lanes_log) ? static_cast<int32_t>(n) : 0;
  for (int first = 0; first < c.n; first += dk::pages::kMaxPools) {
    const int pools = std::min(c.n - first, dk::pages::kMaxPools);
    for (int i = 0; i < pools; ++i) p.pool[i] = c.ptr[first + i];
    p.n_cols = pools * c.heads * p.vecs;
    p.col_groups = static_cast<int32_t>(ceil_div(p.n_cols, int64_t{1} << p.cols_log));
    // a fork's tokens may be copied in any order: enough shares to fill the GPU
    const int64_t units = n * p.col_groups;
    p.splits = p.src ? static_cast<int32_t>(std::max<int64_t>(
                           1, std::min(ceil_div(16LL * sm_count(current_device()), units),
                                       ceil_div(most, static_cast<int64_t>(U) << lanes_log))))
                     : 1;
    const int64_t grid = units * p.splits;
    if (grid > kI32Max) return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many sequences", what);
    if (!launch) continue;
    cudaError_t e = wide          ? move_launch<uint4>(p, grid, first > 0, st)
                    : c.size == 1 ? move_launch<uint8_t>(p, grid, first > 0, st)
                    : c.size == 2 ? move_launch<uint16_t>(p, grid, first > 0, st)
                    : c.size == 4 ? move_launch<uint32_t>(p, grid, first > 0, st)
                                  : move_launch<uint64_t>(p, grid, first > 0, st);
    if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  }
  return DK_OK;
}

int check_table(const void* table, int64_t stride, int64_t rows, int64_t width, int64_t page, const char* what) {
  if (rows < 0 || width < 0 || page <= 0) return fail(DK_ERR_INVALID_ARGUMENT, "%s: negative size or page_size < 1", what);
  if (width > 0 && !table) return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (rows > 1 && stride < width) return fail(DK_ERR_INVALID_ARGUMENT, "%s: block_table_stride < blocks_per_seq", what);
  if (width * page > kI32Max)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: blocks_per_seq * page_size exceeds 2^31 - 1 tokens", what);
  return DK_OK;
}

int check_ws(const void* ws, size_t given, size_t need, const char* what) {
  if (!ws || given < need || (reinterpret_cast<uintptr_t>(ws) & 3u))
    return fail(DK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, given);
  return DK_OK;
}

// A call of nothing leaves the cursor as it is, in its output too.
int keep_cursor(const int32_t* cursor, int32_t* cursor_out, const char* what, cudaStream_t st) {
  if (!cursor || !cursor_out || cursor == cursor_out) return DK_OK;
  cudaError_t e = cudaMemcpyAsync(cursor_out, cursor, sizeof(int32_t), cudaMemcpyDeviceToDevice, st);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

size_t fork_ws_bytes(int64_t rows) { return static_cast<size_t>(dk::pages::kWsMark + 2 * rows) * sizeof(int32_t); }
size_t compact_ws_bytes() { return static_cast<size_t>(dk::pages::kWsMark) * sizeof(int32_t); }

}  // namespace

extern "C" {

int dk_token_logprobs(const void* logits, int64_t stride_row, int64_t n_rows, int32_t n_vocab, int dtype,
                      const int64_t* tokens, float* logprobs, float* entropy, int32_t top_k, int64_t* top_ids,
                      float* top_logprobs, void* stream) {
  const char* what = "token_logprobs";
  if (!valid_dtype(dtype)) return fail(DK_ERR_UNSUPPORTED, "%s: bad dtype", what);
  if (n_rows < 0 || n_vocab <= 0 || top_k < 0 || top_k > n_vocab)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad shape, or more alternatives than logits", what);
  if (top_k > dk::logprobs::kMaxK)
    return fail(DK_ERR_UNSUPPORTED, "%s: more than %d alternatives", what, dk::logprobs::kMaxK);
  if (n_rows == 0) return DK_OK;
  if (!logits || (tokens != nullptr) != (logprobs != nullptr) ||
      (top_k > 0 && (!top_ids || !top_logprobs)))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  const int size = dtype == DK_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: logits lie off their elements' size", what);
  dk::logprobs::Params p{};
  p.x = logits;
  p.stride = stride_row;
  p.n_vocab = n_vocab;
  p.n_rows = n_rows;
  // parts of whole passes, of one while a cluster holds the row
  const int64_t pass = dtype == DK_F32 ? dk::logprobs::Cfg<float, false>::PASS : dk::logprobs::Cfg<__half, false>::PASS;
  p.part = static_cast<int32_t>(ceil_div(ceil_div(n_vocab, pass), dk::logprobs::kMaxParts) * pass);
  p.parts = static_cast<int32_t>(ceil_div(n_vocab, p.part));
  // Rows that leave many SMs idle are split over the CTAs of a cluster.  With 20 alternatives, split and not: 8 rows of 32,000
  // bf16 logits 8.0 and 13.8 us, 74 14.1 and 14.0, 148 16.4 and 14.9; of 185,668 74 rows 30 and 45, 148 51 and 46; of 50,001
  // f32 74 rows 19 and 24, 148 28 and 25.
  p.split = p.parts > 1 && 4 * n_rows <= 3 * sm_count(current_device());
  p.k = top_k;
  p.tokens = tokens;
  p.lp = logprobs;
  p.entropy = entropy;
  p.top_ids = top_ids;
  p.top_lp = top_logprobs;
  // parts that start inside the row end inside 32 bits
  if (n_rows > kI32Max || n_vocab > kI32Max / 2)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many rows or logits", what);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DK_F32) return logprobs_for<float>(p, st);
  if (dtype == DK_F16) return logprobs_for<__half>(p, st);
  return logprobs_for<__nv_bfloat16>(p, st);
}

int dk_tree_accept(const int32_t* parents, const int64_t* tokens, const int64_t* picked, const int32_t* cu_rows,
                   int32_t n_seqs, int32_t n_rows, int32_t max_keep, int32_t* keep, int32_t* n_keep,
                   int64_t* next_tokens, void* stream) {
  const char* what = "tree_accept";
  if (n_seqs < 0 || n_rows < 0 || max_keep <= 0)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: negative size or max_keep < 1", what);
  if (n_seqs == 0) return DK_OK;
  if (!cu_rows || !keep || !n_keep || !next_tokens || (n_rows > 0 && (!parents || !tokens || !picked)))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  dk::accept::Params p{parents, tokens, picked, cu_rows, n_seqs, n_rows, max_keep, keep, n_keep, next_tokens};
  cudaError_t e = launch_pdl(dk::accept::accept_kernel, dim3(static_cast<unsigned>(ceil_div(n_seqs, dk::accept::kThreads / 32))),
                             dim3(dk::accept::kThreads), 0, static_cast<cudaStream_t>(stream), p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

size_t dk_paged_fork_workspace_size(int32_t table_rows) { return table_rows > 0 ? fork_ws_bytes(table_rows) : 0; }

int dk_paged_fork(int32_t* block_table, int64_t block_table_stride, int32_t table_rows, int32_t blocks_per_seq,
                  int32_t* kv_lens, const int32_t* src, const int32_t* dst, int32_t n_forks, int32_t page_size,
                  const int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out,
                  int32_t* shares, int64_t n_blocks, void* const* pools, int32_t n_pools, int64_t pool_stride_block,
                  int64_t pool_stride_head, int64_t pool_stride_tok, int32_t n_heads, int32_t head_dim,
                  int32_t element_size, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "paged_fork";
  int rc = check_table(block_table, block_table_stride, table_rows, blocks_per_seq, page_size, what);
  if (rc) return rc;
  if (n_forks < 0 || n_free < 0 || n_free > kI32Max)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: negative size, or more than 2^31 - 1 free blocks", what);
  if (n_forks > kI32Max - 4096) return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many forks", what);
  const Pools c{pools, n_pools, pool_stride_block, pool_stride_head, pool_stride_tok, n_blocks, n_heads, head_dim,
                element_size};
  rc = check_pools(c, page_size, what);
  if (rc) return rc;
  if (n_forks == 0) return keep_cursor(cursor, cursor_out, what, static_cast<cudaStream_t>(stream));
  if (!kv_lens || !src || !dst || !cursor || !cursor_out || (n_free > 0 && !free_blocks))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  rc = check_ws(workspace, workspace_bytes, fork_ws_bytes(table_rows), what);
  if (rc) return rc;
  dk::pages::ForkParams p{};
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.rows = table_rows;
  p.width = blocks_per_seq;
  p.kv = kv_lens;
  p.src = src;
  p.dst = dst;
  p.n = n_forks;
  p.page = dk::divisor(page_size);
  p.free_list = free_blocks;
  p.n_free = n_free;
  p.cursor_in = cursor;
  p.cursor_out = cursor_out;
  p.shares = shares;
  p.n_blocks = n_blocks;
  p.ws = static_cast<int32_t*>(workspace);
  dk::pages::MoveParams m{};
  m.table = block_table;
  m.table_stride = block_table_stride;
  m.page = p.page;
  m.kv = kv_lens;
  m.src = src;
  m.dst = dst;
  m.all = shares == nullptr;
  m.width = blocks_per_seq;
  m.ws = p.ws;
  const int64_t most = shares ? page_size - 1 : static_cast<int64_t>(blocks_per_seq) * page_size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = move(m, c, n_forks, most, false, what, st);
  if (rc) return rc;
  cudaError_t e = launch_pdl(dk::pages::fork_kernel, dim3(dk::pages::kPlanCtas), dim3(dk::pages::kPlanThreads), 0, st, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return move(m, c, n_forks, most, true, what, st);
}

size_t dk_paged_compact_workspace_size(void) { return compact_ws_bytes(); }

int dk_paged_compact(const int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq,
                     const int32_t* kv_lens, const int32_t* new_lens, const int32_t* n_keep, const int32_t* keep,
                     int64_t keep_stride, int32_t keep_width, int32_t n_seqs, int32_t page_size, int32_t* lens_out,
                     int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out, int32_t* shares,
                     int64_t n_blocks, void* const* pools, int32_t n_pools, int64_t pool_stride_block,
                     int64_t pool_stride_head, int64_t pool_stride_tok, int32_t n_heads, int32_t head_dim,
                     int32_t element_size, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "paged_compact";
  int rc = check_table(block_table, block_table_stride, n_seqs, blocks_per_seq, page_size, what);
  if (rc) return rc;
  if (n_free < 0 || n_free > kI32Max || keep_width < 0 || n_seqs > kI32Max - 4096)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: negative size, or too many sequences or free blocks", what);
  const Pools c{pools, n_pools, pool_stride_block, pool_stride_head, pool_stride_tok, n_blocks, n_heads, head_dim,
                element_size};
  rc = check_pools(c, page_size, what);
  if (rc) return rc;
  if (shares && !free_blocks) return fail(DK_ERR_INVALID_ARGUMENT, "%s: shares need a free list", what);
  if (free_blocks && (!cursor || !cursor_out))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: a free list needs its cursor", what);
  if (shares && static_cast<int64_t>(n_seqs) * blocks_per_seq >= 1LL << 30)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: 2^30 table entries or more with shares", what);
  if (n_seqs == 0) return free_blocks ? keep_cursor(cursor, cursor_out, what, static_cast<cudaStream_t>(stream)) : DK_OK;
  if (!kv_lens || !new_lens || !n_keep || !lens_out || lens_out == kv_lens || lens_out == new_lens || lens_out == n_keep)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer, or lens_out is one of the inputs", what);
  rc = check_ws(workspace, workspace_bytes, compact_ws_bytes(), what);
  if (rc) return rc;
  dk::pages::ReleaseParams p{};
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.width = blocks_per_seq;
  p.kv = kv_lens;
  p.nw = new_lens;
  p.n_keep = n_keep;
  p.keep = keep;
  p.keep_stride = keep_stride;
  p.keep_width = keep_width;
  p.moves = keep && n_pools > 0;
  p.n = n_seqs;
  p.page = dk::divisor(page_size);
  p.lens_out = lens_out;
  p.free_list = free_blocks;
  p.n_free = n_free;
  p.cursor_in = cursor;
  p.cursor_out = cursor_out;
  p.shares = shares;
  p.n_blocks = n_blocks;
  p.ws = static_cast<int32_t*>(workspace);
  dk::pages::MoveParams m{};
  m.table = block_table;
  m.table_stride = block_table_stride;
  m.page = p.page;
  m.kv = kv_lens;
  m.n_keep = n_keep;
  m.keep = keep;
  m.keep_stride = keep_stride;
  m.keep_width = keep_width;
  m.width = blocks_per_seq;
  m.ws = p.ws;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t most = keep ? keep_width : 0;   // without `keep` the first tokens stay where they are
  rc = move(m, c, n_seqs, most, false, what, st);
  if (rc) return rc;
  cudaError_t e = launch_pdl(dk::pages::release_kernel, dim3(dk::pages::kPlanCtas), dim3(dk::pages::kPlanThreads), 0, st, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return move(m, c, n_seqs, most, true, what, st);
}

}  // extern "C"
