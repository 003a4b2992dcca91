// C ABI of the serving operators (see include/detkernels_b200.h): the page plan of a step, the
// per-head norm with rotation into a KV cache, and attention over a shared prefix.
#include <algorithm>

#include "dk_common.cuh"
#include "dk_host.cuh"
#include "dk_paging.cuh"
#include "dk_prefix.cuh"
#include "dk_rope.cuh"

namespace dk {
namespace host {
cudaError_t serving_status(int clear, int* code, int* detail) { return unit_status(clear, code, detail); }
}  // namespace host
}  // namespace dk

using namespace dk::host;

namespace {

constexpr int64_t kI32Max = 0x7fffffffLL;

// ============================ page plan ============================
size_t plan_ws_bytes(int64_t n_seqs) { return static_cast<size_t>(2 + 2 * (n_seqs + 1)) * sizeof(int32_t); }

// ============================ head norm + rotation ============================
template <typename T, int NC, bool INTER>
cudaError_t rope_vec(const dk::rope::Params& p, cudaStream_t st) {
  const int64_t want = ceil_div(p.n_rows * p.upr, dk::rope::kThreads / 32);
  const int64_t cap = 3LL * sm_count(current_device());   // resident CTAs; each walks units
  const int64_t grid = want < cap ? want : cap;
  return launch_pdl(dk::rope::vec_kernel<T, NC, INTER>, dim3(static_cast<unsigned>(grid)), dim3(dk::rope::kThreads), 0,
                    st, p);
}

template <typename T>
int rope_launch(dk::rope::Params& p, cudaStream_t st) {
  constexpr int N = dk::rope::Chunk<T>::N;
  auto ok16 = [](const void* ptr, int64_t a, int64_t b) { return !ptr || (aligned16(ptr) && a % N == 0 && b % N == 0); };
  bool vec = ok16(p.q, p.q_sr, p.q_sh) && ok16(p.k, p.k_sr, p.k_sh) && ok16(p.v, p.v_sr, p.v_sh) &&
             ok16(p.qo, p.qo_sr, p.qo_sh) && ok16(p.ko, p.ko_sr, p.ko_sh) && ok16(p.kc, p.c_sn, p.c_sh) &&
             ok16(p.vc, p.c_st, 0) && aligned16(p.table) && p.D % N == 0;
  int nc = 0;
  if (vec) {
    const int chunks = p.D / N;
    if (p.interleaved) {
      vec = chunks % 2 == 0 && p.rd % N == 0;   // whole chunks are rotated
      nc = 2;
      p.lanes = chunks / 2;
    } else {
      const int hc = p.rd / 2 / N;
      vec = (p.rd / 2) % N == 0 && chunks % hc == 0;
      if (vec) {
        p.lanes = hc;
        nc = chunks / hc;
        vec = nc == 2 || nc == 4;
      }
    }
    vec = vec && p.lanes <= 32;
  }
  cudaError_t e;
  if (vec) {
    p.glog = 0;
    while ((1 << p.glog) < p.lanes) ++p.glog;
    const int gpw = 32 >> p.glog;
    // vectors a warp walks: a whole row when the rows alone fill the GPU (one place look-up and one set of
    // pointers a row), otherwise one vector a group (24 vectors of 64 a row: 8 rows 2.9 us against 4.3 in whole
    // rows, 1000 rows 3.8 against 4.5; 4000 rows 9.2 against 8.4, 10,000 rows 19.8 against 15.6)
    const int64_t full = 16LL * sm_count(current_device());
    const int per = (p.n_rows >= full) ? static_cast<int>(ceil_div(p.nvec, gpw)) : 1;
    p.vpu = per * gpw;
    p.upr = static_cast<int>(ceil_div(p.nvec, p.vpu));
    if (p.n_rows * p.upr > kI32Max - (1 << 20)) return fail(DK_ERR_INVALID_ARGUMENT, "qk_norm_rope: too many rows");
    if (p.interleaved) e = rope_vec<T, 2, true>(p, st);
    else if (nc == 2) e = rope_vec<T, 2, false>(p, st);
    else e = rope_vec<T, 4, false>(p, st);
  } else {
    const int64_t want = ceil_div(p.n_rows * p.nvec, dk::rope::kThreads / 32);
    const int64_t cap = 8LL * sm_count(current_device());
    e = launch_pdl(dk::rope::any_kernel<T>, dim3(static_cast<unsigned>(want < cap ? want : cap)),
                   dim3(dk::rope::kThreads), 0, st, p);
  }
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "qk_norm_rope: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

// ============================ shared prefix ============================
struct PrefixPlan {
  int64_t rg;           // rows * G
  int chunk_blocks, n_chunks, run_blocks, n_runs, n_pairs, per_group;
  bool whole;           // a run is a whole group of chunks
  int max_splits, spu, upt, own_states;   // own tokens: splits a row, splits a unit, units a (tile, head), states a row
};

// Schedule (the bits are the same for every choice).  Prefix: a whole group of chunks a run, or a chunk a
// run, whose states then travel through memory, which costs about two fifths of a chunk's time; the fewer
// units of a chunk's time, counting the waves of CTAs that either takes.  (Bf16, groups against chunks: 512
// rows of 32 heads of 128 on 4, 8191 tokens: 90 against 112 us; 800 rows of 24 on 8, 5000 tokens: 139 against
// 128; 2000 rows of 32 heads of 64 on 8, 2048 tokens: 114 against 138; 160 rows of 32 on 16, 8192: 119 against
// 48.)  Own tokens: all
// splits of a (tile, KV head) by one warp, which then also joins the prefix's states and writes the output,
// when there are 12 such warps an SM (512 rows of 4 KV heads, 1 to 127 tokens: 125 us against 144 split up);
// else enough units for three waves, and combine_kernel.
PrefixPlan plan_prefix(int64_t n_rows, int64_t n_tiles, int64_t hkv, int64_t G, int64_t head_dim, int64_t prefix_len,
                       int64_t max_kv_len) {
  PrefixPlan pl{};
  const int sms = sm_count(current_device());
  pl.rg = n_rows * G;
  const int block = dk::prefix::block_tokens(static_cast<int>(head_dim));
  pl.chunk_blocks = static_cast<int>(dk::prefix::chunk_tokens(prefix_len, static_cast<int>(head_dim)) / block);
  const int64_t blocks = ceil_div(prefix_len, block);
  pl.n_chunks = static_cast<int>(ceil_div(blocks, pl.chunk_blocks));
  pl.n_pairs = static_cast<int>(ceil_div(pl.rg, 2 * dk::prefix::kRows));
  const int gc = dk::prefix::group_chunks(static_cast<int>(head_dim));
  const int64_t groups = ceil_div(pl.n_chunks, gc);
  const int64_t heads = pl.n_pairs * hkv;
  const bool whole = pl.whole = pl.n_chunks > 1 && 5 * ceil_div(groups * heads, sms) * std::min(gc, pl.n_chunks) <=
                                                       7 * ceil_div(pl.n_chunks * heads, sms);
  pl.run_blocks = pl.chunk_blocks * (whole ? gc : 1);
  pl.n_runs = static_cast<int>(whole ? groups : pl.n_chunks);
  pl.per_group = whole ? 1 : gc;
  pl.max_splits = static_cast<int>(ceil_div(max_kv_len, dk::own::kSplit));
  if (pl.max_splits > 0) {
    const int64_t units = n_tiles * hkv;
    const int64_t target = 3LL * (head_dim == 128 ? 9 : 14) * sms;
    int64_t upt = units >= 12LL * sms ? 1 : ceil_div(target, units);
    if (upt > pl.max_splits) upt = pl.max_splits;
    pl.spu = static_cast<int>(ceil_div(pl.max_splits, upt));
    pl.upt = static_cast<int>(ceil_div(pl.max_splits, pl.spu));
    pl.own_states = pl.upt == 1 ? 0 : pl.max_splits;
  }
  return pl;
}

size_t state_o_bytes(const PrefixPlan& pl, int64_t st_rows, int64_t D) {
  const size_t states = static_cast<size_t>(pl.n_runs + pl.own_states) * st_rows;
  return (states * D * sizeof(float) + 255) / 256 * 256;
}
size_t prefix_state_bytes(const PrefixPlan& pl, int64_t st_rows, int64_t D) {
  return state_o_bytes(pl, st_rows, D) + static_cast<size_t>(pl.n_runs + pl.own_states) * st_rows * 2 * sizeof(float);
}

template <typename T, int D, bool WHOLE>
int prefix_launch_as(const dk::prefix::Maps& maps, const dk::prefix::Params& p, cudaStream_t st) {
  using C = dk::prefix::Cfg<D, WHOLE>;
  static bool done[kMaxDevices] = {false};
  auto fn = dk::prefix::prefix_kernel<T, D, WHOLE>;
  int rc = ensure_smem(fn, C::SMEM, done);
  if (rc) return rc;
  static int regs[kMaxDevices] = {0};
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices || regs[dev] == 0) {
    cudaFuncAttributes a{};
    cudaError_t e = cudaFuncGetAttributes(&a, fn);
    if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_shared_prefix: %s", cudaGetErrorString(e));
    if (a.numRegs != dk::prefix::kLaunchRegs)   // the register split of the kernel is exact for this count
      return fail(DK_ERR_UNSUPPORTED, "attention_shared_prefix: built with %d registers a thread, not %d", a.numRegs,
                  dk::prefix::kLaunchRegs);
    if (dev >= 0 && dev < kMaxDevices) regs[dev] = a.numRegs;
  }
  const int64_t items = static_cast<int64_t>(p.n_pairs) * p.hkv * p.n_runs;
  const int sms = sm_count(dev);
  cudaError_t e = launch_pdl(fn, dim3(static_cast<unsigned>(items < sms ? items : sms)), dim3(dk::prefix::kThreads),
                             C::SMEM, st, maps, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_shared_prefix: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

template <typename T, int D>
int prefix_launch(const dk::prefix::Maps& maps, const dk::prefix::Params& p, bool whole, cudaStream_t st) {
  // up to head_dim 64 one form does both
  return D <= 64 || whole ? prefix_launch_as<T, D, true>(maps, p, st) : prefix_launch_as<T, D, D <= 64>(maps, p, st);
}

// Follows prefix_launch on the same stream and starts without waiting for it: prefix_kernel has itself
// waited for whatever wrote the inputs before it lets the next kernel begin.
template <typename T, int D, int NB>
int own_launch_nb(const dk::own::Params& p, cudaStream_t st) {
  using C = dk::own::Cfg<D>;
  auto fn = dk::own::own_kernel<T, D, NB>;
  const int smem = C::smem(NB, p.upt == 1);
  static bool done[kMaxDevices] = {false};
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices || !done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e != cudaSuccess) return fail(DK_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < kMaxDevices) done[dev] = true;
  }
  const int64_t grid = static_cast<int64_t>(p.n_tiles) * p.upt * p.hkv;
  cudaError_t e = launch_pdl(fn, dim3(static_cast<unsigned>(grid)), dim3(32), smem, st, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_shared_prefix: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

// Tiles of at most 8 query rows (a row without row_tiles and up to 8 heads a group) take the form of one
// column half (256 rows of 16 heads, 500 + 639 tokens: 63 us against 73 with two; 512 rows of 8 heads a KV head:
// 36 against 51); a query row's bits are the same in either.
template <typename T, int D>
int own_launch(const dk::own::Params& p, cudaStream_t st) {
  if (!p.tiles && p.G <= 8) return own_launch_nb<T, D, 1>(p, st);
  return own_launch_nb<T, D, 2>(p, st);
}

template <typename T, int D, int Q, int UN>
int combine_launch_q(const dk::prefix::CombineParams& p, cudaStream_t st) {
  using C = dk::prefix::CombineCfg<D, Q>;
  cudaError_t e = launch_pdl(dk::prefix::combine_kernel<T, D, Q, UN>,
                             dim3(static_cast<unsigned>(ceil_div(p.st_rows, 32)), D / C::COLS), dim3(C::WARPS * 32), 0,
                             st, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_shared_prefix: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

// Few CTAs (two an SM at most): one quad a thread and deep batches, since nothing else covers a batch's latency
// (64 rows of 16 heads of 64, 4096 + 640 tokens: 35 us against 42 with four quads; 200 rows of 16 heads of 128:
// 48 against 43).
template <typename T, int D>
int combine_launch(const dk::prefix::CombineParams& p, cudaStream_t st) {
  if (ceil_div(p.st_rows, 32) * (D / 32) <= 2LL * sm_count(current_device())) return combine_launch_q<T, D, 1, 8>(p, st);
  return combine_launch_q<T, D, 4, 2>(p, st);
}

// The entry points of the page plan differ in what becomes of the entries past its totals.
int paged_plan(const char* what, bool pad, int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq,
               const int32_t* kv_lens, const int32_t* new_lens, int32_t n_seqs, int32_t page_size,
               const int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out,
               int32_t* cu_rows, int32_t* row_seq, int32_t* row_pos, int64_t* slots, int32_t* q_lens, int64_t n_rows,
               int32_t* row_tiles, int32_t rows_per_tile, int64_t n_tiles, void* workspace, size_t workspace_bytes,
               void* stream) {
  if (n_seqs < 0 || page_size <= 0 || blocks_per_seq < 0 || n_rows < 0 || n_tiles < 0 || n_free < 0)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: negative size or page_size < 1", what);
  if (n_seqs == 0) return DK_OK;
  if (!kv_lens || !new_lens || !cu_rows || (blocks_per_seq > 0 && !block_table))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (n_seqs > 1 && block_table_stride < blocks_per_seq)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: block_table_stride < blocks_per_seq", what);
  if (static_cast<int64_t>(blocks_per_seq) * page_size > kI32Max)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: blocks_per_seq * page_size exceeds 2^31 - 1 tokens", what);
  if (n_rows > kI32Max || n_tiles > kI32Max || n_free > kI32Max)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: more than 2^31 - 1 rows, tiles or free blocks", what);
  if (free_blocks && (!cursor || !cursor_out))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: a free list needs its cursor", what);
  const bool rows = row_seq != nullptr;
  if (rows != (row_pos != nullptr) || rows != (slots != nullptr) || rows != (q_lens != nullptr))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: row_seq, row_pos, slots and q_lens go together", what);
  if (row_tiles && rows_per_tile <= 0) return fail(DK_ERR_INVALID_ARGUMENT, "%s: rows_per_tile < 1", what);
  if (!workspace || workspace_bytes < plan_ws_bytes(n_seqs) || (reinterpret_cast<uintptr_t>(workspace) & 3u))
    return fail(DK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, plan_ws_bytes(n_seqs),
                workspace_bytes);
  dk::paging::Params p{};
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.width = blocks_per_seq;
  p.kv = kv_lens;
  p.nw = new_lens;
  p.n_seqs = n_seqs;
  p.page = dk::divisor(page_size);
  p.free_list = free_blocks;
  p.n_free = n_free;
  p.cursor_in = cursor;
  p.cursor_out = free_blocks ? cursor_out : nullptr;
  p.cu_rows = cu_rows;
  p.row_seq = row_seq;
  p.row_pos = row_pos;
  p.slots = slots;
  p.q_lens = q_lens;
  p.n_rows = n_rows;
  p.tiles = row_tiles;
  p.tiled = row_tiles != nullptr;
  p.rpt = dk::divisor(row_tiles ? rows_per_tile : 1);
  p.n_tiles = n_tiles;
  p.ws = static_cast<int32_t*>(workspace);
  p.pad = pad;
  p.vec = aligned16(row_seq) && aligned16(row_pos) && aligned16(slots) && aligned16(q_lens);
  // at most so many outputs of each kind (the growth is known on the device only)
  int64_t most = rows ? n_rows : n_tiles;
  if (free_blocks && !rows) {
    const int64_t grow = static_cast<int64_t>(n_seqs) * blocks_per_seq;
    most = std::max(most, std::min(grow, n_free));
  }
  const bool fill = rows || row_tiles || free_blocks;
  // Few outputs, or a row a sequence, are written by the scan's own CTA in one pass: 4.5 us against 5.5 in two
  // launches for 7 rows, 4.5 against 6.0 for 64 sequences of 16, 13.4 against 14.8 for 4000 of one; but 7.8 against
  // 5.8 for 64 of 64.
  const int64_t pass = static_cast<int64_t>(dk::paging::kScanThreads) * dk::paging::kRowVec;
  const bool alone = fill && most <= std::max<int64_t>(pass / 4, std::min<int64_t>(n_seqs, pass));
  const int64_t busy = std::max<int64_t>(n_seqs, alone ? ceil_div(most, dk::paging::kRowVec) : 0);
  const dim3 threads(static_cast<unsigned>(
      std::max<int64_t>(64, std::min<int64_t>(dk::paging::kScanThreads, 32 * ceil_div(busy, 32)))));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = alone ? launch_pdl(dk::paging::scan_kernel<true>, dim3(1), threads, 0, st, p)
                        : launch_pdl(dk::paging::scan_kernel<false>, dim3(1), threads, 0, st, p);
  if (e == cudaSuccess && fill && !alone) {
    const int64_t run = dk::paging::kFillThreads * static_cast<int64_t>(rows ? dk::paging::kRowVec : 1);
    const int64_t want = ceil_div(most, run), cap = 64LL * sm_count(current_device());
    e = launch_pdl(dk::paging::fill_kernel, dim3(static_cast<unsigned>(std::min(want, cap))),
                   dim3(dk::paging::kFillThreads), 0, st, p);
  }
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return DK_OK;
}

}  // namespace

extern "C" {

size_t dk_paged_plan_workspace_size(int64_t n_seqs) { return n_seqs > 0 ? plan_ws_bytes(n_seqs) : 0; }

int dk_paged_plan(int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq, const int32_t* kv_lens,
                  const int32_t* new_lens, int32_t n_seqs, int32_t page_size, const int32_t* free_blocks,
                  int64_t n_free, const int32_t* cursor, int32_t* cursor_out, int32_t* cu_rows, int32_t* row_seq,
                  int32_t* row_pos, int64_t* slots, int32_t* q_lens, int64_t n_rows, int32_t* row_tiles,
                  int32_t rows_per_tile, int64_t n_tiles, void* workspace, size_t workspace_bytes, void* stream) {
  return paged_plan("paged_plan", false, block_table, block_table_stride, blocks_per_seq, kv_lens, new_lens, n_seqs,
                    page_size, free_blocks, n_free, cursor, cursor_out, cu_rows, row_seq, row_pos, slots, q_lens,
                    n_rows, row_tiles, rows_per_tile, n_tiles, workspace, workspace_bytes, stream);
}

int dk_paged_plan_padded(int32_t* block_table, int64_t block_table_stride, int32_t blocks_per_seq,
                         const int32_t* kv_lens, const int32_t* new_lens, int32_t n_seqs, int32_t page_size,
                         const int32_t* free_blocks, int64_t n_free, const int32_t* cursor, int32_t* cursor_out,
                         int32_t* cu_rows, int32_t* row_seq, int32_t* row_pos, int64_t* slots, int32_t* q_lens,
                         int64_t n_rows, int32_t* row_tiles, int32_t rows_per_tile, int64_t n_tiles, void* workspace,
                         size_t workspace_bytes, void* stream) {
  return paged_plan("paged_plan_padded", true, block_table, block_table_stride, blocks_per_seq, kv_lens, new_lens,
                    n_seqs, page_size, free_blocks, n_free, cursor, cursor_out, cu_rows, row_seq, row_pos, slots,
                    q_lens, n_rows, row_tiles, rows_per_tile, n_tiles, workspace, workspace_bytes, stream);
}

int dk_qk_norm_rope(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k, int64_t k_stride_row,
                    int64_t k_stride_head, const void* v, int64_t v_stride_row, int64_t v_stride_head, void* q_out,
                    int64_t q_out_stride_row, int64_t q_out_stride_head, void* k_out, int64_t k_out_stride_row,
                    int64_t k_out_stride_head, void* k_cache, void* v_cache, int64_t cache_stride_slab,
                    int64_t cache_stride_head, int64_t cache_stride_tok, int64_t cache_slabs, int64_t cache_capacity,
                    const int64_t* slots, const void* positions, int positions_64, const void* q_weight,
                    const void* k_weight, int weight_dtype, const float* rope_table, int64_t max_pos, int64_t n_rows,
                    int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t rotary_dim, int interleaved,
                    float eps, int dtype, void* stream) {
  const char* what = "qk_norm_rope";
  if (!valid_dtype(dtype) || !valid_dtype(weight_dtype)) return fail(DK_ERR_UNSUPPORTED, "%s: bad dtype", what);
  if (n_rows < 0 || n_q_heads < 0 || n_kv_heads < 0 || n_q_heads + static_cast<int64_t>(n_kv_heads) * 2 > 65535)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad shape", what);
  if (head_dim <= 0 || head_dim > dk::rope::kMaxDim)
    return fail(DK_ERR_UNSUPPORTED, "%s: head_dim %d not in [1, %d]", what, head_dim, dk::rope::kMaxDim);
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: rotary_dim must be even and in [2, head_dim]", what);
  if (n_rows == 0 || n_q_heads + n_kv_heads == 0) return DK_OK;
  if (n_rows > kI32Max) return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many rows", what);
  if ((n_q_heads && (!q || !q_out || !q_weight)) || (n_kv_heads && (!k || !k_weight)) || !positions || !rope_table ||
      max_pos <= 0)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer or empty table", what);
  const bool cache = k_cache != nullptr;
  if (cache != (v_cache != nullptr) || cache != (slots != nullptr) || cache != (v != nullptr))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: k_cache, v_cache, slots and v go together", what);
  if (!cache && n_kv_heads && !k_out) return fail(DK_ERR_INVALID_ARGUMENT, "%s: no destination for k", what);
  if (cache && (cache_slabs <= 0 || cache_capacity <= 0 || cache_capacity > kI32Max))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad cache extents", what);
  dk::rope::Params p{};
  p.q = q; p.q_sr = q_stride_row; p.q_sh = q_stride_head;
  p.k = k; p.k_sr = k_stride_row; p.k_sh = k_stride_head;
  p.v = v; p.v_sr = v_stride_row; p.v_sh = v_stride_head;
  p.qo = q_out; p.qo_sr = q_out_stride_row; p.qo_sh = q_out_stride_head;
  p.ko = k_out; p.ko_sr = k_out_stride_row; p.ko_sh = k_out_stride_head;
  p.kc = k_cache; p.vc = v_cache;
  p.c_sn = cache_stride_slab; p.c_sh = cache_stride_head; p.c_st = cache_stride_tok;
  p.n_slabs = cache_slabs; p.cap = cache_capacity;
  p.slots = slots;
  p.pos = positions; p.pos64 = positions_64;
  p.qw = q_weight; p.kw = k_weight; p.wdtype = weight_dtype;
  p.table = rope_table; p.max_pos = max_pos;
  p.n_rows = n_rows;
  p.H = n_q_heads; p.Hkv = n_kv_heads; p.D = head_dim; p.rd = rotary_dim; p.interleaved = interleaved ? 1 : 0;
  p.eps = eps;
  p.inv_d = 1.0f / static_cast<float>(head_dim);
  p.nvec = n_q_heads + n_kv_heads * (cache ? 2 : 1);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DK_F32) return rope_launch<float>(p, st);
  if (dtype == DK_F16) return rope_launch<__half>(p, st);
  return rope_launch<__nv_bfloat16>(p, st);
}

size_t dk_attention_shared_prefix_workspace_size(int32_t n_rows, int32_t n_tiles, int32_t n_q_heads, int32_t n_kv_heads,
                                      int32_t head_dim, int32_t prefix_len, int32_t max_kv_len) {
  if (n_rows <= 0 || n_tiles <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads || head_dim <= 0 ||
      prefix_len <= 0 || max_kv_len < 0)
    return 0;
  return prefix_state_bytes(plan_prefix(n_rows, n_tiles, n_kv_heads, n_q_heads / n_kv_heads, head_dim, prefix_len,
                                        max_kv_len),
                            static_cast<int64_t>(n_rows) * n_q_heads, head_dim);
}

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
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "attention_shared_prefix";
  if (dtype != DK_BF16 && dtype != DK_F16) return fail(DK_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", what);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(DK_ERR_UNSUPPORTED, "%s: head_dim %d not in {32, 64, 128}", what, head_dim);
  if (n_rows < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || n_kv_heads > 65535)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad head counts", what);
  const int G = n_q_heads / n_kv_heads;
  if (G > dk::own::kRows) return fail(DK_ERR_UNSUPPORTED, "%s: more than 16 query heads per kv head", what);
  if (prefix_len <= 0) return fail(DK_ERR_INVALID_ARGUMENT, "%s: prefix_len must be positive", what);
  if (max_kv_len < 0) return fail(DK_ERR_INVALID_ARGUMENT, "%s: max_kv_len < 0", what);
  if (n_rows == 0) return DK_OK;
  if (!q || !k_prefix || !v_prefix || !out) return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned16(q) || q_stride_row % 8 || q_stride_head % 8)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: q rows must be 16-byte aligned", what);
  if (!aligned16(k_prefix) || !aligned16(v_prefix) || prefix_stride_tok % 8 || prefix_stride_head % 8 ||
      prefix_stride_block % 8)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: the prefix needs 16-byte aligned rows", what);
  if (prefix_blocks && (prefix_page <= 0 || prefix_page % 64 || prefix_pool_blocks <= 0 || prefix_pool_blocks > kI32Max))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: a paged prefix needs a page size that is a multiple of 64", what);
  const bool own = max_kv_len > 0;
  if (own) {
    if (!k || !v || !kv_lens) return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (!aligned16(k) || !aligned16(v) || kv_stride_seq % 8 || kv_stride_head % 8 || kv_stride_tok % 8)
      return fail(DK_ERR_INVALID_ARGUMENT, "%s: the caches need 16-byte aligned rows", what);
    if (block_table) {
      if (page_size <= 0 || page_size % 64 || blocks_per_seq <= 0 || n_blocks <= 0 || n_blocks > kI32Max ||
          block_table_stride < blocks_per_seq)
        return fail(DK_ERR_INVALID_ARGUMENT,
                    "%s: a paged cache needs page_size a multiple of 64, blocks_per_seq > 0, n_blocks > 0 and "
                    "block_table_stride >= blocks_per_seq", what);
      kv_capacity = static_cast<int64_t>(page_size) * blocks_per_seq;
    }
    // whole splits of the longest row stay inside 32 bits
    if (kv_capacity <= 0 || kv_n_seq <= 0 || kv_capacity > kI32Max - (dk::own::kSplit - 1) || kv_n_seq > kI32Max)
      return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad KV extents", what);
    if (max_kv_len > kv_capacity) max_kv_len = static_cast<int32_t>(kv_capacity);
    if (!row_tiles && kv_n_seq < n_rows) return fail(DK_ERR_INVALID_ARGUMENT, "%s: fewer KV sequences than rows", what);
  }
  if (!row_tiles) n_tiles = n_rows;
  if (n_tiles <= 0) return fail(DK_ERR_INVALID_ARGUMENT, "%s: n_tiles must be positive with row_tiles", what);
  const int64_t st_rows = static_cast<int64_t>(n_rows) * n_q_heads;
  const PrefixPlan pl = plan_prefix(n_rows, n_tiles, n_kv_heads, G, head_dim, prefix_len, max_kv_len);
  if (st_rows > kI32Max || static_cast<int64_t>(n_tiles) * n_kv_heads * (pl.upt > 0 ? pl.upt : 1) > kI32Max ||
      static_cast<int64_t>(pl.n_pairs) * n_kv_heads * pl.n_runs > kI32Max - 2 * sm_count(current_device()))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many rows", what);
  const size_t need = prefix_state_bytes(pl, st_rows, head_dim);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(DK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);

  float* st_o = static_cast<float*>(workspace);
  float* st_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + state_o_bytes(pl, st_rows, head_dim));
  dk::prefix::Params p{};
  p.q = q;
  p.q_sr = q_stride_row;
  p.q_sh = q_stride_head;
  p.hq = n_q_heads;
  p.hkv = n_kv_heads;
  p.G = G;
  p.group = dk::divisor31(G);
  p.rg = static_cast<int32_t>(pl.rg);
  p.prefix_len = prefix_len;
  p.chunk_blocks = pl.chunk_blocks;
  p.run_blocks = pl.run_blocks;
  p.n_runs = pl.n_runs;
  p.n_pairs = pl.n_pairs;
  p.blocks = prefix_blocks;
  p.page = prefix_blocks ? prefix_page : 0;
  p.n_blocks = prefix_blocks ? static_cast<int32_t>(prefix_pool_blocks) : 0;
  p.zero = scale == 0.0f ? 1 : 0;
  p.c = (p.zero ? 1.0f : fabsf(scale)) * 1.4426950408889634f;
  p.flip = scale < 0.0f ? 0x80008000u : 0u;
  p.st_rows = st_rows;
  p.st_o = st_o;
  p.st_ml = st_ml;

  // K/V prefix maps: (d, token, kv head, block); a contiguous prefix is one block of prefix_len tokens,
  // so that what lies behind it reads as zero
  dk::prefix::Maps maps;
  const uint64_t dims[4] = {static_cast<uint64_t>(head_dim),
                            static_cast<uint64_t>(prefix_blocks ? prefix_page : prefix_len),
                            static_cast<uint64_t>(n_kv_heads),
                            static_cast<uint64_t>(prefix_blocks ? prefix_pool_blocks : 1)};
  const uint64_t block_stride = prefix_blocks ? static_cast<uint64_t>(prefix_stride_block) * 2
                                              : static_cast<uint64_t>(prefix_stride_head) * 2;
  const uint64_t strides[3] = {static_cast<uint64_t>(prefix_stride_tok) * 2,
                               static_cast<uint64_t>(prefix_stride_head) * 2, block_stride};
  const uint32_t box[4] = {64, 64, 1, 1};
  const CUtensorMapDataType dt = (dtype == DK_BF16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  int rc = encode_map(&maps.k, dt, 4, k_prefix, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
  if (!rc) rc = encode_map(&maps.v, dt, 4, v_prefix, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
  if (rc) return rc;

  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define DK_DISPATCH_16(FN, ...)                                                                \
  (dtype == DK_BF16 ? (head_dim == 32   ? FN<__nv_bfloat16, 32>(__VA_ARGS__)                   \
                       : head_dim == 64 ? FN<__nv_bfloat16, 64>(__VA_ARGS__)                   \
                                        : FN<__nv_bfloat16, 128>(__VA_ARGS__))                 \
                    : (head_dim == 32   ? FN<__half, 32>(__VA_ARGS__)                          \
                       : head_dim == 64 ? FN<__half, 64>(__VA_ARGS__)                          \
                                        : FN<__half, 128>(__VA_ARGS__)))
  rc = DK_DISPATCH_16(prefix_launch, maps, p, pl.whole, st);
  if (rc) return rc;
  int32_t own_max = 0;
  if (own) {
    dk::own::Params o{};
    o.q = q;
    o.q_sr = q_stride_row;
    o.q_sh = q_stride_head;
    o.k = k;
    o.v = v;
    o.c_sn = kv_stride_seq;
    o.c_sh = kv_stride_head;
    o.c_st = kv_stride_tok;
    o.kv_lens = kv_lens;
    o.tiles = row_tiles;
    o.n_tiles = n_tiles;
    o.n_rows = n_rows;
    o.hq = n_q_heads;
    o.hkv = n_kv_heads;
    o.G = G;
    o.n_seq = static_cast<int32_t>(kv_n_seq);
    o.capacity = max_kv_len;
    o.block_table = block_table;
    o.bt_stride = block_table_stride;
    o.page = block_table ? page_size : 0;
    o.n_blocks = static_cast<int32_t>(n_blocks);
    o.max_splits = pl.max_splits;
    o.spu = pl.spu;
    o.upt = pl.upt;
    o.scale_log2 = scale * 1.4426950408889634f;
    o.st_rows = st_rows;
    o.st_o = st_o + static_cast<int64_t>(pl.n_runs) * st_rows * head_dim;
    o.st_ml = st_ml + static_cast<int64_t>(pl.n_runs) * st_rows * 2;
    if (pl.upt == 1) {
      o.out = out;
      o.o_sr = out_stride_row;
      o.o_sh = out_stride_head;
      o.px_o = st_o;
      o.px_ml = st_ml;
      o.n_runs = pl.n_runs;
      o.per_group = pl.per_group;
    }
    own_max = o.capacity;
    rc = DK_DISPATCH_16(own_launch, o, st);
    if (rc || pl.upt == 1) return rc;
  }
  dk::prefix::CombineParams c{};
  c.st_o = st_o;
  c.st_ml = st_ml;
  c.n_runs = pl.n_runs;
  c.per_group = pl.per_group;
  c.kv_lens = own ? kv_lens : nullptr;
  c.own_max = own_max;
  if (row_tiles) {
    c.tiles = row_tiles;
    c.n_tiles = n_tiles;
    c.n_seq = static_cast<int32_t>(own ? kv_n_seq : kI32Max);   // without own tokens no sequence is read
    c.report = !own;
  }
  c.n_rows = n_rows;
  c.st_rows = st_rows;
  c.rg = pl.rg;
  c.G = G;
  c.group = p.group;
  c.out = out;
  c.o_sr = out_stride_row;
  c.o_sh = out_stride_head;
  return DK_DISPATCH_16(combine_launch, c, st);
}

}  // extern "C"
