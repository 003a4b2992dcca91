// Host side of the decode attention kernel: schedule, argument checks, tensor maps and launch.
#pragma once

#include "dk_attention.cuh"
#include "dk_attention_state.h"
#include "dk_host.cuh"

namespace dk {
namespace host {

struct AttnPlan {
  int n_tiles, rows_cap, max_splits, spu, upt;
  size_t o_bytes, ml_bytes, cnt_bytes, total;
};

// Splits per CTA (schedule only; the arithmetic of a row never depends on it):
// enough CTAs to fill the GPU a few times over, at most 8 splits (2048 tokens)
// per CTA so long rows do not leave a tail.
inline AttnPlan plan_attention(int32_t n_tiles, int32_t rows_per_tile, int32_t hq, int32_t hkv, int32_t D,
                        int32_t max_kv_len) {
  AttnPlan pl{};
  const int G = (hkv > 0) ? hq / hkv : 1;
  pl.n_tiles = n_tiles;
  pl.rows_cap = (rows_per_tile <= 1) ? G : (dk::attn::kRows / G) * G;
  pl.max_splits = static_cast<int>(ceil_div(max_kv_len > 0 ? max_kv_len : 1, dk::attn::kSplit));
  const int64_t pairs = static_cast<int64_t>(n_tiles) * (hkv > 0 ? hkv : 1);
  const int64_t target = 4LL * sm_count(current_device());
  int64_t upt = (pairs >= target) ? 1 : ceil_div(target, pairs);
  if (upt > pl.max_splits) upt = pl.max_splits;
  int spu = static_cast<int>(ceil_div(pl.max_splits, upt));
  if (spu > 8) spu = 8;
  if (spu < 1) spu = 1;
  pl.spu = spu;
  pl.upt = static_cast<int>(ceil_div(pl.max_splits, spu));
  const size_t slots = static_cast<size_t>(n_tiles) * hkv * pl.max_splits * pl.rows_cap;
  pl.o_bytes = ceil_div(slots * D * sizeof(float), 256) * 256;
  pl.ml_bytes = ceil_div(slots * 2 * sizeof(float), 256) * 256;
  pl.cnt_bytes = static_cast<size_t>(n_tiles) * hkv * sizeof(int32_t);
  // scratch only when some tile's splits are spread over several CTAs
  pl.total = (pl.upt > 1) ? (kCounterBytes + pl.o_bytes + pl.ml_bytes) : 0;
  return pl;
}

template <typename T, int D, int KM, bool T1, bool ST>
int attn_launch_km(const dk::attn::KvMaps& maps, const dk::attn::Params& p, int64_t n_items, cudaStream_t st) {
  using C = dk::attn::Cfg<D, T1>;
  static bool done[kMaxDevices] = {false};
  static int resident[kMaxDevices][dk::attn::kRows + 1] = {};   // CTAs per SM, by rows_cap
  auto fn = dk::attn::attn_kernel<T, D, KM, T1, ST>;
  int rc = ensure_smem(fn, C::smem_bytes(dk::attn::kRows), done);
  if (rc) return rc;
  const int dev = current_device();
  const int smem = C::smem_bytes(p.rows_cap);
  int per_sm = 0;
  if (dev >= 0 && dev < kMaxDevices && p.rows_cap >= 0 && p.rows_cap <= dk::attn::kRows)
    per_sm = resident[dev][p.rows_cap];
  if (per_sm <= 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, dk::attn::kThreads, smem) != cudaSuccess ||
        per_sm <= 0)
      per_sm = 1;
    if (dev >= 0 && dev < kMaxDevices && p.rows_cap >= 0 && p.rows_cap <= dk::attn::kRows)
      resident[dev][p.rows_cap] = per_sm;
  }
  // persistent grid: every CTA resident at once, each walking items b, b + grid, ...
  const int64_t cap = static_cast<int64_t>(per_sm) * sm_count(dev);
  const int grid = static_cast<int>(n_items < cap ? n_items : cap);
  if (grid <= 0) return DK_OK;
  cudaError_t e = launch_pdl(fn, dim3(grid), dim3(dk::attn::kThreads), smem, st, maps, p);
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_batch_invariant: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

template <typename T, int D, bool ST>
int attn_launch(const dk::attn::KvMaps& maps, const dk::attn::Params& p, int64_t n_items,
                cudaStream_t st) {
  constexpr int kThr = dk::attn::kConsumerWarps * 32;
  constexpr int kNarrow = (4 < dk::attn::Cfg<D>::KMAX) ? 4 : dk::attn::Cfg<D>::KMAX;
  if (p.rows_cap == 1) return attn_launch_km<T, D, 1, true, ST>(maps, p, n_items, st);
  if (p.rows_cap * D <= kNarrow * kThr) return attn_launch_km<T, D, kNarrow, false, ST>(maps, p, n_items, st);
  return attn_launch_km<T, D, dk::attn::Cfg<D>::KMAX, false, ST>(maps, p, n_items, st);
}

// The invariant decode attention over a contiguous cache (pg == nullptr; kv_stride_seq /
// kv_n_seq / kv_capacity describe it) or a paged one (the strides describe the block pool;
// kv_n_seq is the number of block-table rows and the capacity blocks_per_seq * page).
// ST: each row's softmax states go to st_o / st_ml (see dk::attn::Params) and `out` is not used.
template <bool ST>
int attention_invariant_impl(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k,
                             const void* v, int64_t kv_stride_seq, int64_t kv_stride_head, int64_t kv_stride_tok,
                             int64_t kv_n_seq, int64_t kv_capacity, void* out, int64_t out_stride_row,
                             int64_t out_stride_head, const int32_t* kv_lens, int32_t uniform_kv_len,
                             const int32_t* row_tiles, int32_t n_tiles, int32_t n_rows, int32_t n_q_heads,
                             int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len, float scale, int dtype,
                             void* workspace, size_t workspace_bytes, void* stream, const PagedKV* pg,
                             const char* what, float* st_o = nullptr, float* st_ml = nullptr) {
  if (dtype != DK_BF16 && dtype != DK_F16) return fail(DK_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", what);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(DK_ERR_UNSUPPORTED, "%s: head_dim %d not in {32, 64, 128}", what, head_dim);
  if (n_rows < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad head counts", what);
  const int G = n_q_heads / n_kv_heads;
  if (G > dk::attn::kRows) return fail(DK_ERR_UNSUPPORTED, "%s: more than 16 query heads per kv head", what);
  if (n_kv_heads > 65535) return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many kv heads", what);
  if (n_rows == 0) return DK_OK;
  if (!q || !k || !v || (ST ? (!st_o || !st_ml) : !out)) return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (pg) {
    if (!pg->table || pg->page <= 0 || pg->page % dk::attn::kBlock || pg->blocks_per_seq <= 0 ||
        pg->n_blocks <= 0 || pg->n_blocks > 0x7fffffffLL || pg->table_stride < pg->blocks_per_seq)
      return fail(DK_ERR_INVALID_ARGUMENT,
                  "%s: paged KV needs a block table, page_size a multiple of %d, blocks_per_seq > 0, "
                  "n_blocks > 0 and block_table_stride >= blocks_per_seq", what, dk::attn::kBlock);
    kv_capacity = static_cast<int64_t>(pg->page) * pg->blocks_per_seq;
  }
  if (max_kv_len < 0 || kv_capacity <= 0 || kv_n_seq <= 0 || kv_capacity > 0x7fffffffLL || kv_n_seq > 0x7fffffffLL)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad KV extents", what);
  if (!kv_lens && (uniform_kv_len < 0 || uniform_kv_len > max_kv_len || uniform_kv_len > kv_capacity))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: uniform_kv_len out of range", what);
  if (!row_tiles) {
    n_tiles = n_rows;
    if (kv_n_seq < n_rows) return fail(DK_ERR_INVALID_ARGUMENT, "%s: fewer KV sequences than rows", what);
  } else if (n_tiles <= 0) {
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: n_tiles must be positive with row_tiles", what);
  }
  if (!aligned16(k) || !aligned16(v)) return fail(DK_ERR_INVALID_ARGUMENT, "%s: K/V must be 16-byte aligned", what);
  if ((kv_stride_tok * 2) % 16 || (kv_stride_head * 2) % 16 || (kv_stride_seq * 2) % 16)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: KV strides must be multiples of 8 elements", what);
  if ((reinterpret_cast<uintptr_t>(q) & 3u) || (q_stride_row & 1) || (q_stride_head & 1))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: q rows must be 4-byte aligned", what);

  const AttnPlan pl = plan_attention(n_tiles, row_tiles ? 2 : 1, n_q_heads, n_kv_heads, head_dim, max_kv_len);
  if (static_cast<int64_t>(pl.n_tiles) * pl.upt > 0x7fffffffLL)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: grid too large", what);
  if (pl.total > 0 && (!workspace || workspace_bytes < pl.total))
    return fail(DK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, pl.total, workspace_bytes);
  if (pl.total > 0 && !aligned16(workspace)) return fail(DK_ERR_WORKSPACE, "%s: workspace alignment", what);

  dk::attn::Params p{};
  p.q = q;
  p.q_sr = q_stride_row;
  p.q_sh = q_stride_head;
  p.out = out;
  p.o_sr = out_stride_row;
  p.o_sh = out_stride_head;
  p.kv_lens = kv_lens;
  p.uniform_len = uniform_kv_len;
  p.tiles = row_tiles;
  p.n_tiles = n_tiles;
  p.rows_cap = pl.rows_cap;
  p.n_rows = n_rows;
  p.hq = n_q_heads;
  p.hkv = n_kv_heads;
  p.G = G;
  p.max_splits = pl.max_splits;
  p.spu = pl.spu;
  p.upt = pl.upt;
  p.kv_capacity = static_cast<int32_t>(kv_capacity);
  p.kv_n_seq = static_cast<int32_t>(kv_n_seq);
  if (pg) {
    p.block_table = pg->table;
    p.bt_stride = pg->table_stride;
    p.page = pg->page;
    p.n_blocks = static_cast<int32_t>(pg->n_blocks);
  }
  p.st_o = st_o;
  p.st_ml = st_ml;
  p.scale_log2 = scale * 1.4426950408889634f;
  if (pl.total > 0) {
    if (static_cast<int64_t>(n_tiles) * n_kv_heads > kMaxCounters)
      return fail(DK_ERR_INVALID_ARGUMENT, "%s: %d tiles x %d kv heads exceed the workspace counter area", what,
                  n_tiles, n_kv_heads);
    uint8_t* w = ws_data(workspace);
    p.ws_o = reinterpret_cast<float*>(w);
    p.ws_ml = reinterpret_cast<float*>(w + pl.o_bytes);
    p.counters = static_cast<int32_t*>(workspace);
  }

  // K/V tensor maps: 4-D (d, token, kv head, sequence) -- or (d, token in block, kv head, block);
  // 64-token boxes for whole blocks, 16-token boxes for the tail of a split
  dk::attn::KvMaps maps;
  const int boxd = head_dim < 64 ? head_dim : 64;
  const uint64_t dims[4] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(pg ? pg->page : kv_capacity),
                            static_cast<uint64_t>(n_kv_heads), static_cast<uint64_t>(pg ? pg->n_blocks : kv_n_seq)};
  const uint64_t strides[3] = {static_cast<uint64_t>(kv_stride_tok) * 2, static_cast<uint64_t>(kv_stride_head) * 2,
                               static_cast<uint64_t>(kv_stride_seq) * 2};
  const uint32_t box[4] = {static_cast<uint32_t>(boxd), static_cast<uint32_t>(dk::attn::kBlock), 1, 1};
  const CUtensorMapSwizzle swz = (boxd == 64) ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const CUtensorMapDataType dt = (dtype == DK_BF16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint32_t box16[4] = {static_cast<uint32_t>(boxd), static_cast<uint32_t>(dk::attn::kTailRows), 1, 1};
  int rc = encode_map(&maps.k, dt, 4, k, dims, strides, box, swz, what);
  if (!rc) rc = encode_map(&maps.v, dt, 4, v, dims, strides, box, swz, what);
  if (!rc) rc = encode_map(&maps.k16, dt, 4, k, dims, strides, box16, swz, what);
  if (!rc) rc = encode_map(&maps.v16, dt, 4, v, dims, strides, box16, swz, what);
  if (rc) return rc;

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t n_items = static_cast<int64_t>(pl.n_tiles) * pl.upt * n_kv_heads;
  if (dtype == DK_BF16) {
    if (head_dim == 32) return attn_launch<__nv_bfloat16, 32, ST>(maps, p, n_items, st);
    if (head_dim == 64) return attn_launch<__nv_bfloat16, 64, ST>(maps, p, n_items, st);
    return attn_launch<__nv_bfloat16, 128, ST>(maps, p, n_items, st);
  }
  if (head_dim == 32) return attn_launch<__half, 32, ST>(maps, p, n_items, st);
  if (head_dim == 64) return attn_launch<__half, 64, ST>(maps, p, n_items, st);
  return attn_launch<__half, 128, ST>(maps, p, n_items, st);
}

}  // namespace host
}  // namespace dk
