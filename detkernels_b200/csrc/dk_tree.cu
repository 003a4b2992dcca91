// C ABI of the attention of drafted tokens (see include/detkernels_b200.h).
#include <algorithm>

#include "dk_common.cuh"
#include "dk_host.cuh"
#include "dk_tree.cuh"

namespace dk {
namespace host {
cudaError_t tree_status(int clear, int* code, int* detail) { return unit_status(clear, code, detail); }
}  // namespace host
}  // namespace dk

using namespace dk::host;

namespace {

constexpr int64_t kI32Max = 0x7fffffffLL;

// The most chunks that a sequence of at most max_kv_len tokens, max_rows of them drafts, is cut into.
int64_t max_chunks(int64_t max_kv_len, int64_t max_rows) {
  int64_t most = 1;
  // a chunk's size is constant between these lengths of the cached part, and then grows with it
  for (int64_t kv : {4096, 8192, 16384, 32768}) {
    kv = std::min(kv, max_kv_len);
    most = std::max(most, ceil_div(std::min(kv + max_rows, max_kv_len), dk::tree::chunk_tokens(kv)));
  }
  // beyond, it holds at least a 16th of the cached part, and 2048 tokens
  if (max_kv_len > 32768) most = std::max(most, 16 + ceil_div(max_rows, 2048) + 1);
  return most;
}

size_t state_o_bytes(int64_t chunks, int64_t st_rows, int64_t D) {
  return (static_cast<size_t>(chunks) * st_rows * D * sizeof(float) + 255) / 256 * 256;
}
size_t state_bytes(int64_t chunks, int64_t st_rows, int64_t D) {
  return chunks <= 1 ? 0 : state_o_bytes(chunks, st_rows, D) + static_cast<size_t>(chunks) * st_rows * 2 * sizeof(float);
}
// What the sizes alone decide of a call.
struct Schedule {
  int64_t chunks, st_rows, units;
  bool solo;             // an item a tile
  bool planned;          // more items, at most, than SMs: their order is planned
  size_t states, need;   // bytes of the states, and of the workspace: the states, then the items' order
};
Schedule schedule(int64_t n_seqs, int64_t n_rows, int64_t max_rows, int64_t hq, int64_t hkv, int64_t D, int64_t max_kv_len) {
  Schedule c{};
  c.chunks = max_chunks(max_kv_len, max_rows);
  c.st_rows = n_rows * hq;
  const int64_t tiles = ceil_div(max_rows, dk::tree::kRows / (hq / hkv));
  // Items a (sequence, chunk): pairs of tiles, or pairs of heads where the rows fit one tile; and where single tiles are no
  // more than the SMs, those, whose blocks take less time (4 requests of up to 700 tokens, 8 heads of 64: 12.3 and 14.9 us
  // in a graph; 8 of up to 2776, 3 heads of 128: 17.2 and 21.9).  A few tokens leave nothing to gain by it, and on more than
  // half of the SMs keep the next kernel from beginning beside them (22 requests of up to 18, 4 heads of 128: 8.5 and 6.6).
  const int64_t single = hkv * tiles * n_seqs * c.chunks, sms = sm_count(current_device());
  c.solo = single <= (max_kv_len > 256 ? sms : sms / 2);
  c.units = c.solo ? hkv * tiles : tiles > 1 ? hkv * ceil_div(tiles, 2) : ceil_div(hkv, 2);
  c.planned = c.units * n_seqs * c.chunks > sms;
  c.states = (state_bytes(c.chunks, c.st_rows, D) + 15) / 16 * 16;
  c.need = c.states + (c.planned ? static_cast<size_t>(dk::tree::plan_ints(n_seqs)) * sizeof(int32_t) : 0);
  return c;
}

template <typename T, int D>
int tree_launch(const dk::tree::Maps& maps, dk::tree::Params p, cudaStream_t st) {
  using C = dk::tree::Cfg<D>;
  static bool done[kMaxDevices] = {false};
  auto fn = dk::tree::tree_kernel<T, D>;
  int rc = ensure_smem(fn, C::SMEM, done);
  if (rc) return rc;
  static int regs[kMaxDevices] = {0};
  const int dev = current_device();
  if (dev < 0 || dev >= kMaxDevices || regs[dev] == 0) {
    cudaFuncAttributes a{};
    cudaError_t e = cudaFuncGetAttributes(&a, fn);
    if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_tree: %s", cudaGetErrorString(e));
    // The register split of the kernel is exact for this count, and for a kernel without calls or spills: a build that kept
    // functions out of line had the same count, did not hold its warps to their shares, and failed at launch.
    if (a.numRegs != dk::prefix::kLaunchRegs || a.localSizeBytes != 0)
      return fail(DK_ERR_UNSUPPORTED, "attention_tree: built with %d registers a thread, not %d, and %d bytes of local memory",
                  a.numRegs, dk::prefix::kLaunchRegs, static_cast<int>(a.localSizeBytes));
    if (dev >= 0 && dev < kMaxDevices) regs[dev] = a.numRegs;
  }
  // As many CTAs as SMs share the items, or, where even their bound is not more than that, each takes one at once.
  const int64_t items = static_cast<int64_t>(p.units) * p.n_seqs * p.max_chunks;
  cudaError_t e = cudaSuccess;
  if (p.plan) e = launch_pdl(dk::tree::plan_kernel<D>, dim3(1), dim3(dk::tree::kPlanThreads), 0, st, p);
  if (e == cudaSuccess) e = launch_pdl(fn, dim3(static_cast<unsigned>(std::min<int64_t>(items, sm_count(dev)))),
                             dim3(dk::tree::kThreads), C::SMEM, st, maps, p);
  if (e == cudaSuccess && p.max_chunks > 1) {
    const int64_t row_tiles = ceil_div(static_cast<int64_t>(p.max_rows) * p.G, 32);
    e = launch_pdl(dk::tree::join_kernel<T, D>, dim3(static_cast<unsigned>(row_tiles * p.hkv * p.n_seqs)),
                   dim3(dk::tree::kJoinThreads), 0, st, p, static_cast<int>(row_tiles));
  }
  if (e != cudaSuccess) return fail(DK_ERR_CUDA, "attention_tree: launch failed: %s", cudaGetErrorString(e));
  return DK_OK;
}

template <typename T>
int tree_for(int D, const dk::tree::Maps& maps, const dk::tree::Params& p, cudaStream_t st) {
  return D == 32 ? tree_launch<T, 32>(maps, p, st) : D == 64 ? tree_launch<T, 64>(maps, p, st) : tree_launch<T, 128>(maps, p, st);
}

}  // namespace

extern "C" {

size_t dk_attention_tree_workspace_size(int32_t n_seqs, int32_t n_rows, int32_t max_rows, int32_t n_q_heads,
                                        int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len) {
  if (n_seqs <= 0 || n_rows <= 0 || max_rows <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads ||
      n_q_heads / n_kv_heads > dk::tree::kRows || head_dim <= 0 || max_kv_len <= 0)
    return 0;
  max_rows = std::min(std::min(max_rows, n_rows), max_kv_len);
  return schedule(n_seqs, n_rows, max_rows, n_q_heads, n_kv_heads, head_dim, max_kv_len).need;
}

int dk_attention_tree(const void* q, int64_t q_stride_row, int64_t q_stride_head, const void* k, const void* v,
                      int64_t kv_stride_seq, int64_t kv_stride_head, int64_t kv_stride_tok, int64_t kv_n_seq,
                      int64_t kv_capacity, const int32_t* block_table, int64_t block_table_stride,
                      int32_t blocks_per_seq, int64_t n_blocks, int32_t page_size, void* out, int64_t out_stride_row,
                      int64_t out_stride_head, const int32_t* kv_lens, const int32_t* cu_rows, const int64_t* mask,
                      int64_t mask_stride, int32_t mask_words, int32_t n_seqs, int32_t n_rows, int32_t max_rows,
                      int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_kv_len, float scale,
                      int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "attention_tree";
  if (dtype != DK_BF16 && dtype != DK_F16) return fail(DK_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", what);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(DK_ERR_UNSUPPORTED, "%s: head_dim %d not in {32, 64, 128}", what, head_dim);
  if (n_rows < 0 || n_seqs < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || n_kv_heads > 65535)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad shape or head counts", what);
  const int G = n_q_heads / n_kv_heads;
  if (G > dk::tree::kRows) return fail(DK_ERR_UNSUPPORTED, "%s: more than 128 query heads per kv head", what);
  if (n_rows == 0 || n_seqs == 0) return DK_OK;
  if (mask_words <= 0 || max_rows <= 0 || max_kv_len <= 0)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: mask_words, max_rows and max_kv_len must be positive", what);
  if (!q || !k || !v || !out || !kv_lens || !cu_rows || !mask)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned16(q) || q_stride_row % 8 || q_stride_head % 8)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: q rows must be 16-byte aligned", what);
  if (!aligned16(k) || !aligned16(v) || kv_stride_seq % 8 || kv_stride_head % 8 || kv_stride_tok % 8)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: the caches need 16-byte aligned rows", what);
  if (block_table) {
    if (page_size <= 0 || page_size % 64 || blocks_per_seq <= 0 || n_blocks <= 0 || n_blocks > kI32Max ||
        (n_seqs > 1 && block_table_stride < blocks_per_seq))
      return fail(DK_ERR_INVALID_ARGUMENT,
                  "%s: a paged cache needs page_size a multiple of 64, blocks_per_seq > 0, n_blocks > 0 and "
                  "block_table_stride >= blocks_per_seq", what);
    kv_capacity = static_cast<int64_t>(page_size) * blocks_per_seq;
  } else if (kv_n_seq < n_seqs) {
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: fewer KV sequences than there are", what);
  }
  // whole blocks of the longest sequence stay inside 32 bits
  if (kv_capacity <= 0 || kv_capacity > kI32Max - 4096 || (!block_table && kv_n_seq > kI32Max))
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: bad KV extents", what);
  max_kv_len = static_cast<int32_t>(std::min<int64_t>(max_kv_len, kv_capacity));
  max_rows = std::min(std::min(max_rows, n_rows), max_kv_len);
  const int rpt = dk::tree::kRows / G;
  const Schedule c = schedule(n_seqs, n_rows, max_rows, n_q_heads, n_kv_heads, head_dim, max_kv_len);
  if (c.st_rows > kI32Max - 512 || static_cast<int64_t>(max_rows) * G > kI32Max - 512 ||
      c.units * n_seqs > kI32Max / 8 || c.units * n_seqs * c.chunks > kI32Max - 2 * sm_count(current_device()) ||
      ceil_div(static_cast<int64_t>(max_rows) * G, 32) * n_kv_heads * n_seqs > kI32Max)
    return fail(DK_ERR_INVALID_ARGUMENT, "%s: too many rows or sequences", what);
  if (c.need && (!workspace || workspace_bytes < c.need || !aligned16(workspace)))
    return fail(DK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, c.need, workspace_bytes);

  dk::tree::Params p{};
  p.hkv = n_kv_heads;
  p.G = G;
  p.rpt = rpt;
  p.group = dk::divisor31(G);
  p.n_seqs = n_seqs;
  p.n_rows = n_rows;
  p.max_rows = max_rows;
  p.kv_lens = kv_lens;
  p.cu_rows = cu_rows;
  p.mask = reinterpret_cast<const uint64_t*>(mask);
  p.mask_stride = mask_stride;
  p.words = mask_words;
  p.capacity = max_kv_len;
  p.units = static_cast<int32_t>(c.units);
  p.solo = c.solo ? 1 : 0;
  p.max_chunks = static_cast<int32_t>(c.chunks);
  p.v = v;
  p.c_sn = kv_stride_seq;
  p.c_sh = kv_stride_head;
  p.c_st = kv_stride_tok;
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.page = block_table ? page_size : 0;
  p.n_blocks = block_table ? static_cast<int32_t>(n_blocks) : 0;
  p.zero = scale == 0.0f ? 1 : 0;
  p.c = (p.zero ? 1.0f : fabsf(scale)) * 1.4426950408889634f;
  p.flip = scale < 0.0f ? 0x80008000u : 0u;
  p.out = out;
  p.o_sr = out_stride_row;
  p.o_sh = out_stride_head;
  p.o_vec = aligned16(out) && out_stride_row % 8 == 0 && out_stride_head % 8 == 0;
  p.st_rows = c.st_rows;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (c.states) {
    p.st_o = reinterpret_cast<float*>(ws);
    p.st_ml = reinterpret_cast<float*>(ws + state_o_bytes(c.chunks, c.st_rows, head_dim));
  }
  if (c.planned) p.plan = reinterpret_cast<int32_t*>(ws + c.states);

  dk::tree::Maps maps;
  const uint64_t dims[4] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(block_table ? page_size : kv_capacity),
                            static_cast<uint64_t>(n_kv_heads), static_cast<uint64_t>(block_table ? n_blocks : kv_n_seq)};
  const uint64_t strides[3] = {static_cast<uint64_t>(kv_stride_tok) * 2, static_cast<uint64_t>(kv_stride_head) * 2,
                               static_cast<uint64_t>(kv_stride_seq) * 2};
  const uint32_t box[4] = {64, 64, 1, 1};
  const CUtensorMapDataType dt = (dtype == DK_BF16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t q_dims[3] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(n_q_heads), static_cast<uint64_t>(n_rows)};
  const uint64_t q_strides[2] = {static_cast<uint64_t>(q_stride_head) * 2, static_cast<uint64_t>(q_stride_row) * 2};
  const uint32_t q_box[3] = {64, static_cast<uint32_t>(G), static_cast<uint32_t>(rpt)};
  int rc = encode_map(&maps.q, dt, 3, q, q_dims, q_strides, q_box, CU_TENSOR_MAP_SWIZZLE_128B, what);
  if (!rc) rc = encode_map(&maps.k, dt, 4, k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
  if (!rc) rc = encode_map(&maps.v, dt, 4, v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DK_BF16 ? tree_for<__nv_bfloat16>(head_dim, maps, p, st) : tree_for<__half>(head_dim, maps, p, st);
}

}  // extern "C"
