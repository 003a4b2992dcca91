// Page plan of one step: block-table growth, slot map and attention row tiles from request lengths.
//
// Sequence b holds kv[b] tokens and gets n[b] new ones.  With the exclusive sums over sequences
//   R[b] = sum n,   K[b] = sum (ceil((kv + n) / page) - ceil(kv / page)),   T[b] = sum ceil(n / rpt)
// the new table entries are table[b, ceil(kv / page) + i] = free[cursor + K[b] + i], row r of
// sequence b (r in [R[b], R[b + 1])) is token pos = kv[b] + r - R[b] of it, at slot
// table[b, pos / page] * page + pos % page, and tile T[b] + i covers rows R[b] + i rpt on.
//
// Two launches: one CTA validates the lengths and scans them, then a grid writes rows, table
// entries and tiles, each output element finding its sequence by binary search in the sums.
#pragma once

#include "dk_common.cuh"

namespace dk {
namespace paging {

constexpr int kScanThreads = 1024;
constexpr int kFillThreads = 256;

enum : int {
  kDetLens = 0x600,   // a negative length, or a sequence past its row of the block table
  kDetPool = 0x601,   // the free list is exhausted
  kDetRows = 0x602,   // more rows or tiles than the outputs hold
};

struct Params {
  int32_t* table;
  int64_t table_stride;
  int32_t width;            // entries of a table row
  const int32_t* kv;
  const int32_t* nw;
  int32_t n_seqs;
  int32_t page;
  const int32_t* free_list;  // null: the table does not grow
  int64_t n_free;
  const int32_t* cursor_in;
  int32_t* cursor_out;
  int32_t* cu_rows;         // [n_seqs + 1]
  int32_t* row_seq;         // null: no rows
  int32_t* row_pos;
  int64_t* slots;
  int32_t* q_lens;
  int64_t n_rows;
  int32_t* tiles;           // null: no tiles
  int32_t rpt;
  int64_t n_tiles;
  // scratch: [0] 1 when the plan stands, [1] cursor, then cu_blk [n_seqs + 1], cu_tile [n_seqs + 1]
  int32_t* ws;
};

__device__ __forceinline__ int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Sum3 {
  int64_t r, k, t;
};

__device__ __forceinline__ Sum3 warp_scan(Sum3 v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t r = __shfl_up_sync(0xffffffffu, v.r, d);
    const int64_t k = __shfl_up_sync(0xffffffffu, v.k, d);
    const int64_t t = __shfl_up_sync(0xffffffffu, v.t, d);
    if (lane >= d) {
      v.r += r;
      v.k += k;
      v.t += t;
    }
  }
  return v;
}

__global__ void __launch_bounds__(kScanThreads) scan_kernel(const Params p) {
  __shared__ Sum3 s_warp[32];
  __shared__ int s_bad;
  pdl_wait();
  if (threadIdx.x == 0) {
    pdl_launch_dependents();
    s_bad = 0;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t* cu_blk = p.ws + 2;
  int32_t* cu_tile = cu_blk + p.n_seqs + 1;
  Sum3 base{0, 0, 0};
  for (int b0 = 0; b0 < p.n_seqs; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    Sum3 v{0, 0, 0};
    if (b < p.n_seqs) {
      const int64_t kv = p.kv[b], n = p.nw[b];
      const int64_t have = ceil_div64(kv, p.page), need = ceil_div64(kv + n, p.page);
      if (kv < 0 || n < 0 || need > p.width) {
        s_bad = 1;
      } else {
        v.r = n;
        v.k = need - have;
        v.t = p.rpt > 0 ? ceil_div64(n, p.rpt) : 0;
      }
    }
    const Sum3 incl = warp_scan(v, lane);
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      const Sum3 w = s_warp[lane];
      const Sum3 wi = warp_scan(w, lane);
      s_warp[lane] = wi;
    }
    __syncthreads();
    Sum3 off = base;
    if (warp > 0) {
      off.r += s_warp[warp - 1].r;
      off.k += s_warp[warp - 1].k;
      off.t += s_warp[warp - 1].t;
    }
    if (b < p.n_seqs) {
      p.cu_rows[b] = static_cast<int32_t>(off.r + incl.r - v.r);
      cu_blk[b] = static_cast<int32_t>(off.k + incl.k - v.k);
      cu_tile[b] = static_cast<int32_t>(off.t + incl.t - v.t);
    }
    const Sum3 tot = s_warp[31];
    base.r += tot.r;
    base.k += tot.k;
    base.t += tot.t;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.cu_rows[p.n_seqs] = static_cast<int32_t>(base.r);
    cu_blk[p.n_seqs] = static_cast<int32_t>(base.k);
    cu_tile[p.n_seqs] = static_cast<int32_t>(base.t);
    const int64_t cur = p.free_list ? *p.cursor_in : 0;
    int bad = 0;
    if (s_bad) {
      bad = kDetLens;
    } else if (p.free_list && (cur < 0 || cur + base.k > p.n_free)) {
      bad = kDetPool;
    } else if (base.r > 0x7fffffffLL || (p.row_seq && base.r > p.n_rows) || (p.tiles && base.t > p.n_tiles)) {
      bad = kDetRows;
    }
    if (bad) report_error(DK_ERR_DEVICE_CHECK, bad);
    if (p.cursor_out) *p.cursor_out = static_cast<int32_t>(bad ? cur : cur + base.k);
    p.ws[1] = static_cast<int32_t>(cur);
    p.ws[0] = bad ? 0 : 1;
  }
}

// The last b with cu[b] <= x (cu ascending, cu[0] = 0 <= x < cu[n]): the sequence element x belongs to.
__device__ __forceinline__ int find_seq(const int32_t* cu, int n, int32_t x) {
  int lo = 0, hi = n;   // cu[lo] <= x < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kFillThreads) fill_kernel(const Params p) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  if (p.ws[0] == 0) return;
  const int64_t cursor = p.ws[1];
  const int32_t* cu_blk = p.ws + 2;
  const int32_t* cu_tile = cu_blk + p.n_seqs + 1;
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * kFillThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kFillThreads;
  if (p.row_seq) {
    const int64_t n = p.cu_rows[p.n_seqs];
    for (int64_t r = tid; r < n; r += step) {
      const int b = find_seq(p.cu_rows, p.n_seqs, static_cast<int32_t>(r));
      const int32_t kv = p.kv[b];
      const int32_t pos = kv + static_cast<int32_t>(r) - p.cu_rows[b];
      const int32_t pg = pos / p.page;
      const int32_t have = static_cast<int32_t>(ceil_div64(kv, p.page));
      const int64_t blk = (p.free_list && pg >= have) ? p.free_list[cursor + cu_blk[b] + (pg - have)]
                                                      : p.table[b * p.table_stride + pg];
      p.row_seq[r] = b;
      p.row_pos[r] = pos;
      p.slots[r] = blk * p.page + (pos - pg * p.page);
      p.q_lens[r] = pos + 1;
    }
  }
  if (p.free_list) {
    const int64_t n = cu_blk[p.n_seqs];
    for (int64_t j = tid; j < n; j += step) {
      const int b = find_seq(cu_blk, p.n_seqs, static_cast<int32_t>(j));
      const int64_t have = ceil_div64(p.kv[b], p.page);
      p.table[b * p.table_stride + have + (j - cu_blk[b])] = p.free_list[cursor + j];
    }
  }
  if (p.tiles) {
    const int64_t n = cu_tile[p.n_seqs];
    for (int64_t t = tid; t < n; t += step) {
      const int b = find_seq(cu_tile, p.n_seqs, static_cast<int32_t>(t));
      const int32_t at = static_cast<int32_t>(t - cu_tile[b]) * p.rpt;
      p.tiles[3 * t + 0] = p.cu_rows[b] + at;
      p.tiles[3 * t + 1] = min(p.rpt, p.nw[b] - at);
      p.tiles[3 * t + 2] = b;
    }
  }
}

}  // namespace paging
}  // namespace dk
