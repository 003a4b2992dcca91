// Page plan of one step: block-table growth, slot map and attention row tiles from request lengths.
//
// Sequence b holds kv[b] tokens and gets n[b] new ones.  With the exclusive sums over sequences
//   R[b] = sum n,   K[b] = sum (ceil((kv + n) / page) - ceil(kv / page)),   T[b] = sum ceil(n / rpt)
// the new table entries are table[b, ceil(kv / page) + i] = free[cursor + K[b] + i], row r of
// sequence b (r in [R[b], R[b + 1])) is token pos = kv[b] + r - R[b] of it, at slot
// table[b, pos / page] * page + pos % page, and tile T[b] + i covers rows R[b] + i rpt on.
//
// One CTA validates the lengths and scans them, then rows are written: a CTA takes a run of rows,
// finds the sequences of its two ends by a 32-way search in the sums, and a thread finds the first of
// its four consecutive rows between those.  The row that opens a new page also writes the table entry,
// and the row that opens a tile the tile, so that one search serves all outputs.  Bound by the 20
// bytes stored per row when rows are many, by the latency of the two kernels' loads when they are few.
// Inside a graph: 5 us for 7 sequences, 7 us for 256 prompts (66,377 rows), 23 us for 4099 prompts (2.1 M
// rows, floor 7 us), of which the scan takes 9 and the search and the look-ups 13; the stores add 2.  Padding what lies
// behind the plan's totals adds 0.1 to 0.3 us where nothing does (7, 66,377 and 2.1 M rows).
#pragma once

#include "dk_common.cuh"
#include "dk_divide.cuh"

namespace dk {
namespace paging {

constexpr int kScanThreads = 1024;
constexpr int kScanItems = 8;     // sequences a thread scans in one round, at most
constexpr int kFillThreads = 256;
constexpr int kRowVec = 4;        // consecutive rows of a thread

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
  Divisor page;
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
  int32_t tiled;            // tiles of rpt.d rows are asked for
  Divisor rpt;
  int64_t n_tiles;
  int vec;                  // the row outputs take 16-byte stores
  int pad;                  // entries past the totals (all, when the plan is refused) become neutral
  // scratch: [0] 1 when the plan stands, [1] cursor, then cu_blk [n_seqs + 1], cu_tile [n_seqs + 1]
  int32_t* ws;
};

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

// The last b with cu[b] <= x (cu ascending, cu[0] = 0 <= x < cu[n]): the sequence element x belongs to,
// between lo and hi (cu[lo] <= x < cu[hi]).
__device__ __forceinline__ int find_seq(const int32_t* cu, int lo, int hi, int32_t x) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}
// The same by a whole warp, 32 ways a step.
__device__ __forceinline__ int find_seq_warp(const int32_t* cu, int n, int32_t x, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int at = lo + (lane + 1) * step;
    const int below = __popc(__ballot_sync(0xffffffffu, at < hi && cu[at] <= x));
    lo += below * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Rows, and with them the new table entries and the tiles (block-wide, CTA `cta` of `ctas`).
__device__ void fill_rows(const Params& p, int64_t cursor, int cta, int ctas) {
  __shared__ int s_end[2];
  const int32_t* cu = p.cu_rows;
  const int32_t* cu_blk = p.ws + 2;
  const int32_t* cu_tile = cu_blk + p.n_seqs + 1;
  const int64_t n = cu[p.n_seqs];
  const int64_t run = static_cast<int64_t>(blockDim.x) * kRowVec;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t page = p.page.d;
  for (int64_t r0 = cta * run; r0 < n; r0 += ctas * run) {
    if (warp < 2) {
      const int64_t x = warp == 0 ? r0 : (r0 + run < n ? r0 + run : n) - 1;
      const int b = find_seq_warp(cu, p.n_seqs, static_cast<int32_t>(x), lane);
      if (lane == 0) s_end[warp] = b;
    }
    __syncthreads();
    const int64_t r = r0 + static_cast<int64_t>(threadIdx.x) * kRowVec;
    if (r < n) {
      const int first = static_cast<int>(r);
      const int cnt = n - r < kRowVec ? static_cast<int>(n - r) : kRowVec;
      const int last_seq = s_end[1];
      int b = find_seq(cu, s_end[0], last_seq + 1, first);
      int begin = 0, end = 0;          // rows of sequence b
      uint32_t pg = 0, off = 0, have = 0;
      int32_t kv = 0;
      int64_t blk = 0;
      bool fresh = true;               // the page's block is not known yet
      int seq[kRowVec], pos[kRowVec];
      int64_t slot[kRowVec];
#pragma unroll
      for (int i = 0; i < kRowVec; ++i) {
        if (i < cnt) {
          if (i == 0 || first + i >= end) {
            if (i > 0) b = find_seq(cu, b + 1, last_seq + 1, first + i);
            begin = cu[b];
            end = cu[b + 1];
            kv = p.kv[b];
            have = ceil_div32(kv, p.page);
            const uint32_t at = static_cast<uint32_t>(kv + (first + i - begin));
            pg = div_by(at, p.page);
            off = at - pg * page;
            fresh = true;
          } else if (++off == page) {
            off = 0;
            ++pg;
            fresh = true;
          }
          if (fresh) {
            if (p.free_list && pg >= have) {
              const int32_t got = p.free_list[cursor + cu_blk[b] + (pg - have)];
              // a new page's first token is one of the new rows
              if (off == 0) p.table[b * p.table_stride + pg] = got;
              blk = got;
            } else {
              blk = p.table[b * p.table_stride + pg];
            }
            fresh = false;
          }
          seq[i] = b;
          pos[i] = kv + (first + i - begin);
          slot[i] = blk * page + off;
          if (p.tiles) {
            const uint32_t in = first + i - begin;
            const uint32_t tile = div_by(in, p.rpt);
            if (tile * p.rpt.d == in) {
              int32_t* t = p.tiles + 3 * (static_cast<int64_t>(cu_tile[b]) + tile);
              t[0] = first + i;
              t[1] = min(static_cast<int>(p.rpt.d), end - (first + i));
              t[2] = b;
            }
          }
        }
      }
      if (p.vec && cnt == kRowVec) {
        *reinterpret_cast<int4*>(p.row_seq + r) = make_int4(seq[0], seq[1], seq[2], seq[3]);
        *reinterpret_cast<int4*>(p.row_pos + r) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        *reinterpret_cast<int4*>(p.q_lens + r) = make_int4(pos[0] + 1, pos[1] + 1, pos[2] + 1, pos[3] + 1);
        *reinterpret_cast<longlong2*>(p.slots + r) = make_longlong2(slot[0], slot[1]);
        *reinterpret_cast<longlong2*>(p.slots + r + 2) = make_longlong2(slot[2], slot[3]);
      } else {
#pragma unroll
        for (int i = 0; i < kRowVec; ++i)
          if (i < cnt) {
            p.row_seq[r + i] = seq[i];
            p.row_pos[r + i] = pos[i];
            p.q_lens[r + i] = pos[i] + 1;
            p.slots[r + i] = slot[i];
          }
      }
    }
    __syncthreads();
  }
}

// New table entries and tiles of a call that asks for no rows.
__device__ void fill_without_rows(const Params& p, int64_t cursor, int64_t tid, int64_t step) {
  const int32_t* cu_blk = p.ws + 2;
  const int32_t* cu_tile = cu_blk + p.n_seqs + 1;
  if (p.free_list) {
    const int64_t n = cu_blk[p.n_seqs];
    for (int64_t j = tid; j < n; j += step) {
      const int b = find_seq(cu_blk, 0, p.n_seqs, static_cast<int32_t>(j));
      const int64_t have = ceil_div32(p.kv[b], p.page);
      p.table[b * p.table_stride + have + (j - cu_blk[b])] = p.free_list[cursor + j];
    }
  }
  if (p.tiles) {
    const int64_t n = cu_tile[p.n_seqs];
    for (int64_t t = tid; t < n; t += step) {
      const int b = find_seq(cu_tile, 0, p.n_seqs, static_cast<int32_t>(t));
      const int32_t at = static_cast<int32_t>(t - cu_tile[b]) * static_cast<int32_t>(p.rpt.d);
      p.tiles[3 * t + 0] = p.cu_rows[b] + at;
      p.tiles[3 * t + 1] = min(static_cast<int32_t>(p.rpt.d), p.nw[b] - at);
      p.tiles[3 * t + 2] = b;
    }
  }
}

// Neutral entries past the plan's own rows and tiles: no slot, no tokens, no rows.
__device__ __forceinline__ void pad_rest(const Params& p, int64_t rows, int64_t tiles, int64_t tid, int64_t step) {
  if (p.row_seq)
    for (int64_t r = rows + tid; r < p.n_rows; r += step) {
      p.row_seq[r] = 0;
      p.row_pos[r] = 0;
      p.q_lens[r] = 0;
      p.slots[r] = -1;
    }
  if (p.tiles)
    for (int64_t t = tiles + tid; t < p.n_tiles; t += step)
      p.tiles[3 * t] = p.tiles[3 * t + 1] = p.tiles[3 * t + 2] = 0;
}

// One CTA: checks and sums; ALONE: the rest of the plan as well (few outputs: a second launch costs
// more than one CTA's stores).
template <bool ALONE>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(const Params p) {
  __shared__ Sum3 s_warp[32];
  __shared__ int s_bad, s_ok;
  __shared__ int64_t s_cursor, s_rows, s_tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (threadIdx.x == 0) s_bad = 0;
  if (warp == 0) s_warp[lane] = Sum3{0, 0, 0};   // a block of fewer warps leaves the rest at zero
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  __syncthreads();
  int32_t* cu_blk = p.ws + 2;
  int32_t* cu_tile = cu_blk + p.n_seqs + 1;
  const int threads = blockDim.x;
  const int items = min(kScanItems, (p.n_seqs + threads - 1) / threads);   // consecutive sequences of a thread
  Sum3 base{0, 0, 0};
  for (int64_t b0 = 0; b0 < p.n_seqs; b0 += threads * items) {
    const int64_t b = b0 + static_cast<int64_t>(threadIdx.x) * items;
    int32_t kv[kScanItems], nw[kScanItems];
#pragma unroll
    for (int i = 0; i < kScanItems; ++i) {
      const bool is = i < items && b + i < p.n_seqs;
      kv[i] = is ? p.kv[b + i] : 0;
      nw[i] = is ? p.nw[b + i] : 0;
    }
    Sum3 v{0, 0, 0};
    int32_t blk[kScanItems], til[kScanItems];
#pragma unroll
    for (int i = 0; i < kScanItems; ++i) {
      blk[i] = til[i] = 0;
      if (i < items) {
        // both below 2^31, so their sum is below 2^32
        const uint32_t have = ceil_div32(kv[i], p.page), need = ceil_div32(static_cast<uint32_t>(kv[i]) + nw[i], p.page);
        if (kv[i] < 0 || nw[i] < 0 || need > static_cast<uint32_t>(p.width)) {
          s_bad = 1;
          nw[i] = 0;
        } else {
          blk[i] = need - have;
          if (p.tiled) til[i] = ceil_div32(nw[i], p.rpt);
        }
        v.r += nw[i];
        v.k += blk[i];
        v.t += til[i];
      }
    }
    const Sum3 incl = warp_scan(v, lane);
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      const Sum3 wi = warp_scan(s_warp[lane], lane);
      __syncwarp();
      s_warp[lane] = wi;
    }
    __syncthreads();
    Sum3 at{base.r + incl.r - v.r, base.k + incl.k - v.k, base.t + incl.t - v.t};
    if (warp > 0) {
      at.r += s_warp[warp - 1].r;
      at.k += s_warp[warp - 1].k;
      at.t += s_warp[warp - 1].t;
    }
#pragma unroll
    for (int i = 0; i < kScanItems; ++i) {
      if (i < items && b + i < p.n_seqs) {
        p.cu_rows[b + i] = static_cast<int32_t>(at.r);
        cu_blk[b + i] = static_cast<int32_t>(at.k);
        cu_tile[b + i] = static_cast<int32_t>(at.t);
      }
      at.r += nw[i];
      at.k += blk[i];
      at.t += til[i];
    }
    const Sum3 tot = s_warp[warps - 1];
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
    s_ok = !bad;
    s_cursor = cur;
    s_rows = bad ? 0 : base.r;
    s_tiles = bad ? 0 : base.t;
  }
  if constexpr (ALONE) {
    __syncthreads();
    if (p.pad) pad_rest(p, s_rows, s_tiles, threadIdx.x, blockDim.x);
    if (!s_ok) return;
    if (p.row_seq) fill_rows(p, s_cursor, 0, 1);
    else fill_without_rows(p, s_cursor, threadIdx.x, blockDim.x);
  }
}

__global__ void __launch_bounds__(kFillThreads) fill_kernel(const Params p) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  // all four at once: each is a trip to L2
  const int32_t ok = p.ws[0], cursor = p.ws[1];
  const int32_t rows = p.pad ? p.cu_rows[p.n_seqs] : 0;
  const int32_t tiles = p.pad ? p.ws[2 + 2 * static_cast<int64_t>(p.n_seqs) + 1] : 0;   // cu_tile[n_seqs]
  const int64_t tid = static_cast<int64_t>(blockIdx.x) * kFillThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kFillThreads;
  if (p.pad) pad_rest(p, ok ? rows : 0, ok ? tiles : 0, tid, step);
  if (!ok) return;
  if (p.row_seq)
    fill_rows(p, cursor, blockIdx.x, gridDim.x);
  else
    fill_without_rows(p, cursor, tid, step);
}

}  // namespace paging
}  // namespace dk
