// Forking, compacting and freeing the pages of a KV cache, and moving the tokens that this takes.
//
// A request's tokens lie in the blocks table[b][0], table[b][1], ... of page tokens each.  The free blocks are a
// list with a cursor: what lies before it is handed out (the page plan takes from it), so blocks come back by
// writing them before the cursor and moving it down.  shares[x] counts the further holders of block x (0: one).
//
//   fork      row dst becomes a copy of row src: whole pages are shared (shares[x] += 1) and the open page gets a
//             block of its own, or every page does when there are no shares; the tokens of new blocks are copied.
//   compact   token kv + keep[j] becomes token kv + j, the rest behind kv is dropped; the pages that hold nothing any
//             more lose a holder, and those without one go back to the list in (sequence, page) order.
//
// Either is one kernel that checks everything, and only then changes the tables (fork_kernel, release_kernel), and
// one that moves tokens in all layers' pools (move_kernel).  The first is bound by the latency of a few dependent
// look-ups and barriers: one cluster of eight CTAs, whose barrier needs no memory that anybody has to clear, a warp
// a run of consecutive sequences.  The second is bound by the bytes it copies.
#pragma once

#include "dk_common.cuh"
#include "dk_divide.cuh"

namespace dk {
namespace pages {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;                 // one portable cluster
constexpr int kPlanWarps = kPlanCtas * (kPlanThreads / 32);
constexpr int kMoveThreads = 256;
constexpr int kMaxPools = 128;               // pointers a launch takes

enum : int {
  kDetForkRows = 0x640,   // a source or destination outside the table, equal, or named twice
  kDetForkLens = 0x641,   // a length outside the table row
  kDetBlock = 0x642,      // a block id outside the pools
  kDetPool = 0x643,       // the free list is exhausted, or more comes back than was handed out
  kDetLens = 0x644,       // a negative length, more kept than held, or a sequence past its table row
  kDetKeep = 0x645,       // kept tokens that do not ascend inside the sequence
  kDetShares = 0x646,     // a page with fewer holders than give it back
};

// Scratch, int32: [0] the plan stands, [1 .. 8] a flag a CTA, [16 ..] a count a warp, then a mark a table row (fork).
constexpr int kWsOk = 0, kWsBad = 1, kWsCount = 16, kWsMark = kWsCount + kPlanWarps;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A barrier of the cluster that says whether any thread had `bad`; `round` alternates between calls that follow one
// another (a CTA may still read one round's flags while another writes the next's).
__device__ __forceinline__ bool cluster_any(bool bad, int32_t* flags) {
  const int mine = __syncthreads_or(bad);
  if (threadIdx.x == 0) __stcg(flags + blockIdx.x, mine);
  cluster_sync();
  int any = 0;
#pragma unroll
  for (int c = 0; c < kPlanCtas; ++c) any |= __ldcg(flags + c);
  cluster_sync();   // everyone has read them
  return any != 0;
}

// What the warps before this one counted, and what all did (after a cluster barrier).
__device__ __forceinline__ void warp_prefix(const int32_t* count, int w, int lane, int64_t& before, int64_t& total) {
  int64_t b = 0, t = 0;
#pragma unroll
  for (int i = 0; i < kPlanWarps / 32; ++i) {
    const int64_t c = __ldcg(count + i * 32 + lane);
    t += c;
    if (i * 32 + lane < w) b += c;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    b += __shfl_xor_sync(0xffffffffu, b, d);
    t += __shfl_xor_sync(0xffffffffu, t, d);
  }
  before = b;
  total = t;
}

struct ForkParams {
  int32_t* table;
  int64_t table_stride;
  int32_t rows, width;
  int32_t* kv;
  const int32_t* src;
  const int32_t* dst;
  int32_t n;
  Divisor page;
  const int32_t* free_list;
  int64_t n_free;
  const int32_t* cursor_in;
  int32_t* cursor_out;
  int32_t* shares;        // null: every page is copied
  int64_t n_blocks;
  int32_t* ws;
};

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) fork_kernel(const ForkParams p) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int w = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5);
  const int per = (p.n + kPlanWarps - 1) / kPlanWarps;
  const int i0 = min(static_cast<int64_t>(p.n), static_cast<int64_t>(w) * per), i1 = min(p.n, i0 + per);
  int32_t* mark = p.ws + kWsMark;
  const uint32_t page = p.page.d;
  for (int64_t r = blockIdx.x * kPlanThreads + threadIdx.x; r < p.rows; r += kPlanCtas * kPlanThreads) mark[r] = 0;
  cluster_sync();
  // rows and lengths; what the new pages are
  bool bad = false;
  int64_t need = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const int s = p.src[i], d = p.dst[i];
    if (s < 0 || s >= p.rows || d < 0 || d >= p.rows || s == d) {
      report_error(DK_ERR_DEVICE_CHECK, kDetForkRows);
      bad = true;
      continue;
    }
    atomicOr(&mark[s], 1);
    if (atomicOr(&mark[d], 2) & 2) {
      report_error(DK_ERR_DEVICE_CHECK, kDetForkRows);
      bad = true;
    }
    const int n = p.kv[s];
    if (n < 0 || ceil_div32(n, p.page) > static_cast<uint32_t>(p.width)) {
      report_error(DK_ERR_DEVICE_CHECK, kDetForkLens);
      bad = true;
      continue;
    }
    const uint32_t whole = div_by(n, p.page);
    need += (p.shares ? 0 : whole) + (n != static_cast<int>(whole * page));
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) need += __shfl_xor_sync(0xffffffffu, need, d);
  // beyond 2^31 blocks no list holds them: the sum of the warps' counts stays inside 64 bits and is refused
  if (lane == 0) __stcg(p.ws + kWsCount + w, static_cast<int32_t>(need < 0x7fffffff ? need : 0x7fffffff));
  bad = cluster_any(bad, p.ws + kWsBad);
  int64_t at = 0, total = 0;
  const int64_t cursor = *p.cursor_in;
  if (!bad) {
    warp_prefix(p.ws + kWsCount, w, lane, at, total);
    at += cursor;
    if (cursor < 0 || cursor + total > p.n_free) {
      if (w == 0 && lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetPool);
      bad = true;
    }
    // no destination is a source, and all blocks are of the pool
    int64_t a = at;
    for (int i = i0; i < i1 && !bad; ++i) {
      const int s = p.src[i], n = p.kv[s], np = ceil_div32(n, p.page), whole = div_by(n, p.page);
      const int kept = p.shares ? whole : 0;
      bool wrong = false;
      for (int j = lane; j < np; j += 32) {
        const int x = p.table[s * p.table_stride + j];
        const int y = j < kept ? 0 : p.free_list[a + j - kept];
        wrong |= x < 0 || x >= p.n_blocks || y < 0 || y >= p.n_blocks;
      }
      if (wrong) report_error(DK_ERR_DEVICE_CHECK, kDetBlock);
      if (__ldcg(mark + p.dst[i]) & 1) {
        if (lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetForkRows);
        wrong = true;
      }
      bad = __any_sync(0xffffffffu, wrong);
      a += np - kept;
    }
  }
  bad = cluster_any(bad, p.ws + kWsBad);
  if (w == 0 && lane == 0) {
    p.ws[kWsOk] = bad ? 0 : 1;
    *p.cursor_out = static_cast<int32_t>(bad ? cursor : cursor + total);
  }
  if (bad) return;
  for (int i = i0; i < i1; ++i) {
    const int s = p.src[i], d = p.dst[i], n = p.kv[s], np = ceil_div32(n, p.page), whole = div_by(n, p.page);
    const int kept = p.shares ? whole : 0;
    for (int j = lane; j < np; j += 32) {
      int x;
      if (j < kept) {
        x = p.table[s * p.table_stride + j];
        atomicAdd(&p.shares[x], 1);
      } else {
        x = p.free_list[at + j - kept];
      }
      p.table[d * p.table_stride + j] = x;
    }
    at += np - kept;
    if (lane == 0) p.kv[d] = n;
  }
}

struct ReleaseParams {
  const int32_t* table;
  int64_t table_stride;
  int32_t width;
  const int32_t* kv;       // tokens that stay whatever is kept
  const int32_t* nw;       // tokens behind them
  const int32_t* n_keep;   // of those, how many stay
  const int32_t* keep;     // which, ascending; null: the first n_keep
  int64_t keep_stride;
  int32_t keep_width;
  int32_t n;
  Divisor page;
  int32_t* lens_out;
  int32_t* free_list;      // null: no page comes back
  int64_t n_free;
  const int32_t* cursor_in;
  int32_t* cursor_out;
  int32_t* shares;         // null: every page has one holder
  int64_t n_blocks;
  int32_t* ws;
};

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) release_kernel(const ReleaseParams p) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int w = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5);
  const int per = (p.n + kPlanWarps - 1) / kPlanWarps;
  const int b0 = min(static_cast<int64_t>(p.n), static_cast<int64_t>(w) * per), b1 = min(p.n, b0 + per);
  int32_t* flags = p.ws + kWsBad;
  const bool back = p.free_list != nullptr;
  bool bad = false;
  int64_t given = 0;   // pages of this warp's sequences that come back
  auto first_page = [&](int b) { return static_cast<int>(ceil_div32(p.kv[b] + p.n_keep[b], p.page)); };
  auto last_page = [&](int b) { return static_cast<int>(ceil_div32(p.kv[b] + p.nw[b], p.page)); };
  for (int b = b0; b < b1; ++b) {
    const int64_t kv = p.kv[b], nw = p.nw[b], nk = p.n_keep[b];
    if (kv < 0 || nw < 0 || nk < 0 || nk > nw || kv + nw > 0x7fffffff || (p.keep && nk > p.keep_width) ||
        ceil_div32(static_cast<uint32_t>(kv + nw), p.page) > static_cast<uint32_t>(p.width)) {
      if (lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetLens);
      bad = true;
      continue;
    }
    if (p.keep) {
      const int32_t* row = p.keep + b * p.keep_stride;
      bool wrong = false;
      for (int64_t j = lane; j < nk; j += 32) {
        const int k = row[j];
        wrong |= k < 0 || k >= nw || (j > 0 && row[j - 1] >= k);
      }
      if (wrong) {
        report_error(DK_ERR_DEVICE_CHECK, kDetKeep);
        bad = true;
      }
    }
    if (back) {
      const int lo = first_page(b), hi = last_page(b);
      bool wrong = false;
      for (int j = lo + lane; j < hi; j += 32) {
        const int x = p.table[b * p.table_stride + j];
        wrong |= x < 0 || x >= p.n_blocks;
      }
      if (wrong) {
        report_error(DK_ERR_DEVICE_CHECK, kDetBlock);
        bad = true;
      }
      given += max(0, hi - lo);
    }
  }
  const int64_t cursor = back ? *p.cursor_in : 0;
  // Without shares every page comes back, and that is known here already.
  if (lane == 0) __stcg(p.ws + kWsCount + w, static_cast<int32_t>(given < 0x7fffffff ? given : 0x7fffffff));
  bad = cluster_any(bad, flags);
  auto each_page = [&](auto&& f) {   // (sequence, column, block) of the warp's pages, a lane each; all lanes call f
    for (int b = b0; b < b1; ++b) {
      const int lo = first_page(b), hi = last_page(b);
      for (int j0 = lo; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        f(b, j, j < hi ? p.table[b * p.table_stride + j] : -1);
      }
    }
  };
  // The page's place in the order of all, as a negative number that no count of holders is.
  auto code = [&](int b, int j) { return -2 - (b * p.width + j); };
  int64_t at = 0, total = 0;
  if (back && !bad) {
    if (p.shares) {
      // one holder less a page ...
      each_page([&](int, int, int x) { if (x >= 0) atomicSub(&p.shares[x], 1); });
      cluster_sync();
      bool over = false;
      each_page([&](int, int, int x) { if (x >= 0) over |= __ldcg(p.shares + x) < -1; });
      if (over) report_error(DK_ERR_DEVICE_CHECK, kDetShares);
      bad = cluster_any(over, flags);
      if (!bad) {
        // ... and where none is left, the last of those that gave it up hands it back
        each_page([&](int b, int j, int x) {
          if (x >= 0 && __ldcg(p.shares + x) < 0) atomicMin(&p.shares[x], code(b, j));
        });
        cluster_sync();
        given = 0;
        each_page([&](int b, int j, int x) { given += x >= 0 && __ldcg(p.shares + x) == code(b, j); });
#pragma unroll
        for (int d = 16; d; d >>= 1) given += __shfl_xor_sync(0xffffffffu, given, d);
        if (lane == 0) __stcg(p.ws + kWsCount + w, static_cast<int32_t>(given));
        cluster_sync();
      }
    }
    if (!bad) {
      warp_prefix(p.ws + kWsCount, w, lane, at, total);
      if (total > cursor || cursor > p.n_free) {
        if (w == 0 && lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetPool);
        bad = true;   // the same for every thread
        if (p.shares) {   // the claims go, then the holders come back
          each_page([&](int b, int j, int x) {
            if (x >= 0 && __ldcg(p.shares + x) == code(b, j)) __stcg(p.shares + x, -1);
          });
          cluster_sync();
        }
      }
    }
    if (bad && p.shares) each_page([&](int, int, int x) { if (x >= 0) atomicAdd(&p.shares[x], 1); });
  }
  if (w == 0 && lane == 0) {
    p.ws[kWsOk] = bad ? 0 : 1;
    if (back) *p.cursor_out = static_cast<int32_t>(bad ? cursor : cursor - total);
  }
  if (!bad && back) {
    at += cursor - total;
    each_page([&](int b, int j, int x) {
      const bool mine = x >= 0 && (!p.shares || __ldcg(p.shares + x) == code(b, j));
      const uint32_t who = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        p.free_list[at + __popc(who & ((1u << lane) - 1))] = x;
        if (p.shares) __stcg(p.shares + x, 0);
      }
      at += __popc(who);
    });
  }
  for (int b = b0 + lane; b < b1; b += 32) p.lens_out[b] = p.kv[b] + (bad ? 0 : p.n_keep[b]);
}

// Tokens moved inside the pools.  Fork: tokens [first, n) of row src to the same places of row dst, n = kv[dst],
// first the first token of a new block.  Compact: token kv + keep[j] of a row to kv + j of the same row.
struct MoveParams {
  void* pool[kMaxPools];
  int32_t n_cols;          // pools * heads * vectors a head
  int32_t heads, vecs;     // of a pool; of a head
  int64_t s_block, s_head, s_tok;   // strides in vectors
  const int32_t* table;
  int64_t table_stride;
  Divisor page;
  int64_t n_blocks;
  const int32_t* kv;
  const int32_t* src;      // fork
  const int32_t* dst;
  int all;                 // fork: every page is copied
  const int32_t* n_keep;   // compact
  const int32_t* keep;
  int64_t keep_stride;
  int32_t cols_log;        // log2 of the columns a CTA takes at once; the other threads are token lanes
  int32_t col_groups, splits;
  const int32_t* ws;
};

// A CTA takes 2^cols_log columns (16-byte vectors of a head of a pool, side by side in memory inside a head) and walks
// the tokens, (threads / columns) * U at a time: their places first, into shared memory, then all loads, then all
// stores.  Compacting in place needs no more order than that: a token moves down or not at all, so what one step
// writes lies below everything that a later step reads, and inside a step the barrier parts loads from stores.
template <typename V, int U>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveParams p) {
  __shared__ int64_t s_from[kMoveThreads * U], s_to[kMoveThreads * U];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  if (__ldcg(p.ws + kWsOk) == 0) return;
  const uint32_t group = blockIdx.x % p.col_groups, rest = blockIdx.x / p.col_groups;
  const uint32_t split = rest % p.splits, i = rest / p.splits;
  const int cols = 1 << p.cols_log, lanes = kMoveThreads >> p.cols_log, step = lanes * U;
  const int32_t *row_from, *row_to, *keep = nullptr;
  int base, count;
  if (p.src) {
    const int s = p.src[i], d = p.dst[i], n = p.kv[s];
    row_from = p.table + s * p.table_stride;
    row_to = p.table + d * p.table_stride;
    base = p.all ? 0 : static_cast<int>(div_by(n, p.page) * p.page.d);
    count = n - base;
  } else {
    row_from = row_to = p.table + i * p.table_stride;
    base = p.kv[i];
    count = p.n_keep[i];
    keep = p.keep + i * p.keep_stride;
  }
  // this CTA's share of the tokens, in whole steps (a compaction has one share)
  const int64_t per = ((count + static_cast<int64_t>(step) * p.splits - 1) / (static_cast<int64_t>(step) * p.splits)) * step;
  const int64_t begin = split * per, end = begin + per < count ? begin + per : count;
  const int col = static_cast<int>(group) * cols + (threadIdx.x & (cols - 1));
  const int tl = threadIdx.x >> p.cols_log;
  V* at = nullptr;
  if (col < p.n_cols) {
    const int v = col % p.vecs, hp = col / p.vecs, h = hp % p.heads, pool = hp / p.heads;
    at = static_cast<V*>(p.pool[pool]) + h * p.s_head + v;
  }
  for (int64_t t0 = begin; t0 < end; t0 += step) {
    for (int e = threadIdx.x; e < step; e += kMoveThreads) {
      const int64_t j = t0 + e;
      int64_t from = -1, to = -1;
      if (j < end) {
        const int tf = base + static_cast<int>(keep ? keep[j] : j), tt = base + static_cast<int>(j);
        if (row_from != row_to || tf != tt) {
          const uint32_t pf = div_by(tf, p.page), pt = div_by(tt, p.page);
          const int bf = row_from[pf], bt = row_to[pt];
          if (bf < 0 || bf >= p.n_blocks || bt < 0 || bt >= p.n_blocks) {
            report_error(DK_ERR_DEVICE_CHECK, kDetBlock);
          } else {
            from = bf * p.s_block + (tf - static_cast<int>(pf * p.page.d)) * p.s_tok;
            to = bt * p.s_block + (tt - static_cast<int>(pt * p.page.d)) * p.s_tok;
          }
        }
      }
      s_from[e] = from;
      s_to[e] = to;
    }
    __syncthreads();
    V v[U];
    if (at) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t f = s_from[u * lanes + tl];
        if (f >= 0) v[u] = at[f];
      }
    }
    __syncthreads();   // all of the step's tokens are read
    if (at) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t t = s_to[u * lanes + tl];
        if (t >= 0) at[t] = v[u];
      }
    }
    __syncthreads();   // the places are free for the next step
  }
}

}  // namespace pages
}  // namespace dk
