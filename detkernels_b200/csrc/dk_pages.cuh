// Forking, compacting and freeing the pages of a KV cache, and moving the tokens that this takes.
//
// A request's tokens lie in the blocks table[b][0], table[b][1], ... of page tokens each.  The free blocks are a
// list with a cursor: what lies before it is handed out (the page plan takes from it), so blocks come back by
// writing them before the cursor and moving it down.  shares[x] counts the further holders of block x (0: one).
//
//   fork      row dst becomes a copy of row src: whole pages are shared (shares[x] += 1) and the open page gets a
//             block of its own, or every page does when there are no shares; the tokens of new blocks are copied.
//   compact   token kv + keep[j] becomes token kv + j, the rest behind kv is dropped; the pages that hold nothing any
//             more lose a holder, and those without one go back to the list in (sequence, page) order.  No token goes
//             to a page with further holders.
//
// Either is one kernel that checks everything, and only then changes the tables (fork_kernel, release_kernel), and
// one that moves tokens in all layers' pools (move_kernel).  The first is bound by the latency of a few dependent
// look-ups and barriers: one cluster of eight CTAs, a warp a run of consecutive sequences, whose flags and counts go
// into every CTA's shared memory, so that a barrier of the cluster is all that stands between two phases and no
// scratch has to be cleared.  The second is bound by the bytes it copies.
//
// Measured, both kernels, in a graph: 28 forks of 7 prompts that share their pages, 16 heads of 64 in 8 pools, 14.6 us
// (about 9 of them the first kernel); 24 copied whole, 1.2 GB, 200 us (6.1 TB/s); 256 accepted trees compacted, pages
// shared, 18.2 us (0.4 of them for the blocks and holders of moved tokens), 256 sequences freed 10.2; 8 caches of up
// to 16,000 tokens halved, 1.5 GB, 277 us (5.5 TB/s, half of the 256-byte rows skipped).
#pragma once

#include "dk_common.cuh"
#include "dk_divide.cuh"

namespace dk {
namespace pages {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;                 // one portable cluster
constexpr int kPlanWarps = kPlanCtas * (kPlanThreads / 32);
constexpr int kMoveThreads = 256;
constexpr int kMaxLanesLog = 5;              // of them, token lanes: at most 32 (long caches: 16 279 us, 32 276)
constexpr int kMaxPools = 128;               // pointers a launch takes

enum : int {
  kDetForkRows = 0x640,   // a source or destination outside the table, equal, or named twice
  kDetForkLens = 0x641,   // a length outside the table row
  kDetBlock = 0x642,      // a block id outside the pools
  kDetPool = 0x643,       // the free list is exhausted, or more comes back than was handed out
  kDetLens = 0x644,       // a negative length, more kept than held, or a sequence past its table row
  kDetKeep = 0x645,       // kept tokens that do not ascend inside the sequence
  kDetShares = 0x646,     // a page with fewer holders than give it back
  kDetShared = 0x647,     // a token to move into a page that another sequence holds, too
};

// Scratch, int32: [0] the plan stands, then two marks a table row (fork).
constexpr int kWsOk = 0, kWsMark = 16;

// What the CTAs of the cluster tell one another: by round, whether a CTA has found something wrong; a count a warp.
struct Told {
  int bad[4][kPlanCtas];
  int count[2][kPlanWarps];
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// Writes a word of CTA `rank`'s shared memory.
__device__ __forceinline__ void tell(int* mine, int rank, int v) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
// A barrier of the cluster, with this warp's count for all (slot 0 or 1), that says whether any thread had `bad`.
__device__ __forceinline__ bool cluster_any(Told& told, int round, bool bad, int slot, int count) {
  const int lane = threadIdx.x & 31, w = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5);
  if (lane < kPlanCtas) tell(&told.count[slot][w], lane, count);
  const int mine = __syncthreads_or(bad);
  if (threadIdx.x < kPlanCtas) tell(&told.bad[round][blockIdx.x], threadIdx.x, mine);
  cluster_sync();
  int any = 0;
#pragma unroll
  for (int c = 0; c < kPlanCtas; ++c) any |= told.bad[round][c];
  return any != 0;
}

// What the warps before this one counted, and what all did.
__device__ __forceinline__ void warp_prefix(const int (&count)[kPlanWarps], int w, int lane, int64_t& before, int64_t& total) {
  int64_t b = 0, t = 0;
#pragma unroll
  for (int i = 0; i < kPlanWarps / 32; ++i) {
    const int64_t c = count[i * 32 + lane];
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
  __shared__ Told told;
  cluster_arrive();   // this CTA has begun
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int w = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5);
  const int per = (p.n + kPlanWarps - 1) / kPlanWarps;
  const int i0 = min(static_cast<int64_t>(p.n), static_cast<int64_t>(w) * per), i1 = min(p.n, i0 + per);
  // A row's marks: a fork that it is the source of, and one that it is the destination of.  They are never cleared: what
  // a mark names is looked up.
  int32_t *as_src = p.ws + kWsMark, *as_dst = as_src + p.rows;
  const int64_t cursor = *p.cursor_in;
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
    __stcg(as_src + s, i);
    __stcg(as_dst + d, i);
    const int n = p.kv[s];
    if (n < 0 || ceil_div32(n, p.page) > static_cast<uint32_t>(p.width)) {
      report_error(DK_ERR_DEVICE_CHECK, kDetForkLens);
      bad = true;
      continue;
    }
    const uint32_t whole = div_by(n, p.page);
    need += (p.shares ? 0 : whole) + (n != static_cast<int>(whole * p.page.d));
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) need += __shfl_xor_sync(0xffffffffu, need, d);
  cluster_wait();     // all have begun
  bad = cluster_any(told, 0, bad, 0, static_cast<int>(need < 0x7fffffff ? need : 0x7fffffff));
  int64_t at = 0, total = 0;
  if (!bad) {
    warp_prefix(told.count[0], w, lane, at, total);
    at += cursor;
    if (cursor < 0 || cursor + total > p.n_free) {
      if (w == 0 && lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetPool);
      bad = true;
    }
    // each destination is one fork's, and no source; all blocks are of the pool
    int64_t a = at;
    for (int i = i0; i < i1 && !bad; ++i) {
      const int s = p.src[i], d = p.dst[i], n = p.kv[s], np = ceil_div32(n, p.page), whole = div_by(n, p.page);
      const int kept = p.shares ? whole : 0;
      bool wrong = false;
      for (int j = lane; j < np; j += 32) {
        const int x = p.table[s * p.table_stride + j];
        const int y = j < kept ? 0 : p.free_list[a + j - kept];
        wrong |= x < 0 || x >= p.n_blocks || y < 0 || y >= p.n_blocks;
      }
      if (wrong) report_error(DK_ERR_DEVICE_CHECK, kDetBlock);
      const int named = __ldcg(as_src + d);
      if (__ldcg(as_dst + d) != i || (named >= 0 && named < p.n && p.src[named] == d)) {
        if (lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetForkRows);
        wrong = true;
      }
      bad = __any_sync(0xffffffffu, wrong);
      a += np - kept;
    }
  }
  bad = cluster_any(told, 1, bad, 1, 0);
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
  int moves;               // move_kernel follows: the blocks of the tokens that it moves are checked here
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

// Entries of a row of `keep` that a warp checks at a time, all loaded at once: a few long rows are shared by many warps.
// A token that moves has the blocks that it comes from and goes to looked up as well: nothing may be found wrong once
// lengths, holders and the free list have changed.  No token may go to a block with further holders, who would find it
// among theirs; so none that is read is another sequence's to write, either.  (A holder that gives the block up in the
// same call counts: it may read its own kept tokens there.)
constexpr int kKeepLoads = 8, kKeepRun = 32 * kKeepLoads;

__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) release_kernel(const ReleaseParams p) {
  __shared__ Told told;
  cluster_arrive();   // this CTA has begun
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int w = blockIdx.x * (kPlanThreads / 32) + (threadIdx.x >> 5);
  const int per = (p.n + kPlanWarps - 1) / kPlanWarps;
  const int b0 = min(static_cast<int64_t>(p.n), static_cast<int64_t>(w) * per), b1 = min(p.n, b0 + per);
  const bool back = p.free_list != nullptr;
  const int64_t cursor = back ? *p.cursor_in : 0;
  bool bad = false;
  int64_t given = 0;   // pages of this warp's sequences that come back
  auto first_page = [&](int b) { return static_cast<int>(ceil_div32(p.kv[b] + p.n_keep[b], p.page)); };
  auto last_page = [&](int b) { return static_cast<int>(ceil_div32(p.kv[b] + p.nw[b], p.page)); };
  auto bad_lens = [&](int64_t kv, int64_t nw, int64_t nk) {
    return kv < 0 || nw < 0 || nk < 0 || nk > nw || kv + nw > 0x7fffffff || (p.keep && nk > p.keep_width) ||
           ceil_div32(static_cast<uint32_t>(kv + nw), p.page) > static_cast<uint32_t>(p.width);
  };
  auto block_at = [&](int b, int tok) { return p.table[b * p.table_stride + div_by(static_cast<uint32_t>(tok), p.page)]; };
  auto there = [&](int x) { return x >= 0 && x < p.n_blocks; };
  if (p.keep) {
    const int runs = (p.keep_width + kKeepRun - 1) / kKeepRun;
    for (int64_t e = w; e < static_cast<int64_t>(p.n) * runs; e += kPlanWarps) {
      const int b = static_cast<int>(e / runs);
      const int64_t j0 = (e - static_cast<int64_t>(b) * runs) * kKeepRun;
      const int kv = p.kv[b], nw = p.nw[b], nk = p.n_keep[b];
      if (bad_lens(kv, nw, nk)) continue;   // refused below
      const int32_t* row = p.keep + b * p.keep_stride;
      int k[kKeepLoads];
#pragma unroll
      for (int i = 0; i < kKeepLoads; ++i) k[i] = j0 + 32 * i + lane < nk ? row[j0 + 32 * i + lane] : 0x7fffffff;
      int last = lane == 31 && j0 > 0 && j0 < nk ? row[j0 - 1] : -1;   // lane 31: the entry before the next 32
      bool wrong = false, lost = false, shared = false;
#pragma unroll
      for (int i = 0; i < kKeepLoads; ++i) {
        const int before = __shfl_sync(0xffffffffu, lane == 31 ? last : k[i], (lane + 31) & 31);
        const int64_t j = j0 + 32 * i + lane;
        if (j < nk) {
          const bool in = k[i] >= 0 && k[i] < nw;
          wrong |= !in || before >= k[i];
          if (p.moves && in && k[i] != j) {
            const int to = block_at(b, kv + static_cast<int>(j));
            lost |= !there(block_at(b, kv + k[i])) || !there(to);
            shared |= p.shares && there(to) && p.shares[to] > 0;
          }
        }
        last = k[i];
      }
      if (wrong || lost || shared) {
        report_error(DK_ERR_DEVICE_CHECK, wrong ? kDetKeep : lost ? kDetBlock : kDetShared);
        bad = true;
      }
    }
  }
  for (int b = b0; b < b1; ++b) {
    if (bad_lens(p.kv[b], p.nw[b], p.n_keep[b])) {
      if (lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetLens);
      bad = true;
      continue;
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
  cluster_wait();     // all have begun
  // Without shares every page comes back, and that is known here already.
  bad = cluster_any(told, 0, bad, 0, static_cast<int>(given < 0x7fffffff ? given : 0x7fffffff));
  auto each_page = [&](auto&& f) {   // (sequence, column, block) of the warp's pages, a lane each; all lanes call f
    for (int b = b0; b < b1; ++b) {
      const int lo = first_page(b), hi = last_page(b);
      for (int j0 = lo; j0 < hi; j0 += 32) {
        const int j = j0 + lane;
        f(b, j, j < hi ? p.table[b * p.table_stride + j] : -1);
      }
    }
  };
  // The page's place in the order of all, as a number below any that a count of holders falls to.
  constexpr int kClaim = -(1 << 30);
  auto code = [&](int b, int j) { return kClaim - (b * p.width + j); };
  int64_t at = 0, total = 0;
  if (back && !bad) {
    if (p.shares) {
      // one holder less a page ...
      each_page([&](int, int, int x) { if (x >= 0) atomicSub(&p.shares[x], 1); });
      cluster_sync();
      // ... and where none is left, the last of those that gave it up hands it back
      bool over = false;
      each_page([&](int b, int j, int x) {
        if (x < 0) return;
        const int v = __ldcg(p.shares + x);
        if (v == -1 || v <= kClaim) atomicMin(&p.shares[x], code(b, j));
        else if (v < -1) over = true;
      });
      if (over) report_error(DK_ERR_DEVICE_CHECK, kDetShares);
      bad = cluster_any(told, 1, over, 1, 0);
      given = 0;
      each_page([&](int b, int j, int x) { given += x >= 0 && __ldcg(p.shares + x) == code(b, j); });
#pragma unroll
      for (int d = 16; d; d >>= 1) given += __shfl_xor_sync(0xffffffffu, given, d);
      cluster_any(told, 2, false, 0, static_cast<int>(given));
    }
    if (!bad) {
      warp_prefix(told.count[0], w, lane, at, total);
      if (total > cursor || cursor > p.n_free) {
        if (w == 0 && lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetPool);
        bad = true;   // the same for every thread
      }
    }
    if (bad && p.shares) {   // the claims go, then the holders come back
      each_page([&](int b, int j, int x) {
        if (x >= 0 && __ldcg(p.shares + x) == code(b, j)) __stcg(p.shares + x, -1);
      });
      cluster_sync();
      each_page([&](int, int, int x) { if (x >= 0) atomicAdd(&p.shares[x], 1); });
    }
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
  int32_t keep_width, width;   // width: entries of a table row
  int32_t sorted;          // compact: so many sequences, the longest first; 0: any number in their order
  int32_t cols_log;        // log2 of the columns a CTA takes at once; the other threads are token lanes
  int32_t col_groups, splits;
  const int32_t* ws;
};

// A CTA takes 2^cols_log columns (16-byte vectors of a head of a pool, side by side in memory inside a head) and walks
// the tokens, (threads / columns) * U at a time: their places first, into shared memory, then all loads, then all
// stores.  Compacting in place needs no more order than that: a token moves down or not at all, so what one step
// writes lies below everything that a later step reads, and inside a step the barrier parts loads from stores.
// FORK: the destinations' rows are fork_kernel's, so nothing is read before it has ended.  A compaction reads its first
// tokens while release_kernel still runs, which has itself waited for whatever wrote them, and changes none of what is
// read here; it stores once that has said that all is well.
// (Loads of the next step before the stores of this one: 279 against 286 us on the long caches, but 20 against 18 on the
// accepted trees; four CTAs an SM instead of three, in 64 registers: 330 on the long ones.)
template <typename V, int U, bool FORK>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveParams p) {
  __shared__ int64_t s_from[U << kMaxLanesLog], s_to[U << kMaxLanesLog];
  if (FORK) {
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    if (__ldcg(p.ws + kWsOk) == 0) return;
  }
  const uint32_t group = blockIdx.x % p.col_groups, rest = blockIdx.x / p.col_groups;
  const uint32_t split = rest % p.splits;
  uint32_t i = rest / p.splits;
  if (!FORK && p.sorted > 0) {   // the sequence with that many longer ones, by a lane a sequence
    const int lane = threadIdx.x & 31, mine = lane < p.sorted ? p.n_keep[lane] : 0;
    int longer = 0;
    for (int q = 0; q < p.sorted; ++q) {
      const int other = __shfl_sync(0xffffffffu, mine, q);
      longer += other > mine || (other == mine && q < lane);
    }
    i = __ffs(__ballot_sync(0xffffffffu, lane < p.sorted && longer == static_cast<int>(i))) - 1;
  }
  const int cols = 1 << p.cols_log, lanes = kMoveThreads >> p.cols_log, step = lanes * U;
  const int32_t *row_from, *row_to, *keep = nullptr;
  int base, count;
  if (FORK) {
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
    // (what release_kernel refuses is not looked up out of bounds either, here and below)
    if (base < 0 || count < 0 || count > p.keep_width) base = count = 0;
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
  bool waited = FORK;
  for (int64_t t0 = begin; t0 < end; t0 += step) {
    for (int e = threadIdx.x; e < step; e += kMoveThreads) {
      const int64_t j = t0 + e;
      int64_t from = -1, to = -1;
      if (j < end) {
        const int64_t tf = base + static_cast<int64_t>(FORK ? j : keep[j]), tt = base + j;
        if (FORK || tf != tt) {
          const uint32_t pf = div_by(static_cast<uint32_t>(tf), p.page), pt = div_by(static_cast<uint32_t>(tt), p.page);
          const bool in = tf >= 0 && tf <= 0x7fffffff && tt <= 0x7fffffff && pf < static_cast<uint32_t>(p.width) &&
                          pt < static_cast<uint32_t>(p.width);
          const int bf = in ? row_from[pf] : -1, bt = in ? row_to[pt] : -1;
          if (bf >= 0 && bf < p.n_blocks && bt >= 0 && bt < p.n_blocks) {
            from = bf * p.s_block + (tf - static_cast<int64_t>(pf) * p.page.d) * p.s_tok;
            to = bt * p.s_block + (tt - static_cast<int64_t>(pt) * p.page.d) * p.s_tok;
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
    if (!waited) {
      pdl_wait();
      if (threadIdx.x == 0) pdl_launch_dependents();
      if (__ldcg(p.ws + kWsOk) == 0) return;
      waited = true;
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
  if (!waited) pdl_wait();   // a kernel's end means the end of all before it
}

}  // namespace pages
}  // namespace dk
