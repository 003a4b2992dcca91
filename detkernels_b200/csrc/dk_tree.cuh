// Attention of drafted tokens: the rows of a sequence are the nodes of a tree (or any other set) of drafts whose keys
// and values lie behind the sequence's kv cached tokens; a row sees all of those, and of the drafts the ones that its
// mask names.
//
// The query heads of all of a sequence's rows on KV head h are the rows of one matrix Q [t G, D], so that the cache is
// read once for the whole tree: S = Q K^T scale, out = softmax(S + mask) V.  Fixed reduction structure (the definition of
// a row's bits): the sequence's tokens are cut into chunks whose size follows kv only (chunk_tokens), a
// chunk's softmax state (m, l, O) is formed block by block as in dk_prefix.cuh, and the chunks' states are joined in
// order.  No step looks at another row: a chunk of which a row sees nothing joins with weight 0.
//
// Work: an item is (sequence, up to two tiles of at most 128 rows, chunk): two tiles of one KV head, which then share K
// and V, or, where the rows fit one tile, the tiles of two KV heads, each with its own K and V.  Either way both softmax
// warpgroups have work, and take turns on the exponential unit (and where all single tiles find an SM, an item is one).  One persistent CTA an SM takes items in an order that
// plan_kernel has made of the lengths, the most expensive first, so that the CTAs end together; several pairs of tiles of a
// KV head come side by side, and find a chunk's keys in L2.  A TMA warp, an MMA warp a tile (scores, weights and
// accumulator apart in TMEM), a warpgroup a tile for the softmax, a row a thread, and a warp that fetches the queries and
// makes the values of draft blocks safe: 0 weights must meet neither what lies behind the sequence in its last page nor a non-finite value of a draft that
// some rows do not see.  Those elements become 0 in shared memory, and rows that do see them have them added back from the
// cache (which no ordinary call does).
//
// Measured, all kernels, in a graph: 64 requests of 8 to 32 drafts behind 200 to 4000 tokens, 32 heads of 128 on 8, bf16,
// 131 us (4.4 TB/s of keys, values and queries; floor 89); 9 of 40 to 64 drafts behind 8000 to 20,000 tokens, 32 heads of
// 128 on 4, f16, 168 us (750 TFLOP/s; floor 78 by its products); 4 of up to 6 behind up to 700, 8 heads of 64, 12 us.  Bound by a
// block's chain from its scores to its weights (two tiles in turn: tensor pipe 47 % and exponential unit 45 % busy on the
// long ones), the states of the chunks (out of the way in L2, then joined) and the last items.  In sustained runs the power
// cap lowers the clocks: 148 and 196 us.
#pragma once

#include "dk_common.cuh"
#include "dk_divide.cuh"
#include "dk_prefix.cuh"

namespace dk {
namespace tree {

using own::exp2_hw;
using own::join;
using own::join4;
using own::join_weights;
using own::pack2;
using prefix::add2;
using prefix::fma2;
using prefix::kRows;
using prefix::kSoftWarps;
using prefix::warp_wait;

constexpr int kThreads = prefix::kThreads;   // softmax warps, then TMA, two for MMA, and one for queries and draft values

enum : int {
  kDetEmpty = 0x670,
  kDetFull = 0x671,
  kDetScores = 0x672,
  kDetProbs = 0x673,
  kDetOut = 0x674,
  kDetQ = 0x675,
  kDetOutFree = 0x676,
  kDetQFree = 0x66f,
  kDetDrain = 0x677,
  kDetDone = 0x678,
  kDetScoresFree = 0x679,
  kDetPage = 0x67a,   // a block id outside the pool
  kDetTurn = 0x67b,
  kDetRaw = 0x67c,
  kDetLens = 0x67d,   // a negative length, rows that do not ascend or exceed their bound, or tokens beyond the cache
};

struct Maps {
  CUtensorMap q;            // (d, head, row): boxes of 64 elements of a tile's heads and rows
  CUtensorMap k, v;         // (d, token, KV head, sequence or block): boxes of 64 elements x 64 tokens
};

struct Params {
  int32_t hkv, G;
  int32_t rpt;              // rows a tile: its query rows are rpt G
  Divisor31 group;          // by G
  int32_t n_seqs, n_rows, max_rows;
  const int32_t* kv_lens;
  const int32_t* cu_rows;
  const uint64_t* mask;     // [n_rows][words]
  int64_t mask_stride;
  int32_t words;
  int32_t capacity;         // tokens a sequence may have, drafts included
  int32_t units;            // items a (sequence, chunk), at most
  int solo;                 // an item has one tile
  int32_t max_chunks;
  int32_t* plan;            // the items' order; null: CTA c takes item c of (chunk, sequence, unit)
  const void* v;            // for what is added back
  int64_t c_sn, c_sh, c_st;
  const int32_t* table;     // null: contiguous
  int64_t table_stride;
  int32_t page, n_blocks;
  float c;                  // |scale| * log2(e)
  uint32_t flip;            // sign mask for q (0x80008000 when scale < 0)
  int zero;                 // scale is 0
  void* out;
  int64_t o_sr, o_sh;
  int o_vec;                // out takes 16-byte stores
  float* st_o;              // [max_chunks][D / 4][st_rows][4]
  float* st_ml;             // [max_chunks][st_rows][2]
  int64_t st_rows;          // hkv * n_rows * G: state row kvh * n_rows * G + row * G + head in the group
};

template <int D>
struct Cfg {
  static constexpr int DP = D < 64 ? 64 : D;
  static constexpr int NH = DP / 64;
  static constexpr int BLK = prefix::block_tokens(D);
  static constexpr int BOX = 64 * 128;
  static constexpr int HALF = BLK / 64 * BOX;
  static constexpr int STAGE = NH * HALF;         // 16 KB
  static constexpr int STAGES = D == 128 ? 8 : 10;
  static constexpr int QHALF = kRows * 128;
  static constexpr int QTILE = NH * QHALF;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * QTILE + 512;
  static constexpr uint32_t S_COL = 0, P_COL = 2 * BLK, O_COL = 512 - 2 * DP;
  static_assert(P_COL + BLK <= O_COL, "TMEM");
};

// Tokens a chunk: a function of the cached tokens alone.  Short chunks give a small batch enough items to fill the SMs, but
// each costs a row a state of D floats out and in again, about three blocks' time a tile.  Measured in chunks of 512, 768
// and 1024: 64 requests of 200 to 4000 tokens 145, 131 and 126 us, 8 of one to two rows and up to 2776 tokens 17, 18 and 21;
// of 1024, 1536 and 2048: 9 requests of 8000 to 20,000 tokens 191, 164 and 162 us, one of 6000 28, 37 and 45.
__host__ __device__ inline int64_t chunk_tokens(int64_t kv) {
  if (kv <= 4096) return 768;
  if (kv <= 8192) return 1024;
  if (kv <= 16384) return 1536;
  if (kv <= 32768) return 2048;
  return ((kv + 15) / 16 + 127) / 128 * 128;
}

// A sequence's extents; nothing (rows = 0) where they are bad.
struct Seq {
  int row0, rows, kv, total, chunk, n_chunks;
};
// WARP: called by a whole converged warp; what is loaded is then one value for it as the compiler sees it, too (the MMA
// issuers' operands stay in uniform registers).
template <int D, bool WARP>
__device__ __forceinline__ Seq seq_at(const Params& p, int b, bool report) {
  Seq s;
  s.row0 = p.cu_rows[b];
  int r1 = p.cu_rows[b + 1];
  s.kv = p.kv_lens[b];
  if (WARP) {
    s.row0 = __shfl_sync(0xffffffffu, s.row0, 0);
    r1 = __shfl_sync(0xffffffffu, r1, 0);
    s.kv = __shfl_sync(0xffffffffu, s.kv, 0);
  }
  s.rows = r1 - s.row0;
  const bool bad = s.row0 < 0 || r1 < s.row0 || r1 > p.n_rows || s.rows > p.max_rows ||
                   (s.rows > 0 && (s.kv < 0 || s.kv > p.capacity - s.rows));
  if (bad && report) report_error(DK_ERR_DEVICE_CHECK, kDetLens);
  if (bad || s.rows == 0) {
    s.rows = s.total = s.n_chunks = s.kv = 0;
    s.chunk = 1;
    return s;
  }
  s.total = s.kv + s.rows;
  s.chunk = static_cast<int>(chunk_tokens(s.kv));
  s.n_chunks = (s.total + s.chunk - 1) / s.chunk;
  return s;
}

// The items of a sequence: units (KV heads, or pairs of them where the rows fit a tile), of each its chunks, of each the
// pairs of tiles, which so find the chunk's keys in L2; and their cost, in blocks.
struct Cost {
  int units;
  int inner;             // items a (unit, chunk): pairs of tiles (solo: tiles), or one where the rows fit a tile
  int chunk, last;       // cost of an item of a whole chunk, of the last one
};
// What an item costs beside its blocks (states out, the first scores), in blocks.
template <int D>
constexpr int kItemCost = D == 128 ? 3 : 2;

template <int D>
__device__ __forceinline__ Cost cost_of(const Params& p, const Seq& s) {
  constexpr int BLK = Cfg<D>::BLK;
  Cost c;
  const int nt = (s.rows + p.rpt - 1) / p.rpt;
  c.units = nt > 1 || (nt == 1 && p.solo) ? p.hkv : nt == 1 ? (p.hkv + 1) >> 1 : 0;
  c.inner = nt <= 1 ? 1 : p.solo ? nt : (nt + 1) >> 1;
  c.chunk = s.chunk / BLK + kItemCost<D>;
  c.last = (s.total - (s.n_chunks - 1) * s.chunk + BLK - 1) / BLK + kItemCost<D>;
  return c;
}

// The order of the items: by falling cost, in groups of a sequence's items of one cost (its whole chunks, its last ones),
// dealt to the CTAs there and back.  So the CTAs' shares end within about the smallest items' cost of one another (64
// requests, 148 CTAs: 197,000 cycles for the last CTA and 185,000 on average; runs of neighbouring items had 239,000 for the
// last and 198,000 for the median).  Items taken one by one as a CTA gets to them end no closer, and the walk through shared
// memory that this needs made every warp slower (131 -> 146 us).  The order decides no bit.
// One CTA, bound by its barriers and look-ups: 6.4 us alone for 64 requests (1024 threads: 8.4), of which about 2 are hidden.
// Scratch, int32: [0] groups, [1] items, then by group its sequence (times 2, plus 1 for last chunks) and its first item.
__host__ __device__ inline int64_t plan_ints(int64_t n_seqs) { return 4 + 4 * n_seqs; }

constexpr int kPlanThreads = 256;
template <int D>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ Params p) {
  __shared__ int bucket[kPlanThreads];   // by cost, the most expensive first: groups, then their places
  __shared__ int warps[kPlanThreads / 32];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  int32_t *group = p.plan + 4, *first = group + 2 * p.n_seqs;
  auto scan = [&](int mine, int& total) {   // exclusive, block-wide
    int v = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 32; ++i) {
      if (i < warp) before += warps[i];
      total += warps[i];
    }
    return before + v - mine;
  };
  auto place = [](int cost) { return kPlanThreads - 1 - min(cost, kPlanThreads - 1); };
  bucket[tid] = 0;
  __syncthreads();
  for (int b = tid; b < p.n_seqs; b += kPlanThreads) {
    const Seq s = seq_at<D, false>(p, b, true);
    if (s.n_chunks == 0) continue;
    const Cost c = cost_of<D>(p, s);
    if (s.n_chunks > 1) atomicAdd(&bucket[place(c.chunk)], 1);
    atomicAdd(&bucket[place(c.last)], 1);
  }
  __syncthreads();
  int groups;
  const int at = scan(bucket[tid], groups);
  __syncthreads();
  bucket[tid] = at;
  __syncthreads();
  for (int b = tid; b < p.n_seqs; b += kPlanThreads) {
    const Seq s = seq_at<D, false>(p, b, false);
    if (s.n_chunks == 0) continue;
    const Cost c = cost_of<D>(p, s);
    const int each = c.units * c.inner;   // items a chunk
    if (s.n_chunks > 1) {
      const int g = atomicAdd(&bucket[place(c.chunk)], 1);
      group[g] = 2 * b;
      first[g] = each * (s.n_chunks - 1);
    }
    const int g = atomicAdd(&bucket[place(c.last)], 1);
    group[g] = 2 * b + 1;
    first[g] = each;
  }
  int items = 0;
  for (int g0 = 0; g0 < groups; g0 += kPlanThreads) {
    __syncthreads();
    const int g = g0 + tid;
    int total;
    const int before = scan(g < groups ? first[g] : 0, total);
    if (g < groups) first[g] = items + before;
    items += total;
  }
  if (tid == 0) {
    p.plan[0] = groups;
    p.plan[1] = items;
  }
}

// A CTA's walk over its items, by a whole warp: a lane looks one of the next 32 up.
template <int D>
struct Walk {
  static constexpr int BLK = Cfg<D>::BLK;
  // of the lane's item
  int l_b, l_u, l_chunk, l_pair, l_row0, l_rows, l_kv;
  int round, n_rounds;       // the item, and how many there are for this CTA
  // of the item
  Seq s;
  int b, chunk, kvh;         // sequence, chunk, KV head of tile 0
  int row0[2];               // first row of the sequence that is a tile's
  int tiles, streams;        // tiles with work; K/V streams (2: tile 1 is the next KV head)
  int t_begin, tokens, n_blocks;
  bool last_reader;          // no later item reads this one's keys

  __device__ __forceinline__ explicit Walk(const Params& p) {
    round = 0;
    if (p.plan) {
      const int items = p.plan[1], cta = static_cast<int>(blockIdx.x), n = static_cast<int>(gridDim.x);
      n_rounds = __shfl_sync(0xffffffffu, items / n + (items / n % 2 ? cta >= n - items % n : cta < items % n), 0);
    } else {
      n_rounds = 1;   // an item a CTA, as far as there are any
    }
    if (n_rounds > 0) {
      look_up(p);
      settle(p);
    }
  }
  __device__ __forceinline__ bool more() const { return round < n_rounds; }
  __device__ __forceinline__ void next(const Params& p) {
    if (++round >= n_rounds) return;
    if ((round & 31) == 0) look_up(p);
    settle(p);
  }
  __device__ __forceinline__ void look_up(const Params& p) {
    const int lane = static_cast<int>(threadIdx.x & 31), n = static_cast<int>(gridDim.x);
    l_b = l_u = l_chunk = l_pair = l_row0 = l_rows = l_kv = 0;
    if (p.plan) {
      const int k = round + lane, cta = static_cast<int>(blockIdx.x);
      if (k < n_rounds) {
        const int item = k * n + (k & 1 ? n - 1 - cta : cta);
        const int32_t *group = p.plan + 4, *first = group + 2 * p.n_seqs;
        int lo = 0, hi = p.plan[0];
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (first[mid] <= item) lo = mid; else hi = mid;
        }
        const int g = group[lo];
        l_b = g >> 1;
        const Seq q = seq_at<D, false>(p, l_b, false);
        const Cost c = cost_of<D>(p, q);
        int r = item - first[lo];
        const int chunks = g & 1 ? 1 : q.n_chunks - 1;    // of the group: [unit][chunk][pair]
        l_pair = r % c.inner;
        r /= c.inner;
        l_u = r / chunks;
        l_chunk = g & 1 ? q.n_chunks - 1 : r - l_u * chunks;
        l_row0 = q.row0;
        l_rows = q.rows;
        l_kv = q.kv;
      }
    } else {
      // item (chunk, sequence, unit) of the CTA's number
      const uint32_t w = blockIdx.x, r = w / static_cast<uint32_t>(p.units);
      const int u = static_cast<int>(w - r * p.units);
      l_chunk = static_cast<int>(r / static_cast<uint32_t>(p.n_seqs));
      l_b = static_cast<int>(r - l_chunk * static_cast<uint32_t>(p.n_seqs));
      const Seq q = seq_at<D, false>(p, l_b, lane == 0 && u == 0 && l_chunk == 0);
      const Cost c = cost_of<D>(p, q);
      l_u = u / c.inner;
      l_pair = u - l_u * c.inner;
      l_row0 = q.row0;
      l_rows = q.rows;
      l_kv = q.kv;
      const bool there = l_chunk < q.n_chunks && l_u < c.units;
      if (!__shfl_sync(0xffffffffu, there, 0)) n_rounds = 0;
    }
  }
  __device__ __forceinline__ void settle(const Params& p) {
    auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, round & 31); };
    b = of(l_b);
    chunk = of(l_chunk);
    const int u = of(l_u), pair = of(l_pair);
    s.row0 = of(l_row0);
    s.rows = of(l_rows);
    s.kv = of(l_kv);
    s.total = s.kv + s.rows;
    s.chunk = static_cast<int>(chunk_tokens(s.kv));
    s.n_chunks = (s.total + s.chunk - 1) / s.chunk;
    const int nt = (s.rows + p.rpt - 1) / p.rpt;
    if (nt > 1) {
      kvh = u;
      row0[0] = pair * (p.solo ? 1 : 2) * p.rpt;
      row0[1] = row0[0] + p.rpt;
      tiles = !p.solo && row0[1] < s.rows ? 2 : 1;
      streams = 1;
      last_reader = row0[0] + tiles * p.rpt >= s.rows;
    } else {
      kvh = p.solo ? u : 2 * u;
      row0[0] = row0[1] = 0;
      tiles = streams = !p.solo && kvh + 1 < p.hkv ? 2 : 1;
      last_reader = true;
    }
    t_begin = chunk * s.chunk;
    tokens = min(s.total - t_begin, s.chunk);
    n_blocks = (tokens + BLK - 1) / BLK;
  }
  // a block that holds drafts
  __device__ __forceinline__ bool drafts(int block) const { return t_begin + (block + 1) * BLK > s.kv; }
  __device__ __forceinline__ int head(int t) const { return kvh + (streams == 2 ? t : 0); }
};

// A whole warp's wait for fill f of a ring of N stages, whose barriers complete once a lap.  A parity tells a lap only from
// its neighbours, so whoever waits must know that fill f - N has landed: the number of stages is even, as is that of an
// item's fills, so fill f - N was this tile's own, or shared, and either way its issuer has waited for it (a tile without
// work in a shared item waits all the same).  Nor can the barrier be ahead: f is not released before this tile has met it.
template <int N>
__device__ __forceinline__ bool wait_fill(uint64_t* full, uint32_t f, bool& abort_flag) {
  static_assert(N % 2 == 0, "stages");
  return warp_wait(&full[f % N], (f / N) & 1, kDetFull, abort_flag);
}

// Which of the 64 tokens from p0 on a row sees (word: the first of its mask).
__device__ __forceinline__ uint64_t sees64(const Params& p, const Seq& s, const uint64_t* row, uint64_t word, int p0) {
  if (p0 >= s.total) return 0;
  const int off = p0 - s.kv;
  uint64_t bits;
  if (off <= -64) {
    bits = ~0ull;
  } else if (off < 0) {
    bits = (word << -off) | ((1ull << -off) - 1);
  } else {
    const int w = off >> 6, sh = off & 63;
    bits = w == 0 ? word >> sh : w < p.words ? row[w] >> sh : 0;
    if (sh && w + 1 < p.words) bits |= row[w + 1] << (64 - sh);
  }
  const int left = s.total - p0;
  return left < 64 ? bits & ((1ull << left) - 1) : bits;
}
// A row that sees nothing at all (asked only where the weights sum up to 0).
__device__ __forceinline__ bool sees_nothing(const Params& p, const Seq& s, const uint64_t* row) {
  if (s.kv > 0) return false;
#pragma unroll 1
  for (int p0 = 0; p0 < s.total; p0 += 64)
    if (sees64(p, s, row, row[0], p0)) return false;
  return true;
}

__device__ __forceinline__ bool wild16(uint32_t u, uint32_t expo) {
  return (u & expo) == expo || ((u >> 16) & expo) == expo;
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t expo_bits() {
  return std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
}
// The word without its non-finite halves.
__device__ __forceinline__ uint32_t tamed(uint32_t u, uint32_t expo) {
  if ((u & expo) == expo) u &= 0xffff0000u;
  if (((u >> 16) & expo) == expo) u &= 0xffffu;
  return u;
}

// The non-finite values of the drafts of this chunk that the row sees, added to 32 columns of its accumulator.  (Inlined, as
// all of the kernel is: with a function call in it the two register budgets of its warps would not hold.)
template <typename T>
__device__ __forceinline__ void add_back(const Params& p, const Seq& s, const uint64_t* row, int b, int kvh, int begin, int end,
                                         int col, float (&o)[32]) {
#pragma unroll 1
  for (int t = max(begin, s.kv); t < end; ++t) {
    if (!(sees64(p, s, row, row[0], t) & 1)) continue;
    int64_t at = b;
    int tok = t;
    if (p.table) {
      const int pg = t / p.page;
      at = p.table[b * p.table_stride + pg];
      if (at < 0 || at >= p.n_blocks) at = 0;
      tok -= pg * p.page;
    }
    const T* v = static_cast<const T*>(p.v) + at * p.c_sn + kvh * p.c_sh + tok * p.c_st + col;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float x = to_f32<T>(v[i]);
      if (!(fabsf(x) < INFINITY)) o[i] += x;
    }
  }
}

// Keys and values that no other item reads leave L2 before the states, which are read again.
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void tma_load_4d_once(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z,
                                                 int w, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
      "[%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const __grid_constant__ Maps maps,
                                                           const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int BLK = C::BLK;
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = base;
  uint8_t* s_q = ring + C::STAGES * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_q + 2 * C::QTILE);
  uint64_t* empty = full + C::STAGES;
  uint64_t* raw = empty + C::STAGES;      // values landed that are still to be cleaned
  uint64_t* s_full = raw + C::STAGES;     // [2] by tile: scores formed
  uint64_t* s_free = s_full + 2;          // [2] by tile: scores in registers
  uint64_t* p_ready = s_free + 2;         // [2] by tile: weights in TMEM
  uint64_t* o_full = p_ready + 2;         // [2] by tile: P.V of a block done
  uint64_t* o_free = o_full + 2;          // [2] by tile: the accumulator has been read
  uint64_t* q_full = o_free + 2;          // [2] by tile: queries landed
  uint64_t* q_ready = q_full + 2;         // [2] by tile: and their sign is right
  uint64_t* q_free = q_ready + 2;         // [2] by tile: all scores of them are formed
  uint64_t* turn = q_free + 2;            // [8] by softmax warp: the exponential unit is its
  uint64_t* done = turn + kSoftWarps;     // [2]
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(done + 2);
  uint32_t* s_wild = s_tmem + 1;          // by stage: its values had non-finite elements
  static_assert((3 * C::STAGES + 16 + kSoftWarps + 2) * 8 + 4 + 4 * C::STAGES <= 512, "barriers");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);   // both MMA issuers, or the one whose stage it is twice
      mbar_init(&raw[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], 128);
      mbar_init(&p_ready[t], 128);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 128);
      mbar_init(&q_full[t], 1);
      mbar_init(&q_ready[t], 1);
      mbar_init(&q_free[t], 1);
    }
    for (int i = 0; i < kSoftWarps; ++i) mbar_init(&turn[i], 1);
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    fence_mbar_init();
  }
  if (warp == kSoftWarps && lane == 0) {
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (warp == kSoftWarps + 1) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();

  bool abort_flag = false;
  // Stages of an item's block b: K of stream i in fill f0 + 2 streams b + i, V behind the K's of the block.
  // A block that holds drafts has its values cleaned.
  if (warp >= kSoftWarps) {
    prefix::reg_dec<prefix::kIoRegs>();
    if (warp == kSoftWarps) {
      // ---------------- TMA producer ----------------
      int stage = 0;
      uint32_t phase = 0;
      uint32_t fills = 0;
      const uint64_t policy = evict_first();
      for (Walk<D> it(p); it.more() && !abort_flag; it.next(p)) {
        for (int b = 0; b < it.n_blocks && !abort_flag; ++b) {
          int tok[BLK / 64], slab[BLK / 64], boxes = 0;   // 64-token boxes that hold a token
#pragma unroll
          for (int h = 0; h < BLK / 64; ++h) {
            tok[h] = it.t_begin + b * BLK + 64 * h;
            slab[h] = it.b;
            if (b * BLK + 64 * h >= it.tokens) continue;
            boxes = h + 1;
            if (p.table) {   // a page holds whole boxes
              const int pg = tok[h] / p.page;
              tok[h] -= pg * p.page;
              slab[h] = p.table[it.b * p.table_stride + pg];
              if (slab[h] < 0 || slab[h] >= p.n_blocks) {
                if (lane == 0) report_error(DK_ERR_DEVICE_CHECK, kDetPage);
                slab[h] = 0;
              }
            }
          }
          const bool clean = it.drafts(b);
          for (int e = 0; e < 2 * it.streams; ++e) {
            const bool val = e >= it.streams;
            const int kvh = it.kvh + (val ? e - it.streams : e);
            if (!warp_wait(&empty[stage], phase ^ 1u, kDetEmpty, abort_flag)) break;
            uint8_t* st = ring + stage * C::STAGE;
            uint64_t* bar = val && clean ? &raw[stage] : &full[stage];
            if (lane == 0) {
              mbar_arrive_expect_tx(bar, boxes * C::NH * C::BOX);
#pragma unroll
              for (int h = 0; h < BLK / 64; ++h)
#pragma unroll
                for (int n = 0; n < C::NH; ++n)
                  if (h < boxes) {
                    uint8_t* to = st + n * C::HALF + h * C::BOX;
                    const CUtensorMap* from = val ? &maps.v : &maps.k;
                    if (it.last_reader) tma_load_4d_once(to, from, bar, n * 64, tok[h], kvh, slab[h], policy);
                    else tma_load_4d(to, from, bar, n * 64, tok[h], kvh, slab[h]);
                  }
            }
            __syncwarp();
            ++fills;
            if (++stage == C::STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      // every copy has landed before the CTA may end (a cleaned stage's barrier completes behind its copies)
      bool drain = false;
      for (uint32_t f = (fills > C::STAGES ? fills - C::STAGES : 0); f < fills; ++f)
        warp_wait(&full[f % C::STAGES], static_cast<uint32_t>((f / C::STAGES) & 1), kDetDrain, drain);
    } else if (warp == kSoftWarps + 1 || warp == kSoftWarps + 2) {
      // ---------------- MMA issuers, one a tile ----------------
      const int t = warp - (kSoftWarps + 1);
      constexpr uint32_t idesc_s = umma_idesc_f16(FMT, 0, 0, kRows, BLK);
      constexpr uint32_t idesc_o = umma_idesc_f16(FMT, 0, 1, kRows, C::DP);
      const uint64_t k_desc = umma_sdesc(smem_u32(ring), 16, 1024, 2);
      const uint64_t v_desc = umma_sdesc(smem_u32(ring), C::HALF, 1024, 2);
      const uint64_t q_desc = umma_sdesc(smem_u32(s_q) + t * C::QTILE, 16, 1024, 2);
      const uint32_t s_col = tmem + C::S_COL + t * BLK, p_col = tmem + C::P_COL + t * (BLK / 2);
      const uint32_t o_col = tmem + C::O_COL + t * C::DP;
      const bool leader = prefix::elect_one();
      uint64_t* const q_bar = (p.flip | p.zero) ? &q_ready[t] : &q_full[t];
      uint32_t fill = 0;
      uint32_t qph = 0, sph = 0, pph = 0;    // q_bar, s_free, p_ready parities
      uint32_t oph = 1;                      // o_free parity (the first wait passes)
      bool mine = false;                     // the item's tiles have stages of their own
      auto landed = [&](uint32_t f) { return wait_fill<C::STAGES>(full, f, abort_flag); };
      auto release = [&](uint32_t f) {
        tc_commit(&empty[f % C::STAGES]);
        if (mine) tc_commit(&empty[f % C::STAGES]);
      };
      auto issue_qk = [&](uint32_t f, bool last_q) {      // scores from the K block of fill f
        if (leader) {
          const uint64_t kd = k_desc + static_cast<uint64_t>((f % C::STAGES) * (C::STAGE / 16));
#pragma unroll
          for (int j = 0; j < C::DP / 16; ++j)
            tc_mma_f16(s_col, q_desc + static_cast<uint64_t>(((j >> 2) * C::QHALF + (j & 3) * 32) / 16),
                       kd + static_cast<uint64_t>(((j >> 2) * C::HALF + (j & 3) * 32) / 16), idesc_s, j > 0 ? 1u : 0u);
          tc_commit(&s_full[t]);
          release(f);
          if (last_q) tc_commit(&q_free[t]);
        }
        __syncwarp();
      };
      for (Walk<D> it(p); it.more() && !abort_flag; it.next(p)) {
        const int nb = it.n_blocks;
        const uint32_t per = 2 * it.streams;
        const uint32_t f0 = fill + (it.streams == 2 ? t : 0);   // K of block b: f0 + per b; V: streams further
        fill += per * nb;
        mine = it.streams == 2;
        if (t >= it.tiles) {
          // not this tile's item: its stages still need this warp's release, in order
          for (uint32_t f = f0; f != fill; ++f) {
            if (!landed(f)) break;
            if (leader) mbar_arrive(&empty[f % C::STAGES]);
          }
          continue;
        }
        if (!warp_wait(q_bar, qph, kDetQ, abort_flag)) break;
        qph ^= 1u;
        if (!landed(f0)) break;
        tc_fence_after();
        issue_qk(f0, nb == 1);
        for (int b = 0; b < nb; ++b) {
          const bool more = b + 1 < nb;
          const uint32_t fv = f0 + per * b + it.streams, fk = f0 + per * (b + 1);
          // the next scores, as soon as these are in registers (the last block's release is for the next item)
          if (more && !landed(fk)) break;
          if (!warp_wait(&s_free[t], sph, kDetScoresFree, abort_flag)) break;
          sph ^= 1u;
          tc_fence_after();
          if (more) issue_qk(fk, b + 2 == nb);
          if (!landed(fv)) break;
          const int valid = min(BLK, it.tokens - b * BLK);
          const int steps = (valid + 15) >> 4;   // 16-token steps of P.V that hold a token
          if (b == 0) {
            if (!warp_wait(&o_free[t], oph, kDetOutFree, abort_flag)) break;
            oph ^= 1u;
          }
          if (!warp_wait(&p_ready[t], pph, kDetProbs, abort_flag)) break;
          pph ^= 1u;
          tc_fence_after();
          if (leader) {
            const uint64_t vd = v_desc + static_cast<uint64_t>((fv % C::STAGES) * (C::STAGE / 16));
#pragma unroll
            for (int j = 0; j < BLK / 16; ++j)
              if (j < steps)
                prefix::mma_ts(o_col, p_col + j * 8, vd + static_cast<uint64_t>(j * (2048 / 16)), idesc_o,
                               (b == 0 && j == 0) ? 0u : 1u);
            tc_commit(&o_full[t]);
            release(fv);
          }
          __syncwarp();
        }
      }
      // all issued MMAs are complete before TMEM is freed
      if (leader) tc_commit(&done[t]);
      __syncwarp();
      bool fin = false;
      warp_wait(&done[t], 0, kDetDone, fin);
    } else if (warp == kSoftWarps + 3) {
      // ---------------- an item's queries, values of draft blocks ----------------
      constexpr uint32_t expo = expo_bits<T>();
      uint32_t fill = 0;
      uint32_t seen = 0;                     // raw parities, a bit a stage
      uint32_t fph = 3u, qph = 0u;           // q_free (the first wait passes) and q_full parities, a bit a tile
      for (Walk<D> it(p); it.more() && !abort_flag; it.next(p)) {
        for (int t = 0; t < it.tiles && !abort_flag; ++t) {
          if (!warp_wait(&q_free[t], (fph >> t) & 1u, kDetQFree, abort_flag)) break;
          fph ^= 1u << t;
          uint8_t* at = s_q + t * C::QTILE;
          const int bytes = p.rpt * p.G * 128;   // of a 64-element half; rows behind the tensor's are zero
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[t], C::NH * bytes);
            for (int n = 0; n < C::NH; ++n)
              tma_load_3d(at + n * C::QHALF, &maps.q, &q_full[t], n * 64, it.head(t) * p.G, it.s.row0 + (t ? it.row0[1] : it.row0[0]));
          }
          __syncwarp();
          if (p.flip | p.zero) {
            if (!warp_wait(&q_full[t], (qph >> t) & 1u, kDetQ, abort_flag)) break;
            qph ^= 1u << t;
            for (int e = lane; e < C::NH * bytes / 16; e += 32) {
              const int n = e / (bytes / 16);
              uint4* v = reinterpret_cast<uint4*>(at + n * C::QHALF) + (e - n * (bytes / 16));
              uint4 x = *v;
              x.x ^= p.flip;
              x.y ^= p.flip;
              x.z ^= p.flip;
              x.w ^= p.flip;
              *v = p.zero ? prefix::times_zero<T>(x) : x;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready[t]);
          }
        }
        const uint32_t per = 2 * it.streams, f0 = fill;
        fill += per * it.n_blocks;
        const int first = max(0, (it.s.kv - it.t_begin) / BLK);   // the first block with drafts, if any
        for (int b = first; b < it.n_blocks && !abort_flag; ++b) {
          if (!it.drafts(b)) continue;
          for (int i = 0; i < it.streams; ++i) {
            const uint32_t f = f0 + per * b + it.streams + i, stage = f % C::STAGES;
            if (!warp_wait(&raw[stage], (seen >> stage) & 1u, kDetRaw, abort_flag)) break;
            seen ^= 1u << stage;
            uint8_t* vb = ring + stage * C::STAGE;
            const int begin = max(0, it.s.kv - it.t_begin - b * BLK);    // rows of the block
            const int valid = min(BLK, it.tokens - b * BLK), end = (valid + 15) & ~15;
            bool wild = false;
            for (int e = lane; e < (end - begin) * C::NH * 8; e += 32) {
              const int r = begin + e / (C::NH * 8), c = e % (C::NH * 8);
              uint4* at = reinterpret_cast<uint4*>(vb + (c >> 3) * C::HALF + r * 128 + (c & 7) * 16);
              if (r >= valid) {
                *at = make_uint4(0, 0, 0, 0);
                continue;
              }
              const uint4 v = *at;
              if (wild16(v.x, expo) || wild16(v.y, expo) || wild16(v.z, expo) || wild16(v.w, expo)) {
                wild = true;
                *at = make_uint4(tamed(v.x, expo), tamed(v.y, expo), tamed(v.z, expo), tamed(v.w, expo));
              }
            }
            wild = __any_sync(0xffffffffu, wild);
            if (lane == 0) s_wild[stage] = wild ? 1u : 0u;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
          }
        }
      }
    }
  } else {
    // ---------------- softmax: one row a thread ----------------
    prefix::reg_inc<prefix::kSoftRegs>();
    const int t = warp >> 2;                    // tile of the item
    const int r = threadIdx.x & 127;            // row of the tile
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_t = tmem + lane_base + C::O_COL + t * C::DP;
    const uint32_t s_t = tmem + lane_base + C::S_COL + t * BLK, p_t = tmem + lane_base + C::P_COL + t * (BLK / 2);
    uint32_t sph = 0;                           // s_full parity
    uint32_t tph = t ^ 1;                       // turn parity (tile 0 goes first)
    uint32_t ocnt = 0;                          // blocks of this tile whose weights are handed over
    uint32_t oseen = 0;                         // of them, those whose P.V this warp has waited for
    uint32_t fill = 0;
    const int i_r = static_cast<int>(div_by(static_cast<uint32_t>(r), p.group)), g_r = r - i_r * p.G;   // draft and head of it
    // All P.V so far are done; each warp takes every phase of o_full once and in order (see dk_prefix.cuh).
    auto pv_done = [&]() {
      if (oseen == ocnt) return true;
      const bool ok = warp_wait(&o_full[t], oseen & 1, kDetOut, abort_flag);
      tc_fence_after();
      oseen = ocnt;
      return ok;
    };
    for (Walk<D> it(p); it.more() && !abort_flag; it.next(p)) {
      const uint32_t per = 2 * it.streams;
      const uint32_t fv0 = fill + it.streams + (it.streams == 2 ? t : 0);   // V of block b: fv0 + per b
      fill += per * it.n_blocks;
      if (t >= it.tiles) continue;
      const int kvh = it.head(t), i0 = t ? it.row0[1] : it.row0[0], here = min(p.rpt, it.s.rows - i0);   // drafts of the tile
      const bool valid_row = i_r < here;
      const bool warp_live = (warp & 3) * 32 < here * p.G;
      const int row = it.s.row0 + i0 + (valid_row ? i_r : 0);
      const uint64_t* mask = p.mask + row * p.mask_stride;
      const uint64_t word = it.drafts(it.n_blocks - 1) ? mask[0] : 0;   // on its way long before it is asked for
      float m = -INFINITY, l = 0.0f;
      bool wild = false;
      for (int b = 0; b < it.n_blocks; ++b) {
        const bool first = b == 0, last = b + 1 == it.n_blocks;
        const bool drafts = it.drafts(b);
        if (!warp_wait(&s_full[t], sph, kDetScores, abort_flag)) break;
        sph ^= 1u;
        tc_fence_after();
        if (warp_live) {
          constexpr int NR = BLK / 32;
          float s[NR][32];
#pragma unroll
          for (int c = 0; c < NR; ++c) tmem_ld_32x32b_x32(s_t + c * 32, s[c]);
          tmem_ld_wait();
          tc_fence_before();
          mbar_arrive(&s_free[t]);
          if (drafts) {
#pragma unroll
            for (int h = 0; h < NR / 2; ++h) {
              const uint64_t sees = valid_row ? sees64(p, it.s, mask, word, it.t_begin + b * BLK + 64 * h) : 0;
#pragma unroll
              for (int i = 0; i < 64; ++i) s[2 * h + (i >> 5)][i & 31] = (sees >> i & 1u) ? s[2 * h + (i >> 5)][i & 31] : -INFINITY;
            }
          }
          float mx = -INFINITY;
          {
            float part[2 * NR];
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) {
              const float* v = &s[c >> 1][(c & 1) * 16];
              part[c] = fmaxf(v[0], v[1]);
#pragma unroll
              for (int i = 2; i < 16; i += 2) part[c] = fmaxf(part[c], fmaxf(v[i], v[i + 1]));
            }
#pragma unroll
            for (int c = 0; c < 2 * NR; ++c) mx = fmaxf(mx, part[c]);
          }
          mx = __fmul_rn(mx, p.c);
          float alpha = 1.0f;
          if (first) {
            m = mx;
            l = 0.0f;
          } else if (mx > m + prefix::kLazy) {   // m = -inf: any finite maximum is above it
            alpha = exp2_hw(__fsub_rn(m, mx));
            m = mx;
          }
          if (!first && __any_sync(0xffffffffu, alpha != 1.0f)) {
            // rescale the accumulator once the previous block's P.V is done
            if (!pv_done()) break;
#pragma unroll 1
            for (int c = 0; c < C::DP / 16; ++c) {
              uint32_t o[16];
              prefix::tmem_ld_x16(o_t + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__fmul_rn(__uint_as_float(o[i]), alpha));
              prefix::tmem_st_x16(o_t + c * 16, o);
            }
            l = __fmul_rn(l, alpha);
          }
          // the last block's P.V has read its weights (long since)
          if (!pv_done()) break;
          // the two tiles' warps of a scheduler take turns on its exponential unit (see dk_prefix.cuh)
          if (it.tiles == 2) {
            if (!warp_wait(&turn[warp], tph, kDetTurn, abort_flag)) break;
            tph ^= 1u;
          }
          const float neg = (m == -INFINITY) ? 0.0f : -m;
          const float2 c2 = make_float2(p.c, p.c), n2 = make_float2(neg, neg);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
          __syncwarp();
#pragma unroll
          for (int c = 0; c < NR; ++c) {
            uint32_t pk[16];
            if (c == NR / 2) prefix::arrive_if(&turn[warp ^ 4], it.tiles == 2 && lane == 0);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float2 e = fma2(make_float2(s[c][i], s[c][i + 1]), c2, n2);
              e.x = exp2_hw(e.x);
              e.y = exp2_hw(e.y);
              sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
              pk[i >> 1] = pack2<T>(e.x, e.y);
            }
            prefix::tmem_st_x16(p_t + c * 16, pk);
          }
          tmem_st_wait();
          const float2 ps = add2(sum[0], sum[1]);
          l = __fadd_rn(l, __fadd_rn(ps.x, ps.y));
        } else {
          mbar_arrive(&s_free[t]);
          if (it.tiles == 2) {
            if (!warp_wait(&turn[warp], tph, kDetTurn, abort_flag)) break;
            tph ^= 1u;
            if (lane == 0) mbar_arrive(&turn[warp ^ 4]);
          }
          if (!pv_done()) break;
        }
        if (drafts) {   // (its values stay until this tile's weights have met them)
          const uint32_t f = fv0 + per * b;
          if (!wait_fill<C::STAGES>(full, f, abort_flag)) break;
          wild |= s_wild[f % C::STAGES] != 0;
        }
        tc_fence_before();
        mbar_arrive(&p_ready[t]);
        ++ocnt;
        if (last) {
          if (!pv_done()) break;
          if (warp_live) {
            // state row
            const int64_t n = (kvh * static_cast<int64_t>(p.n_rows) + row) * p.G + g_r;
            const bool whole = it.s.n_chunks == 1;   // the output, at once
            float4* dst = reinterpret_cast<float4*>(p.st_o) + static_cast<int64_t>(it.chunk) * (D / 4) * p.st_rows + n;
            T* out = static_cast<T*>(p.out) + row * p.o_sr + (kvh * p.G + g_r) * p.o_sh;
            const bool empty = whole && valid_row && l == 0.0f && sees_nothing(p, it.s, mask);
            const float inv = __frcp_rn(l);   // one more rounding of 2^-24 an output, before the type's
            if (!whole && valid_row)
              *reinterpret_cast<float2*>(p.st_ml + 2 * (it.chunk * p.st_rows + n)) = make_float2(m, l);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              __syncwarp();   // rows part in what they store, the load is the whole warp's
              tmem_ld_32x32b_x32(o_t + c * 32, o);
              tmem_ld_wait();
              if (wild && valid_row)
                add_back<T>(p, it.s, mask, it.b, kvh, it.t_begin, it.t_begin + it.tokens, c * 32, o);
              if (valid_row && !whole) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  dst[i * p.st_rows] = make_float4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
                dst += 8 * p.st_rows;
              } else if (valid_row) {
                uint32_t u[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  u[i] = empty ? 0u : pack2<T>(__fmul_rn(o[2 * i], inv), __fmul_rn(o[2 * i + 1], inv));
                if (p.o_vec) {
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(out + c * 32 + i * 8) = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
                } else {
#pragma unroll
                  for (int i = 0; i < 16; ++i) {
                    out[c * 32 + 2 * i] = *reinterpret_cast<const T*>(&u[i]);
                    out[c * 32 + 2 * i + 1] = *(reinterpret_cast<const T*>(&u[i]) + 1);
                  }
                }
              }
            }
          }
          __syncwarp();
          tc_fence_before();
          mbar_arrive(&o_free[t]);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// out = O / l of a row's chunks, joined in order.  A CTA takes 32 state rows of a (sequence, KV head), a lane each; its
// warps take column quads (one coalesced load a state), and the outputs leave through shared memory.  Bound by the states'
// bytes and latency: alone, behind a flushed L2, 20 us for the 71 MB of the 64 requests (3.5 TB/s).
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads, 3) join_kernel(const __grid_constant__ Params p, int row_tiles) {
  constexpr int WARPS = kJoinThreads / 32, Q = D / 4 / WARPS, UN = Q >= 4 ? 2 : 4;   // quads a warp; states in flight
  __shared__ __align__(16) T s_out[32][D + 2];
  // (lengths and offsets were there before tree_kernel, which has waited for them before it let this kernel begin)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t tile = blockIdx.x % row_tiles, rest = blockIdx.x / row_tiles;
  const int kvh = static_cast<int>(rest % p.hkv), b = static_cast<int>(rest / p.hkv);
  const Seq s = seq_at<D, true>(p, b, false);
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int m0 = static_cast<int>(tile) * 32, mg = s.rows * p.G;
  if (s.n_chunks <= 1 || m0 >= mg) return;
  const bool live = m0 + lane < mg;
  const int64_t n = (kvh * static_cast<int64_t>(p.n_rows) + s.row0) * p.G + m0 + (live ? lane : 0);
  const float4* src = reinterpret_cast<const float4*>(p.st_o) + static_cast<int64_t>(warp) * Q * p.st_rows + n;
  const float2* mls = reinterpret_cast<const float2*>(p.st_ml) + n;
  const int64_t state = p.st_rows * (D / 4);
  float tm = -INFINITY, tl = 0.0f;
  float4 to[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) to[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int c0 = 0; c0 < s.n_chunks; c0 += UN) {
    float2 ml[UN];
    float4 o[UN][Q];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (c0 + u < s.n_chunks) {
        ml[u] = __ldcg(mls + (c0 + u) * p.st_rows);
#pragma unroll
        for (int i = 0; i < Q; ++i) o[u][i] = __ldcg(src + (c0 + u) * state + i * p.st_rows);
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (c0 + u < s.n_chunks) {
        const bool head = c0 + u == 0;
        float a = 0.0f, w = 1.0f;
        if (head) {
          tm = ml[u].x;
          tl = ml[u].y;
        } else {
          tm = join_weights(tm, ml[u].x, a, w);
          tl = join(tl, a, ml[u].y, w);
        }
#pragma unroll
        for (int i = 0; i < Q; ++i) to[i] = head ? o[u][i] : join4(to[i], a, o[u][i], w);
      }
    }
  }
  const int row = s.row0 + (live ? static_cast<int>(div_by(static_cast<uint32_t>(m0 + lane), p.group)) : 0);
  const bool empty = live && tl == 0.0f && sees_nothing(p, s, p.mask + row * p.mask_stride);
  const float inv = __frcp_rn(tl);
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    T* d = &s_out[lane][(warp * Q + i) * 4];
    *reinterpret_cast<uint32_t*>(d) = empty ? 0u : pack2<T>(__fmul_rn(to[i].x, inv), __fmul_rn(to[i].y, inv));
    *reinterpret_cast<uint32_t*>(d + 2) = empty ? 0u : pack2<T>(__fmul_rn(to[i].z, inv), __fmul_rn(to[i].w, inv));
  }
  __syncthreads();
  for (int k = warp; k < 32 && m0 + k < mg; k += WARPS) {
    const int mk = m0 + k, rk = static_cast<int>(div_by(static_cast<uint32_t>(mk), p.group));
    T* dst = static_cast<T*>(p.out) + (s.row0 + rk) * p.o_sr + (kvh * p.G + mk - rk * p.G) * p.o_sh;
#pragma unroll
    for (int d = 0; d < D; d += 32) dst[d + lane] = s_out[k][d + lane];
  }
}

}  // namespace tree
}  // namespace dk
