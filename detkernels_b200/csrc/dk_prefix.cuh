// Attention over a prefix that every row of the batch shares, computed once for all rows.
//
// The query heads of all rows that read KV head h are the rows of one matrix Q_h [R * G, D]; with
// S = Q_h K_h^T * scale, the prefix contributes to each row the softmax state (m, l, O) with
// l = sum 2^(S log2e - m), O = sum 2^(S log2e - m) V, which joins the states of the row's own tokens
// (dk_own.cuh) in combine_kernel: out = O / l.
//
// Fixed reduction structure (the definition of a row's bits):
//   * The prefix is cut into chunks whose size follows the prefix length and head_dim only
//     (chunk_tokens).
//   * Inside a chunk, blocks of block_tokens(D) tokens in order: S from tcgen05.mma (f32 accumulation over D in
//     16-deep steps), a reference maximum m that is raised only when a block's maximum exceeds it
//     by more than 8 (a factor 256, so the weights stay in range of either 16-bit type), weights
//     2^(S c - m) rounded to the input type for P.V (the MMA takes 16-bit operands) as the left operand of a
//     second tcgen05.mma in TMEM, l summed in f32 in a fixed order from the weights before that rounding, which
//     keeps the sums beside the exponentials; over a block's many tokens the roundings average out.
//   * The chunks' states are joined in order inside groups of group_chunks(D) chunks, the groups' states
//     in order, and the states of the row's own tokens last.
// No step looks at another row, so a row's bits do not depend on the batch.
//
// Work: an item is (up to two tiles of 128 rows, KV head, run of tokens), one persistent CTA per SM.
// One warp streams K and V blocks with TMA, one warp a tile issues its MMAs, and a warpgroup a tile does
// the softmax, a row a thread.  The tiles share K and V.  TMEM holds, for either tile, the scores, the
// weights and the accumulator apart, so that the next scores are formed as soon as these are in
// registers and the softmax, whose chain of a block (load, maximum, exponentials) bounds the kernel, does not wait
// for products (exponential unit 50 to 66 % busy, tensor pipe 49 to 32 %): blocks of
// 128 tokens for head_dim <= 64, of 64 for 128 (whose accumulators take half of TMEM).  A run is a whole
// group, whose chunks are joined on chip, or, when that leaves SMs idle, one chunk, whose state
// combine_kernel joins; both give the same bits.  The joined accumulators of head_dim 128 need 128 KB: three
// quarters of them lie where half of the ring would be, the rest in TMEM's last free columns (512 rows of 32
// heads behind 8191 tokens: 101 us against 120 with every chunk's state through memory), so that form
// is one of its own, WHOLE, and a chunk a run keeps the long ring (32 rows behind 32768 tokens: 52 us; 57
// with the short one).
#pragma once

#include "dk_common.cuh"
#include "dk_divide.cuh"
#include "dk_own.cuh"

namespace dk {
namespace prefix {

using own::exp2_hw;
using own::join;
using own::join4;
using own::join_weights;
using own::pack2;

constexpr int kRows = 128;       // rows a tile
constexpr int kSoftWarps = 8;    // a warpgroup a tile
constexpr int kThreads = 384;    // softmax warps, then one for TMA, two for MMA and an idle one
constexpr int kLaunchRegs = 168; // registers a thread at launch; 384 * 168 = 256 * 208 + 128 * 88
constexpr int kSoftRegs = 208;
constexpr int kIoRegs = 88;
constexpr float kLazy = 8.0f;

enum : int {
  kDetEmpty = 0x620,
  kDetFull = 0x621,
  kDetScores = 0x622,
  kDetProbs = 0x623,
  kDetOut = 0x624,
  kDetQ = 0x625,
  kDetOutFree = 0x626,
  kDetDrain = 0x627,
  kDetDone = 0x628,
  kDetScoresFree = 0x629,
  kDetTurn = 0x62b,
  kDetPage = 0x62a,   // a prefix block id outside the pool
};

// Tokens a block.
__host__ __device__ constexpr int block_tokens(int head_dim) { return head_dim <= 64 ? 128 : 64; }

// Chunks a group.
__host__ __device__ constexpr int group_chunks(int head_dim) { return head_dim <= 64 ? 8 : 4; }

// Tokens a chunk: a function of the prefix length and head_dim alone.  Short chunks give a small
// batch enough items to fill the SMs; every chunk of a 128-wide head that is a run of its own costs each row a
// 512-byte state through memory, so those are longer.  Measured: 1500 to 2048 tokens in chunks of 512 and 1024, 4
// rows of 8 heads of 64: 12 and 16 us, 64 rows of 16: 15 and 18, 1000 rows of 16: 51 and 45; 8191 tokens in chunks of
// 512, 1024 and 2048, heads of 128, 4 rows: 21, 24 and 36 us, 128 rows: 47, 39 and 52; 32768 tokens in 16, 24 and 36
// chunks, 32 rows of 32 heads of 128 on 8: 51, 64 and 59 (128, 192 and 288 items for 148 SMs), on 4: 50, 46 and 47.
__host__ __device__ inline int64_t chunk_tokens(int64_t prefix_len, int head_dim) {
  if (prefix_len <= 2048) return 512;
  if (head_dim <= 64) return 1024 * ((prefix_len + 32767) / 32768);
  if (prefix_len <= 16384) return 1024;
  return ((prefix_len + 15) / 16 + 127) / 128 * 128;
}

struct Params {
  const void* q;
  int64_t q_sr, q_sh;
  int32_t hq, hkv, G;
  int32_t rg;             // rows * G
  Divisor31 group;        // by G
  int32_t prefix_len;
  int32_t chunk_blocks;   // blocks a chunk
  int32_t run_blocks;     // blocks a run: a chunk or a group
  int32_t n_runs;
  int32_t n_pairs;        // row tile pairs a KV head
  const int32_t* blocks;  // paged prefix: block ids; null: contiguous
  int32_t page;
  int32_t n_blocks;
  float c;                // |scale| * log2(e)
  uint32_t flip;          // sign mask for q (0x80008000 when scale < 0)
  int zero;               // scale is 0: q is multiplied by it on the way in
  float* st_o;            // [n_runs][D / 4][st_rows][4]: a column of four for 32 rows is one store of a warp
  float* st_ml;           // [n_runs][st_rows][2]
  int64_t st_rows;        // hkv * rows * G: state row (kvh * rows + row) * G + head in the group
};

struct Maps {
  CUtensorMap k, v;       // boxes of 64 elements x 64 tokens
};

template <int D, bool WHOLE>
struct Cfg {
  static constexpr int DP = D < 64 ? 64 : D;      // columns in shared memory and TMEM (D = 32: zero filled)
  static constexpr int NH = DP / 64;              // 64-element halves
  static constexpr int BLK = block_tokens(D);
  static constexpr int BOX = 64 * 128;            // bytes of a 64-token box of 64 elements
  static constexpr int HALF = BLK / 64 * BOX;     // a block's 64-element half
  static constexpr int STAGE = NH * HALF;         // a K or V block
  static constexpr bool GROUPED = D <= 64 || WHOLE;
  static constexpr int STAGES = D == 128 && WHOLE ? 4 : 8;
  static constexpr int QHALF = kRows * 128;       // bytes of a query tile's 64-element half
  static constexpr int QTILE = NH * QHALF;
  static constexpr int RC = D == 128 ? 96 : D;    // columns of the joined chunks in shared memory; the rest in TMEM
  static constexpr int RUN = GROUPED ? 2 * kRows * RC * 4 : 0;   // both tiles [tile][RC / 4][row][4]
  static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * QTILE + RUN + 512;
  // TMEM columns: scores, weights (16-bit pairs) and accumulator of tile t at X_COL + t * width
  static constexpr uint32_t S_COL = 0, P_COL = 2 * BLK, R_COL = P_COL + BLK, O_COL = 512 - 2 * DP;
  static_assert(R_COL + 2 * (D - RC) <= O_COL, "TMEM");
};

// True for one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

template <uint32_t N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <uint32_t N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// D[tmem] (+)= A[tmem] * B[smem desc]: the left operand's 16-bit pairs packed in 32-bit columns.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}

// Two f32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

template <typename T>
__device__ __forceinline__ uint4 times_zero(uint4 v) {
  uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T lo = *reinterpret_cast<const T*>(&u[i]), hi = *(reinterpret_cast<const T*>(&u[i]) + 1);
    u[i] = pack2<T>(__fmul_rn(to_f32<T>(lo), 0.0f), __fmul_rn(to_f32<T>(hi), 0.0f));
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// An arrival of the lanes with `yes`, without a branch that would part them from the warp.
__device__ __forceinline__ void arrive_if(uint64_t* bar, bool yes) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(yes ? 1 : 0)
      : "memory");
}

// Bounded wait by a whole warp, with one answer for all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int detail, bool& abort_flag) {
  const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, detail, abort_flag));
  abort_flag = !ok;
  return ok;
}

struct Item {
  int pair, kvh, run, tiles;
  int t_begin, n_blocks, tokens;   // first token, blocks, tokens
};
template <int BLK>
__device__ __forceinline__ Item item_at(const Params& p, uint32_t w) {
  Item it;
  const uint32_t r = w / static_cast<uint32_t>(p.n_pairs);
  it.pair = static_cast<int>(w - r * p.n_pairs);
  it.run = static_cast<int>(r / static_cast<uint32_t>(p.hkv));
  it.kvh = static_cast<int>(r - it.run * static_cast<uint32_t>(p.hkv));
  it.tiles = (it.pair * 2 + 1) * kRows < p.rg ? 2 : 1;
  it.t_begin = it.run * p.run_blocks * BLK;
  it.tokens = min(p.prefix_len - it.t_begin, p.run_blocks * BLK);
  it.n_blocks = (it.tokens + BLK - 1) / BLK;
  return it;
}

template <typename T, int D, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 1) prefix_kernel(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<D, WHOLE>;
  constexpr int BLK = C::BLK;
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = base;
  uint8_t* s_q = ring + C::STAGES * C::STAGE;
  float4* s_run = reinterpret_cast<float4*>(s_q + 2 * C::QTILE);
  uint64_t* full = reinterpret_cast<uint64_t*>(s_q + 2 * C::QTILE + C::RUN);
  uint64_t* empty = full + C::STAGES;
  uint64_t* s_full = empty + C::STAGES;   // [2] by tile: scores formed
  uint64_t* s_free = s_full + 2;          // [2] by tile: scores in registers
  uint64_t* p_ready = s_free + 2;         // [2] by tile: weights in TMEM
  uint64_t* o_full = p_ready + 2;         // [2] by tile: P.V of a block done
  uint64_t* o_free = o_full + 2;          // [2] by tile: the accumulator has been read
  uint64_t* q_ready = o_free + 2;         // [2] by tile
  uint64_t* turn = q_ready + 2;           // [8] by softmax warp: the exponential unit is its
  uint64_t* done = turn + kSoftWarps;     // [2]
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(done + 2);

  // one value for the whole warp as the compiler sees it: the MMA issuer's operands then stay in
  // uniform registers (from per-thread ones each tcgen05.mma took ~140 cycles to issue)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);   // both MMA issuers
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_free[t], 128);
      mbar_init(&p_ready[t], 128);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 128);
      mbar_init(&q_ready[t], 128);
    }
    for (int i = 0; i < kSoftWarps; ++i) mbar_init(&turn[i], 1);
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    fence_mbar_init();
  }
  if (warp == kSoftWarps && lane == 0) {
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

  const uint32_t n_items = static_cast<uint32_t>(p.n_pairs) * p.hkv * p.n_runs;   // < 2^31 (the host checks)
  bool abort_flag = false;

  if (warp >= kSoftWarps) {
    reg_dec<kIoRegs>();
    if (warp == kSoftWarps && lane == 0) {
      // ---------------- TMA producer: K block, V block, K block, ... ----------------
      int stage = 0;
      uint32_t phase = 0;
      uint32_t fills = 0;
      for (uint32_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
        const Item it = item_at<BLK>(p, w);
        for (int b = 0; b < it.n_blocks && !abort_flag; ++b) {
          int tok[BLK / 64], slab[BLK / 64], boxes = 0;   // 64-token boxes that hold a token
#pragma unroll
          for (int h = 0; h < BLK / 64; ++h) {
            tok[h] = it.t_begin + b * BLK + 64 * h;
            slab[h] = 0;
            if (b * BLK + 64 * h >= it.tokens) continue;
            boxes = h + 1;
            if (p.blocks) {   // a page holds whole boxes
              const int pg = tok[h] / p.page;
              tok[h] -= pg * p.page;
              slab[h] = p.blocks[pg];
              if (slab[h] < 0 || slab[h] >= p.n_blocks) {
                report_error(DK_ERR_DEVICE_CHECK, kDetPage);
                slab[h] = 0;
              }
            }
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (!mbar_wait(&empty[stage], phase ^ 1u, kDetEmpty, abort_flag)) break;
            uint8_t* st = ring + stage * C::STAGE;
            mbar_arrive_expect_tx(&full[stage], boxes * C::NH * C::BOX);
#pragma unroll
            for (int h = 0; h < BLK / 64; ++h)
#pragma unroll
              for (int n = 0; n < C::NH; ++n)
                if (h < boxes)
                  tma_load_4d(st + n * C::HALF + h * C::BOX, kv ? &maps.v : &maps.k, &full[stage], n * 64, tok[h], it.kvh,
                              slab[h]);
            ++fills;
            if (++stage == C::STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      // every copy has landed before the CTA may end
      bool drain = false;
      for (uint32_t f = (fills > C::STAGES ? fills - C::STAGES : 0); f < fills; ++f)
        mbar_wait(&full[f % C::STAGES], static_cast<uint32_t>((f / C::STAGES) & 1), kDetDrain, drain);
    } else if (warp == kSoftWarps + 1 || warp == kSoftWarps + 2) {
      // ---------------- MMA issuers, one a tile ----------------
      const int t = warp - (kSoftWarps + 1);
      constexpr uint32_t idesc_s = umma_idesc_f16(FMT, 0, 0, kRows, BLK);
      constexpr uint32_t idesc_o = umma_idesc_f16(FMT, 0, 1, kRows, C::DP);
      // descriptors of stage 0; an offset of n bytes adds n / 16
      const uint64_t k_desc = umma_sdesc(smem_u32(ring), 16, 1024, 2);
      const uint64_t v_desc = umma_sdesc(smem_u32(ring), C::HALF, 1024, 2);
      const uint64_t q_desc = umma_sdesc(smem_u32(s_q) + t * C::QTILE, 16, 1024, 2);
      const uint32_t s_col = tmem + C::S_COL + t * BLK, p_col = tmem + C::P_COL + t * (BLK / 2);
      const uint32_t o_col = tmem + C::O_COL + t * C::DP;
      const bool leader = elect_one();
      uint32_t fill = 0;                     // stages taken: K, V, K, V, ... in the order of the loads
      uint32_t qph = 0, sph = 0, pph = 0;    // q_ready, s_free, p_ready parities
      uint32_t oph = 1;                      // o_free parity (the first wait passes)
      auto wait_fill = [&](uint32_t f) {
        return warp_wait(&full[f % C::STAGES], (f / C::STAGES) & 1, kDetFull, abort_flag);
      };
      auto issue_qk = [&](uint32_t f) {      // scores from the K block of fill f
        if (leader) {
          const uint64_t kd = k_desc + static_cast<uint64_t>((f % C::STAGES) * (C::STAGE / 16));
#pragma unroll
          for (int j = 0; j < C::DP / 16; ++j)
            tc_mma_f16(s_col, q_desc + static_cast<uint64_t>(((j >> 2) * C::QHALF + (j & 3) * 32) / 16),
                       kd + static_cast<uint64_t>(((j >> 2) * C::HALF + (j & 3) * 32) / 16), idesc_s, j > 0 ? 1u : 0u);
          tc_commit(&s_full[t]);
          tc_commit(&empty[f % C::STAGES]);
        }
        __syncwarp();
      };
      for (uint32_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
        const Item it = item_at<BLK>(p, w);
        const int nb = it.n_blocks;
        const uint32_t f0 = fill;            // block b: K in fill f0 + 2 b, V in f0 + 2 b + 1
        fill += 2 * nb;
        if (t >= it.tiles) {
          // not this tile's item: its stages still need this warp's release, in order
          for (uint32_t f = f0; f != fill; ++f) {
            if (!wait_fill(f)) break;
            if (leader) mbar_arrive(&empty[f % C::STAGES]);
          }
          continue;
        }
        if (!warp_wait(&q_ready[t], qph, kDetQ, abort_flag)) break;
        qph ^= 1u;
        if (!wait_fill(f0)) break;
        tc_fence_after();
        issue_qk(f0);
        int in_chunk = 0;
        for (int b = 0; b < nb; ++b) {
          const bool more = b + 1 < nb;
          const bool fresh = in_chunk == 0;      // a new chunk overwrites the accumulator
          if (++in_chunk == p.chunk_blocks) in_chunk = 0;
          const uint32_t fv = f0 + 2 * b + 1;
          if (!wait_fill(fv) || (more && !wait_fill(fv + 1))) break;
          // the next scores, as soon as these are in registers (the last block's release is for the next item)
          if (!warp_wait(&s_free[t], sph, kDetScoresFree, abort_flag)) break;
          sph ^= 1u;
          tc_fence_after();
          if (more) issue_qk(fv + 1);
          const int valid = min(BLK, it.tokens - b * BLK);
          const int steps = (valid + 15) >> 4;   // 16-token steps of P.V that hold a token
          if (valid & 15) {
            // tokens past the prefix inside the last step: zero rows of V (whatever the cache holds
            // there must not meet their zero weights); both issuers write the same zeros
            uint8_t* vb = ring + (fv % C::STAGES) * C::STAGE;
            const int rows = steps * 16 - valid;
            for (int e = lane; e < rows * C::NH * 8; e += 32) {
              const int r = valid + e / (C::NH * 8), c = e % (C::NH * 8);
              *reinterpret_cast<uint4*>(vb + (c >> 3) * C::HALF + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (fresh) {
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
                mma_ts(o_col, p_col + j * 8, vd + static_cast<uint64_t>(j * (2048 / 16)), idesc_o, (fresh && j == 0) ? 0u : 1u);
            tc_commit(&o_full[t]);
            tc_commit(&empty[fv % C::STAGES]);
          }
          __syncwarp();
        }
      }
      // all issued MMAs are complete before TMEM is freed
      if (leader) tc_commit(&done[t]);
      __syncwarp();
      bool fin = false;
      warp_wait(&done[t], 0, kDetDone, fin);
    }
  } else {
    // ---------------- softmax: one row a thread ----------------
    reg_inc<kSoftRegs>();
    const int t = warp >> 2;                    // tile of the item
    const int r = threadIdx.x & 127;            // row of the tile
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_t = tmem + lane_base + C::O_COL + t * C::DP;
    const uint32_t r_t = tmem + lane_base + C::R_COL + t * (D - C::RC);
    const uint32_t s_t = tmem + lane_base + C::S_COL + t * BLK, p_t = tmem + lane_base + C::P_COL + t * (BLK / 2);
    uint32_t sph = 0;                           // s_full parity
    uint32_t tph = t ^ 1;                       // turn parity (tile 0 goes first)
    uint32_t ocnt = 0;                          // blocks of this tile whose weights are handed over
    uint32_t oseen = 0;                         // of them, those whose P.V this warp has waited for
    // All P.V so far are done.  Each warp takes every phase of o_full once and in order: a block's weights
    // go out only after the previous P.V has been seen, so the barrier is never two phases ahead, where its
    // parity would say nothing.  The fence orders what the warp does to TMEM next (the weights it overwrites
    // are the left operand that P.V has read) behind that completion.
    auto pv_done = [&]() {
      if (oseen == ocnt) return true;
      const bool ok = warp_wait(&o_full[t], oseen & 1, kDetOut, abort_flag);
      tc_fence_after();
      oseen = ocnt;
      return ok;
    };
    // The tile's query rows into the swizzled K-major operand tile, asynchronously: neighbouring threads
    // take neighbouring chunks of a row ...
    const int tt = threadIdx.x & 127;
    constexpr int CPR = C::DP / 8;              // 16-byte chunks a row
    constexpr int QN = kRows * CPR / 128;       // chunks a thread
    auto q_at = [&](int i) {
      const int e = i * 128 + tt, row = e / CPR, c = e % CPR;
      return s_q + t * C::QTILE + (c >> 3) * C::QHALF + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    };
    auto fetch_q = [&](const Item& it) {
#pragma unroll 4
      for (int i = 0; i < QN; ++i) {
        const int e = i * 128 + tt, c = e % CPR;
        const uint32_t mrow = (it.pair * 2 + t) * kRows + e / CPR;
        const bool valid = mrow < static_cast<uint32_t>(p.rg) && c < D / 8;
        const uint32_t row = valid ? div_by(mrow, p.group) : 0, gh = valid ? mrow - row * p.G : 0;
        own::cp_async16(smem_u32(q_at(i)), static_cast<const T*>(p.q) + row * p.q_sr + (it.kvh * p.G + gh) * p.q_sh +
                                               (valid ? c * 8 : 0), valid);
      }
    };
    // ... and, once there, handed to the tensor cores.
    auto q_here = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (p.flip | p.zero) {
#pragma unroll 1
        for (int i = 0; i < QN; ++i) {
          uint4* at = reinterpret_cast<uint4*>(q_at(i));
          uint4 v = *at;
          v.x ^= p.flip;
          v.y ^= p.flip;
          v.z ^= p.flip;
          v.w ^= p.flip;
          *at = p.zero ? times_zero<T>(v) : v;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&q_ready[t]);
    };
    bool q_loaded = false;
    for (uint32_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
      const Item it = item_at<BLK>(p, w);
      if (t >= it.tiles) continue;
      const int m0 = (it.pair * 2 + t) * kRows;   // first row of the tile
      const bool warp_live = m0 + (warp & 3) * 32 < p.rg;
      if (!q_loaded) {   // the CTA's first item with this tile; later ones are fetched ahead
        fetch_q(it);
        q_here();
      }
      q_loaded = false;
      float run_m = -INFINITY, run_l = 0.0f;
      float m = -INFINITY, l = 0.0f;
      int in_chunk = 0;
      for (int b = 0; b < it.n_blocks; ++b) {
        const bool first = in_chunk == 0;
        if (++in_chunk == p.chunk_blocks) in_chunk = 0;
        const int valid = min(BLK, it.tokens - b * BLK);
        if (!warp_wait(&s_full[t], sph, kDetScores, abort_flag)) break;
        sph ^= 1u;
        tc_fence_after();
        const bool last = b + 1 == it.n_blocks;
        if (last) {   // all scores of this item are formed: q's place is free for the next one with this tile
          for (uint32_t wn = w + gridDim.x; wn < n_items && !q_loaded; wn += gridDim.x) {
            const Item next = item_at<BLK>(p, wn);
            if (t < next.tiles) {
              fetch_q(next);
              q_loaded = true;
            }
          }
        }
        if (warp_live) {
          constexpr int NR = BLK / 32;
          float s[NR][32];
#pragma unroll
          for (int c = 0; c < NR; ++c) tmem_ld_32x32b_x32(s_t + c * 32, s[c]);
          tmem_ld_wait();
          tc_fence_before();
          mbar_arrive(&s_free[t]);
          if (valid < BLK) {
#pragma unroll
            for (int c = 0; c < NR; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) s[c][i] = (c * 32 + i < valid) ? s[c][i] : -INFINITY;
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
          } else if (mx > m + kLazy) {   // m = -inf: any finite maximum is above it
            alpha = exp2_hw(__fsub_rn(m, mx));
            m = mx;
          }
          if (!first && __any_sync(0xffffffffu, alpha != 1.0f)) {
            // rescale the accumulator once the previous block's P.V is done
            if (!pv_done()) break;
#pragma unroll 1
            for (int c = 0; c < C::DP / 16; ++c) {
              uint32_t o[16];
              tmem_ld_x16(o_t + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__fmul_rn(__uint_as_float(o[i]), alpha));
              tmem_st_x16(o_t + c * 16, o);
            }
            l = __fmul_rn(l, alpha);
          }
          // the last block's P.V has read its weights (long since); no wait below, so that the chunks overlap
          if (!pv_done()) break;
          // The two tiles' warps of a scheduler take turns on its exponential unit, a warp's first half beside the
          // other's second: left alone they fall into step, share it, and leave it idle together (6776 rows of 16
          // heads of 64 behind 4096 tokens: 267 us; taken whole, 240 us; so, 232 us).
          if (it.tiles == 2) {
            if (!warp_wait(&turn[warp], tph, kDetTurn, abort_flag)) break;
            tph ^= 1u;
          }
          const float neg = (m == -INFINITY) ? 0.0f : -m;
          const float2 c2 = make_float2(p.c, p.c), n2 = make_float2(neg, neg);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int c = 0; c < NR; ++c) {
            uint32_t pk[16];
            if (c == NR / 2) arrive_if(&turn[warp ^ 4], it.tiles == 2 && lane == 0);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float2 e = fma2(make_float2(s[c][i], s[c][i + 1]), c2, n2);
              e.x = exp2_hw(e.x);
              e.y = exp2_hw(e.y);
              sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
              pk[i >> 1] = pack2<T>(e.x, e.y);
            }
            tmem_st_x16(p_t + c * 16, pk);
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
        tc_fence_before();
        mbar_arrive(&p_ready[t]);
        ++ocnt;
        if (q_loaded) q_here();
        if (in_chunk == 0 || last) {
          // the chunk's state joins the run's, which leaves with the last chunk
          if (!pv_done()) break;
          if (warp_live) {
            const bool head = b < p.chunk_blocks;   // the run's first chunk
            float wa = 0.0f, wb = 1.0f;
            if (head) {
              run_m = m;
              run_l = l;
            } else {
              run_m = join_weights(run_m, m, wa, wb);
              run_l = join(run_l, wa, l, wb);
            }
            const bool valid_row = m0 + r < p.rg;
            const int n = it.kvh * p.rg + m0 + r;   // state row
            if (last && valid_row)
              *reinterpret_cast<float2*>(p.st_ml + 2 * (it.run * p.st_rows + n)) = make_float2(run_m, run_l);
            float4* dst = reinterpret_cast<float4*>(p.st_o) + static_cast<int64_t>(it.run) * (D / 4) * p.st_rows + n;
            float4* run = s_run + t * (C::RC / 4) * kRows + r;   // this row's joined chunks
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld_32x32b_x32(o_t + c * 32, o);
              tmem_ld_wait();
              if (C::GROUPED && c * 32 >= C::RC) {   // columns joined in TMEM
                if (!head) {
                  float u[32];
                  tmem_ld_32x32b_x32(r_t, u);
                  tmem_ld_wait();
#pragma unroll
                  for (int i = 0; i < 32; ++i) o[i] = join(u[i], wa, o[i], wb);
                }
                if (!last) {
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    uint32_t w16[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w16[i] = __float_as_uint(o[16 * h + i]);
                    tmem_st_x16(r_t + 16 * h, w16);
                  }
                  tmem_st_wait();
                } else if (valid_row) {
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    dst[i * p.st_rows] = make_float4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
                }
                continue;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float4 v = make_float4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
                if (C::GROUPED && !head) {
                  const float4 u = *run;
                  v = make_float4(join(u.x, wa, v.x, wb), join(u.y, wa, v.y, wb), join(u.z, wa, v.z, wb),
                                  join(u.w, wa, v.w, wb));
                }
                if (C::GROUPED && !last) {
                  *run = v;
                } else if (valid_row) {
                  *dst = v;
                }
                run += kRows;
                dst += p.st_rows;
              }
            }
          }
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

// out[row, head] = O / l of the joined states: the prefix's runs (per_group of them at a time), then
// the row's own tokens.  A CTA takes 32 state rows, a lane each; its warps take four columns each
// (one coalesced load a state), and the outputs go through shared memory so that a head's row leaves
// whole.
struct CombineParams {
  const float* st_o;        // [states][D / 4][st_rows][4]
  const float* st_ml;       // [states][st_rows][2]
  int n_runs, per_group;
  const int32_t* kv_lens;   // null: no row has tokens of its own
  int own_max;              // the longest length a row may have
  const int32_t* tiles;     // the row tiles, null: every row is its own
  int32_t n_tiles, n_rows, n_seq;
  int report;               // a malformed tile is reported here (own_kernel does where it runs)
  int64_t st_rows, rg;      // hkv * rows * G, rows * G
  int G;
  Divisor31 group;          // by G
  void* out;
  int64_t o_sr, o_sh;
};

// Q: column quads a thread; UN: states a batch (the next batch is in flight while one is joined).  Many CTAs
// keep memory busy with wide threads (4, 2), few with deep ones (1, 8).
template <int D, int Q>
struct CombineCfg {
  static constexpr int WARPS = Q == 1 ? 8 : D / 4 / Q;
  static constexpr int COLS = WARPS * Q * 4;   // columns a CTA takes of its 32 state rows
};

template <typename T, int D, int Q, int UN>
__global__ void __launch_bounds__(CombineCfg<D, Q>::WARPS * 32) combine_kernel(const CombineParams p) {
  using C = CombineCfg<D, Q>;
  __shared__ __align__(16) T s_out[32][C::COLS + 2];
  __shared__ uint32_t s_covered;   // which of the 32 state rows are written
  if (threadIdx.x == 0) s_covered = 0u;
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const bool live = n < p.st_rows;
  const int quad = static_cast<int>(blockIdx.y) * (C::COLS / 4) + warp * Q;
  const uint32_t rg = static_cast<uint32_t>(p.rg);
  const float4* src = reinterpret_cast<const float4*>(p.st_o) + static_cast<int64_t>(quad) * p.st_rows + n;
  const float2* mls = reinterpret_cast<const float2*>(p.st_ml) + n;
  const int64_t state = p.st_rows * (D / 4);
  float2 ml[2][UN];
  float4 o[2][UN][Q];
  auto fetch = [&](int buf, int s0, int begin, int end) {   // states s0 .. s0 + UN - 1 that lie in [begin, end)
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s0 + u >= begin && s0 + u < end) {
        ml[buf][u] = __ldcg(mls + (s0 + u) * p.st_rows);
#pragma unroll
        for (int i = 0; i < Q; ++i) o[buf][u][i] = __ldcg(src + (s0 + u) * state + i * p.st_rows);
      }
    }
  };
  const int runs = live ? p.n_runs : 0;
  fetch(0, 0, 0, runs);        // the prefix's states do not wait for the row's length
  // A row of a tile with a length outside the cache has no own states (own_kernel has reported it and left the
  // whole tile out) and keeps what `out` holds.
  int n_own = 0;
  bool good = true;
  if (live && p.kv_lens) {
    const uint32_t mrow = static_cast<uint32_t>(n) % rg;
    const int len = p.kv_lens[div_by(mrow, p.group)];
    good = len >= 0 && len <= p.own_max;
    n_own = good ? (len + own::kSplit - 1) / own::kSplit : 0;
  }
  const int total = runs + n_own;
  fetch(0, 0, runs, total);
  if (!p.tiles) {
    const uint32_t mine = __ballot_sync(0xffffffffu, good);
    if (threadIdx.x == 0) s_covered = mine;
  } else {
    // so does a row that no tile covers
    __syncthreads();
    const int row = live ? static_cast<int>(div_by(static_cast<uint32_t>(n) % rg, p.group)) : -1;
    const int low = __reduce_min_sync(0xffffffffu, live ? row : p.n_rows), high = __reduce_max_sync(0xffffffffu, row);
    bool covered = false;
    for (int t0 = warp * 32; t0 < p.n_tiles; t0 += C::WARPS * 32) {
      const int t = t0 + lane;
      int r0 = 0, nr = 0;
      if (t < p.n_tiles) {
        r0 = p.tiles[3 * static_cast<int64_t>(t)];
        nr = p.tiles[3 * static_cast<int64_t>(t) + 1];
        const int seq = p.tiles[3 * static_cast<int64_t>(t) + 2];
        if (!own::tile_fits(r0, nr, seq, p.G, own::kRows, p.n_rows, p.n_seq)) {
          if (p.report && nr != 0 && blockIdx.x == 0 && blockIdx.y == 0) report_error(DK_ERR_DEVICE_CHECK, own::kDetTile);
          nr = 0;
        }
      }
      uint32_t hits = __ballot_sync(0xffffffffu, nr > 0 && r0 <= high && r0 + nr > low);
      while (hits) {
        const int src = __ffs(hits) - 1;
        hits &= hits - 1;
        const int a = __shfl_sync(0xffffffffu, r0, src), c = __shfl_sync(0xffffffffu, nr, src);
        const int len = p.kv_lens && lane < c ? p.kv_lens[a + lane] : 0;
        if (__any_sync(0xffffffffu, len < 0 || len > p.own_max)) continue;
        covered |= row >= a && row < a + c;
      }
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, covered);
    if (lane == 0 && mine) atomicOr(&s_covered, mine);
  }
  float tm = -INFINITY, tl = 0.0f;          // the groups joined so far
  float gm = -INFINITY, gl = 0.0f;          // the open group
  float4 to[Q], go[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) to[i] = go[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  int in_group = 0;
  for (int s0 = 0; s0 < total; s0 += 2 * UN) {
#pragma unroll
    for (int buf = 0; buf < 2; ++buf) {
      fetch(buf ^ 1, s0 + (buf + 1) * UN, 0, total);
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int s = s0 + buf * UN + u;
        if (s < total) {
          float a = 0.0f, b = 1.0f;
          const bool head = in_group == 0;
          if (head) {
            gm = ml[buf][u].x;
            gl = ml[buf][u].y;
          } else {
            gm = join_weights(gm, ml[buf][u].x, a, b);
            gl = join(gl, a, ml[buf][u].y, b);
          }
#pragma unroll
          for (int i = 0; i < Q; ++i) go[i] = head ? o[buf][u][i] : join4(go[i], a, o[buf][u][i], b);
          ++in_group;
          if (s < p.n_runs ? in_group == p.per_group || s + 1 == p.n_runs : s + 1 == total) {
            in_group = 0;
            const bool only = s < p.per_group && s < p.n_runs;   // the first group
            if (only) {
              tm = gm;
              tl = gl;
            } else {
              tm = join_weights(tm, gm, a, b);
              tl = join(tl, a, gl, b);
            }
#pragma unroll
            for (int i = 0; i < Q; ++i) to[i] = only ? go[i] : join4(to[i], a, go[i], b);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    T* d = &s_out[lane][(warp * Q + i) * 4];
    *reinterpret_cast<uint32_t*>(d) = pack2<T>(__fdiv_rn(to[i].x, tl), __fdiv_rn(to[i].y, tl));
    *reinterpret_cast<uint32_t*>(d + 2) = pack2<T>(__fdiv_rn(to[i].z, tl), __fdiv_rn(to[i].w, tl));
  }
  __syncthreads();
  T* out = static_cast<T*>(p.out) + blockIdx.y * C::COLS + lane;
#pragma unroll
  for (int k = warp; k < 32; k += C::WARPS) {
    const uint32_t nk = blockIdx.x * 32u + k;
    if (nk < p.st_rows && (s_covered >> k & 1u)) {
      const uint32_t kh = nk / rg, mk = nk - kh * rg, rk = div_by(mk, p.group);
      T* dst = out + rk * p.o_sr + (kh * p.G + mk - rk * p.G) * p.o_sh;
#pragma unroll
      for (int d = 0; d < C::COLS; d += 32) dst[d] = s_out[k][lane + d];
    }
  }
}

}  // namespace prefix
}  // namespace dk
