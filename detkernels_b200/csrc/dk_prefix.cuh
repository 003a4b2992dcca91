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
//   * Inside a chunk, blocks of 128 tokens in order: S from tcgen05.mma (f32 accumulation over D in
//     16-deep steps), a reference maximum m that is raised only when a block's maximum exceeds it
//     by more than 8 (a factor 256, so the weights stay in range of either 16-bit type), weights
//     2^(S c - m) rounded to the input type for P.V as the left operand of a second tcgen05.mma in
//     TMEM, l summed in f32 from the unrounded weights in a fixed order.
//   * The chunks' states are joined in order inside groups of kGroup chunks (head_dim <= 64 only),
//     the groups' states in order, and the states of the row's own tokens last.
// No step looks at another row, so a row's bits do not depend on the batch.
//
// Work: an item is (up to two tiles of 128 rows, KV head, run of tokens), one persistent CTA per SM.
// Warp 8 streams K and V blocks with TMA, warp 9 issues the MMAs, two warpgroups hold one row a
// thread and do the softmax.  The two tiles of an item share K and V and alternate on the tensor
// cores; an item of one tile alternates two score buffers instead.  A run is a whole group, whose
// chunks are joined in TMEM (which has room for that beside two 64-wide accumulators, not 128-wide
// ones), or, when that leaves SMs idle, one chunk, whose state combine_kernel joins; both give the
// same bits.
#pragma once

#include "dk_common.cuh"
#include "dk_own.cuh"

namespace dk {
namespace prefix {

using own::exp2_hw;
using own::join;
using own::join_weights;
using own::pack2;

constexpr int kBlock = 128;      // tokens a block
constexpr int kRows = 128;       // rows a tile
constexpr int kSoftThreads = 256;
constexpr int kThreads = 384;    // two softmax warpgroups; TMA, MMA and two idle warps
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
  kDetPage = 0x62a,   // a prefix block id outside the pool
};

// Chunks a group.
__host__ __device__ constexpr int group_chunks(int head_dim) { return head_dim <= 64 ? 8 : 1; }

// Tokens a chunk: a function of the prefix length and head_dim alone.  Short chunks give a small
// batch enough items to fill the SMs; every chunk of a 128-wide head costs each row a 512-byte state
// through memory, so those are longer.
__host__ __device__ inline int64_t chunk_tokens(int64_t prefix_len, int head_dim) {
  if (head_dim <= 64) return 512 * ((prefix_len + 16383) / 16384);
  if (prefix_len <= 4096) return 512;
  if (prefix_len <= 16384) return 1024;
  return ((prefix_len + 15) / 16 + kBlock - 1) / kBlock * kBlock;
}

struct Params {
  const void* q;
  int64_t q_sr, q_sh;
  int32_t hq, hkv, G;
  int64_t rg;             // rows * G
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
  float* st_o;            // [n_runs][rows][hq][D]
  float* st_ml;           // [n_runs][rows][hq][2]
  int64_t st_rows;        // rows * hq
};

struct Maps {
  CUtensorMap k, v;       // boxes of 64 elements x 64 tokens
};

template <int D>
struct Cfg {
  static constexpr int DP = D < 64 ? 64 : D;      // columns in shared memory and TMEM (D = 32: zero filled)
  static constexpr int NH = DP / 64;              // 64-element halves
  static constexpr int BOX = 64 * 128;            // bytes of a 64-token box
  static constexpr int HALF = 2 * BOX;            // 128 tokens x 64 elements
  static constexpr int STAGE = NH * HALF;         // a K or V block
  static constexpr int STAGES = D == 128 ? 4 : 8;
  static constexpr int QTILE = NH * HALF;
  static constexpr int TPAD = 20;                 // floats a row of a warp's transpose buffer (16 used)
  static constexpr int TBUF = 32 * TPAD * 4;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * QTILE + 8 * TBUF + 512;
  static constexpr uint32_t S_COL = 0;            // two score buffers of 128 columns
  static constexpr uint32_t O_COL = 256;          // two accumulators of DP columns
  static constexpr bool GROUPED = group_chunks(D) > 1;
  static constexpr uint32_t R_COL = 384;          // grouped: the joined chunks of either tile, DP columns each
};

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
__device__ __forceinline__ Item item_at(const Params& p, int64_t w) {
  Item it;
  it.pair = static_cast<int>(w % p.n_pairs);
  const int64_t r = w / p.n_pairs;
  it.kvh = static_cast<int>(r % p.hkv);
  it.run = static_cast<int>(r / p.hkv);
  it.tiles = (static_cast<int64_t>(it.pair) * 2 + 1) * kRows < p.rg ? 2 : 1;
  it.t_begin = it.run * p.run_blocks * kBlock;
  it.tokens = min(p.prefix_len - it.t_begin, p.run_blocks * kBlock);
  it.n_blocks = (it.tokens + kBlock - 1) / kBlock;
  return it;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) prefix_kernel(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<D>;
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = base;
  uint8_t* s_q = ring + C::STAGES * C::STAGE;
  float* s_t = reinterpret_cast<float*>(s_q + 2 * C::QTILE);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(s_t) + 8 * C::TBUF);
  uint64_t* empty = full + C::STAGES;
  // score barriers: 0 and 1 by tile, 2 the second buffer of a one-tile item (tile 1's columns); each
  // has one warpgroup that waits for every phase of it in order
  uint64_t* s_full = empty + C::STAGES;   // [3]
  uint64_t* p_ready = s_full + 3;         // [3]
  uint64_t* o_full = p_ready + 3;         // [2] by tile: P.V of a block done
  uint64_t* o_free = o_full + 2;          // [2] by tile: the accumulator has been read
  uint64_t* q_ready = o_free + 2;         // [2] by tile
  uint64_t* done = q_ready + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 128);
      mbar_init(&q_ready[t], 128);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (warp == 9) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();

  const int64_t n_items = static_cast<int64_t>(p.n_pairs) * p.hkv * p.n_runs;
  bool abort_flag = false;

  if (warp >= 8) {
    reg_dec<kIoRegs>();
    if (warp == 8 && lane == 0) {
      // ---------------- TMA producer: K block, V block, K block, ... ----------------
      int stage = 0;
      uint32_t phase = 0;
      int64_t fills = 0;
      for (int64_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
        const Item it = item_at(p, w);
        for (int b = 0; b < it.n_blocks && !abort_flag; ++b) {
          const int t0 = it.t_begin + b * kBlock;
          const int halves = (it.tokens - b * kBlock > 64) ? 2 : 1;
          int tok[2], slab[2];
          for (int h = 0; h < halves; ++h) {
            tok[h] = t0 + 64 * h;
            slab[h] = 0;
            if (p.blocks) {
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
            mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(halves * C::NH * C::BOX));
            for (int h = 0; h < halves; ++h)
              for (int n = 0; n < C::NH; ++n)
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
      for (int64_t f = (fills > C::STAGES ? fills - C::STAGES : 0); f < fills; ++f)
        mbar_wait(&full[f % C::STAGES], static_cast<uint32_t>((f / C::STAGES) & 1), kDetDrain, drain);
    } else if (warp == 9) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc_s = umma_idesc_f16(FMT, 0, 0, kRows, kBlock);
      constexpr uint32_t idesc_o = umma_idesc_f16(FMT, 0, 1, kRows, C::DP);
      const uint32_t ring_a = smem_u32(ring), q_a = smem_u32(s_q);
      int64_t used = 0;                      // stages taken so far (K, V, K, V, ...)
      uint32_t pc[3] = {0, 0, 0};            // p_ready phases seen
      uint32_t qc[2] = {0, 0}, oc[2] = {0, 0};
      auto wait_stage = [&](int64_t f) {
        return warp_wait(&full[f % C::STAGES], static_cast<uint32_t>((f / C::STAGES) & 1), kDetFull, abort_flag);
      };
      // scores of tile t, block with K in stage f, by score barrier sb
      auto issue_qk = [&](int t, int sb, int64_t f) {
        if (lane == 0) {
          const uint32_t kb = ring_a + static_cast<uint32_t>(f % C::STAGES) * C::STAGE;
          const uint32_t qb = q_a + t * C::QTILE;
#pragma unroll
          for (int j = 0; j < C::DP / 16; ++j) {
            const uint32_t off = (j >> 2) * C::HALF + (j & 3) * 32;
            tc_mma_f16(tmem + C::S_COL + (sb ? 128 : 0), umma_sdesc(qb + off, 16, 1024, 2), umma_sdesc(kb + off, 16, 1024, 2),
                       idesc_s, j > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[sb]);
        }
        __syncwarp();
      };
      for (int64_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
        const Item it = item_at(p, w);
        const int nb = it.n_blocks;
        for (int t = 0; t < it.tiles; ++t) {
          if (!warp_wait(&q_ready[t], qc[t] & 1, kDetQ, abort_flag)) break;
          ++qc[t];
        }
        if (abort_flag) break;
        const int64_t f0 = used;   // block b: K in fill f0 + 2b, V in f0 + 2b + 1
        used += 2 * static_cast<int64_t>(nb);
        tc_fence_after();
        if (!wait_stage(f0)) break;
        for (int t = 0; t < it.tiles; ++t) issue_qk(t, t, f0);
        if (lane == 0) tc_commit(&empty[f0 % C::STAGES]);
        for (int b = 0; b < nb && !abort_flag; ++b) {
          const bool more = b + 1 < nb;
          const int64_t fk = f0 + 2 * (b + 1), fv = f0 + 2 * b + 1;
          if (it.tiles == 1 && more) {   // the next block's scores go to the other buffer
            if (!wait_stage(fk)) break;
            issue_qk(0, (b + 1) & 1 ? 2 : 0, fk);
            if (lane == 0) tc_commit(&empty[fk % C::STAGES]);
          }
          const int valid = min(kBlock, it.tokens - b * kBlock);
          const int steps = (valid + 15) >> 4;   // 16-token steps of P.V that hold a token
          for (int t = 0; t < it.tiles; ++t) {
            const int sb = it.tiles == 2 ? t : (b & 1 ? 2 : 0);
            if (!warp_wait(&p_ready[sb], pc[sb] & 1, kDetProbs, abort_flag)) break;
            ++pc[sb];
            if (b % p.chunk_blocks == 0) {   // a new chunk overwrites the accumulator
              if (!warp_wait(&o_free[t], (oc[t] & 1) ^ 1u, kDetOutFree, abort_flag)) break;
              ++oc[t];
            }
            if (t == 0) {
              if (!wait_stage(fv)) break;
              if (valid & 15) {
                // tokens past the prefix inside the last step: zero rows of V (whatever the cache
                // holds there must not meet their zero weights)
                uint8_t* vb = ring + (fv % C::STAGES) * C::STAGE;
                const int rows = steps * 16 - valid;
                for (int e = lane; e < rows * C::NH * 8; e += 32) {
                  const int r = valid + e / (C::NH * 8), c = e % (C::NH * 8);
                  *reinterpret_cast<uint4*>(vb + (c >> 3) * C::HALF + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            tc_fence_after();
            if (lane == 0) {
              const uint32_t vb = ring_a + static_cast<uint32_t>(fv % C::STAGES) * C::STAGE;
              for (int j = 0; j < steps; ++j)
                mma_ts(tmem + C::O_COL + t * C::DP, tmem + C::S_COL + (sb ? 128 : 0) + j * 8,
                       umma_sdesc(vb + j * 2048, C::HALF, 1024, 2), idesc_o,
                       (b % p.chunk_blocks != 0 || j > 0) ? 1u : 0u);
              tc_commit(&o_full[t]);
              if (t + 1 == it.tiles) tc_commit(&empty[fv % C::STAGES]);
            }
            __syncwarp();
            if (it.tiles == 2 && more) {
              if (t == 0 && !wait_stage(fk)) break;
              issue_qk(t, t, fk);
              if (t == 1 && lane == 0) tc_commit(&empty[fk % C::STAGES]);
            }
          }
        }
      }
      // all issued MMAs are complete before TMEM is freed
      if (lane == 0) tc_commit(done);
      __syncwarp();
      bool fin = false;
      warp_wait(done, 0, kDetDone, fin);
    }
  } else {
    // ---------------- softmax: one row a thread ----------------
    reg_inc<kSoftRegs>();
    const int t = warp >> 2;                    // tile of the item
    const int r = threadIdx.x & 127;            // row of the tile
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_t = tmem + lane_base + C::O_COL + t * C::DP;
    float* tb = s_t + warp * (C::TBUF / 4);
    uint32_t sc[2] = {0, 0};                    // score phases consumed: own barrier, second buffer
    uint32_t ocnt = 0;                          // P.V completions of this tile so far
    for (int64_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
      const Item it = item_at(p, w);
      if (t >= it.tiles) continue;
      const int64_t m0 = (static_cast<int64_t>(it.pair) * 2 + t) * kRows;   // first row of the tile
      const int64_t mrow = m0 + r;
      const bool valid_row = mrow < p.rg;
      const bool warp_live = m0 + (warp & 3) * 32 < p.rg;
      {
        // this row's query vector into the swizzled K-major operand tile
        uint8_t* qt = s_q + t * C::QTILE + r * 128;
        const int64_t row = mrow / p.G;
        const T* src = static_cast<const T*>(p.q) + row * p.q_sr + (it.kvh * p.G + (mrow - row * p.G)) * p.q_sh;
#pragma unroll
        for (int c = 0; c < C::DP / 8; ++c) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (valid_row && c < D / 8) {
            v = *reinterpret_cast<const uint4*>(src + c * 8);
            v.x ^= p.flip;
            v.y ^= p.flip;
            v.z ^= p.flip;
            v.w ^= p.flip;
            if (p.zero) v = times_zero<T>(v);
          }
          *reinterpret_cast<uint4*>(qt + (c >> 3) * C::HALF + (((c & 7) ^ (r & 7)) << 4)) = v;
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_ready[t]);
      }
      float run_m = -INFINITY, run_l = 0.0f;
      float m = -INFINITY, l = 0.0f;
      for (int b = 0; b < it.n_blocks; ++b) {
        const int second = it.tiles == 1 ? (b & 1) : 0;   // a one-tile item's second buffer
        const int sb = second ? 2 : t;
        const bool first = b % p.chunk_blocks == 0;
        const int valid = min(kBlock, it.tokens - b * kBlock);
        if (!warp_wait(&s_full[sb], sc[second] & 1, kDetScores, abort_flag)) break;
        ++sc[second];
        tc_fence_after();
        if (warp_live) {
          const uint32_t s_t0 = tmem + lane_base + C::S_COL + (sb ? 128 : 0);
          float s[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_t0 + c * 32, s[c]);
          tmem_ld_wait();
          if (valid < kBlock) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) s[c][i] = (c * 32 + i < valid) ? s[c][i] : -INFINITY;
          }
          float mx4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            mx4[c] = fmaxf(s[c][0], s[c][1]);
#pragma unroll
            for (int i = 2; i < 32; i += 2) mx4[c] = fmaxf(mx4[c], fmaxf(s[c][i], s[c][i + 1]));
          }
          const float mx = __fmul_rn(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), p.c);
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
            if (!warp_wait(&o_full[t], (ocnt - 1) & 1, kDetOut, abort_flag)) break;
            tc_fence_after();
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
          const float neg = (m == -INFINITY) ? 0.0f : -m;
          const float2 c2 = make_float2(p.c, p.c), n2 = make_float2(neg, neg);
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float2 e = fma2(make_float2(s[c][i], s[c][i + 1]), c2, n2);
              e.x = exp2_hw(e.x);
              e.y = exp2_hw(e.y);
              sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
              pk[i >> 1] = pack2<T>(e.x, e.y);
            }
            tmem_st_x16(s_t0 + c * 16, pk);
          }
          const float2 ps = add2(sum[0], sum[1]);
          l = __fadd_rn(l, __fadd_rn(ps.x, ps.y));
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(&p_ready[sb]);
        ++ocnt;
        const bool last = b + 1 == it.n_blocks;
        if ((b + 1) % p.chunk_blocks == 0 || last) {
          // the chunk's state joins the run's, which leaves with the last chunk
          if (!warp_wait(&o_full[t], (ocnt - 1) & 1, kDetOut, abort_flag)) break;
          tc_fence_after();
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
            const int64_t st0 = static_cast<int64_t>(it.run) * p.st_rows;
            int64_t dst[4];
            if (last) {
              if (valid_row) {
                const int64_t row = mrow / p.G;
                const int64_t idx = st0 + row * p.hq + it.kvh * p.G + (mrow - row * p.G);
                *reinterpret_cast<float2*>(p.st_ml + 2 * idx) = make_float2(run_m, run_l);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) {   // rows this lane writes, 16 bytes of each a piece
                const int64_t mm = m0 + (warp & 3) * 32 + j * 8 + (lane >> 2);
                const int64_t row = mm / p.G;
                dst[j] = mm < p.rg ? (st0 + row * p.hq + it.kvh * p.G + (mm - row * p.G)) * D + (lane & 3) * 4 : -1;
              }
            }
            const uint32_t r_t = tmem + lane_base + C::R_COL + t * C::DP;
#pragma unroll 2
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16], r[16];
              tmem_ld_x16(o_t + c * 16, o);
              if (C::GROUPED && !head) tmem_ld_x16(r_t + c * 16, r);
              tmem_ld_wait();
              if (C::GROUPED && !head) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  o[i] = __float_as_uint(join(__uint_as_float(r[i]), wa, __uint_as_float(o[i]), wb));
              }
              if (C::GROUPED && !last) {
                tmem_st_x16(r_t + c * 16, o);
              } else {
                // transposed, so that a row's 64 bytes leave together
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  *reinterpret_cast<uint4*>(tb + lane * C::TPAD + i * 4) =
                      make_uint4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 v = *reinterpret_cast<const float4*>(tb + (j * 8 + (lane >> 2)) * C::TPAD + (lane & 3) * 4);
                  if (dst[j] >= 0) *reinterpret_cast<float4*>(p.st_o + dst[j] + c * 16) = v;
                }
              }
            }
            if (C::GROUPED && !last) tmem_st_wait();
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
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// out[row, head] = O / l of the joined states: the prefix's runs (per_group of them at a time), then
// the row's own tokens (own_splits states, or one where a warp joined them all).  One warp a (row,
// head), UN states in flight.
constexpr int kCombineWarps = 4;

struct CombineParams {
  const float* st_o;
  const float* st_ml;
  int n_runs, per_group;
  const int32_t* kv_lens;   // null: no row has tokens of its own
  int own_max;              // states the own tokens may have: 1 (joined already) or the split limit
  int64_t st_rows;
  int hq;
  void* out;
  int64_t o_sr, o_sh;
};

template <typename T, int D>
__global__ void __launch_bounds__(kCombineWarps * 32) combine_kernel(const CombineParams p) {
  constexpr int V = D / 32;
  constexpr int UN = 8;
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t m = static_cast<int64_t>(blockIdx.x) * kCombineWarps + (threadIdx.x >> 5);
  if (m >= p.st_rows) return;
  const int64_t row = m / p.hq;
  int n_own = 0;
  if (p.kv_lens) n_own = min(max((p.kv_lens[row] + own::kSplit - 1) / own::kSplit, 0), p.own_max);
  const int n = p.n_runs + n_own;
  float tm = -INFINITY, tl = 0.0f, to[V];   // the groups joined so far
  float gm = -INFINITY, gl = 0.0f, go[V];   // the open group
#pragma unroll
  for (int i = 0; i < V; ++i) to[i] = go[i] = 0.0f;
  for (int s0 = 0; s0 < n; s0 += UN) {
    float2 ml[UN];
    float o[UN][V];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s0 + u < n) {
        const int64_t idx = (s0 + u) * p.st_rows + m;
        ml[u] = __ldcg(reinterpret_cast<const float2*>(p.st_ml + 2 * idx));
        const float* src = p.st_o + idx * D + lane * V;
        if constexpr (V == 4) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
          o[u][0] = f.x;
          o[u][1] = f.y;
          o[u][2] = f.z;
          o[u][3] = f.w;
        } else if constexpr (V == 2) {
          const float2 f = __ldcg(reinterpret_cast<const float2*>(src));
          o[u][0] = f.x;
          o[u][1] = f.y;
        } else {
          o[u][0] = __ldcg(src);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int s = s0 + u;
      if (s < n) {
        const bool head = s < p.n_runs ? s % p.per_group == 0 : s == p.n_runs;
        const bool tail = s < p.n_runs ? (s + 1) % p.per_group == 0 || s + 1 == p.n_runs : s + 1 == n;
        float a = 0.0f, b = 1.0f;
        if (head) {
          gm = ml[u].x;
          gl = ml[u].y;
        } else {
          gm = join_weights(gm, ml[u].x, a, b);
          gl = join(gl, a, ml[u].y, b);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) go[i] = head ? o[u][i] : join(go[i], a, o[u][i], b);
        if (tail) {
          const bool only = s < p.per_group && s < p.n_runs;   // the first group
          if (only) {
            tm = gm;
            tl = gl;
          } else {
            tm = join_weights(tm, gm, a, b);
            tl = join(tl, a, gl, b);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) to[i] = only ? go[i] : join(to[i], a, go[i], b);
        }
      }
    }
  }
  T* dst = static_cast<T*>(p.out) + row * p.o_sr + (m - row * p.hq) * p.o_sh + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) dst[i] = from_f32<T>(__fdiv_rn(to[i], tl));
}

}  // namespace prefix
}  // namespace dk
