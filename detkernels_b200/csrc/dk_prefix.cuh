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
// One warp streams K and V blocks with TMA, one warp a tile issues its MMAs, and a warpgroup a tile does
// the softmax, a row a thread.  The two tiles of an item share K and V and alternate on the tensor
// cores; when there is one tile only, it alternates between two score buffers instead.  A run is a whole group, whose
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
  kDetTurn = 0x629,
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
  int32_t rg;             // rows * G
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

template <int D>
struct Cfg {
  static constexpr int DP = D < 64 ? 64 : D;      // columns in shared memory and TMEM (D = 32: zero filled)
  static constexpr int NH = DP / 64;              // 64-element halves
  static constexpr int BOX = 64 * 128;            // bytes of a 64-token box
  static constexpr int HALF = 2 * BOX;            // 128 tokens x 64 elements
  static constexpr int STAGE = NH * HALF;         // a K or V block
  static constexpr int STAGES = D == 128 ? 4 : 8;
  static constexpr int QTILE = NH * HALF;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * QTILE + 512;
  static constexpr uint32_t S_COL = 0;            // two score buffers of 128 columns
  static constexpr uint32_t O_COL = 256;          // two accumulators of DP columns
  static constexpr int FMA_OF_4 = 0;              // weights of every four whose 2^x takes the FMA pipe
  static constexpr bool GROUPED = group_chunks(D) > 1;
  static constexpr uint32_t R_COL = 384;          // grouped: the joined chunks of either tile, DP columns each
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

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x for x <= 2^20 on the FMA pipe, two at a time: x = n + f with n the nearest integer (by adding and
// taking away 1.5 * 2^23), 2^f by the degree-4 polynomial of least relative error on [-1/2, 1/2] (Remez
// exchange; 2^-18.5), times 2^n.  Below -127 the factor and so the result is 0; NaN stays NaN.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  const float2 magic = make_float2(12582912.0f, 12582912.0f), nmagic = make_float2(-12582912.0f, -12582912.0f);
  x.x = max_nan(x.x, -127.0f);
  x.y = max_nan(x.y, -127.0f);
  const float2 t = add2(x, magic);
  const float2 n = add2(t, nmagic);
  const float2 f = fma2(n, make_float2(-1.0f, -1.0f), x);
  float2 p = make_float2(0.009570102207362652f, 0.009570102207362652f);
  p = fma2(p, f, make_float2(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  const float2 s = make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                               __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u));
  return mul2(p, s);
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
__device__ __forceinline__ Item item_at(const Params& p, uint32_t w) {
  Item it;
  const uint32_t r = w / static_cast<uint32_t>(p.n_pairs);
  it.pair = static_cast<int>(w - r * p.n_pairs);
  it.run = static_cast<int>(r / static_cast<uint32_t>(p.hkv));
  it.kvh = static_cast<int>(r - it.run * static_cast<uint32_t>(p.hkv));
  it.tiles = (it.pair * 2 + 1) * kRows < p.rg ? 2 : 1;
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
  uint64_t* full = reinterpret_cast<uint64_t*>(s_q + 2 * C::QTILE);
  uint64_t* empty = full + C::STAGES;
  // score barriers: 0 and 1 by tile, 2 the second buffer of a lone tile (tile 1's columns); each
  // has one warpgroup that waits for every phase of it in order
  uint64_t* s_full = empty + C::STAGES;   // [3]
  uint64_t* p_ready = s_full + 3;         // [3]
  uint64_t* p_half = p_ready + 3;         // [3] the first 64 tokens' weights are in TMEM (p_ready: the others')
  uint64_t* o_full = p_half + 3;         // [2] by tile: P.V of a block done
  uint64_t* o_free = o_full + 2;          // [2] by tile: the accumulator has been read
  uint64_t* q_ready = o_free + 2;         // [2] by tile
  uint64_t* turn = q_ready + 2;           // [2] by tile: the other tile's issuer has issued its group
  uint64_t* done = turn + 2;              // [2]
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
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&p_half[i], 128);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&o_full[t], 1);
      mbar_init(&o_free[t], 128);
      mbar_init(&q_ready[t], 128);
      mbar_init(&turn[t], 1);
    }
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
  // At most 128 rows: tile 0 alone alternates between both score buffers.  (Not in an item whose second
  // tile is empty while others have two: the buffer is then the other issuer's.)
  const bool dbl = p.rg <= kRows;
  bool abort_flag = false;

  if (warp >= kSoftWarps) {
    reg_dec<kIoRegs>();
    if (warp == kSoftWarps && lane == 0) {
      // ---------------- TMA producer: K block, V block, K block, ... ----------------
      int stage = 0;
      uint32_t phase = 0;
      uint32_t fills = 0;
      for (uint32_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
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
      for (uint32_t f = (fills > C::STAGES ? fills - C::STAGES : 0); f < fills; ++f)
        mbar_wait(&full[f % C::STAGES], static_cast<uint32_t>((f / C::STAGES) & 1), kDetDrain, drain);
    } else if (warp == kSoftWarps + 1 || warp == kSoftWarps + 2) {
      // ---------------- MMA issuers, one a tile ----------------
      const int t = warp - (kSoftWarps + 1);
      constexpr uint32_t idesc_s = umma_idesc_f16(FMT, 0, 0, kRows, kBlock);
      constexpr uint32_t idesc_o = umma_idesc_f16(FMT, 0, 1, kRows, C::DP);
      // descriptors of stage 0; an offset of n bytes adds n / 16
      const uint64_t k_desc = umma_sdesc(smem_u32(ring), 16, 1024, 2);
      const uint64_t v_desc = umma_sdesc(smem_u32(ring), C::HALF, 1024, 2);
      const uint64_t q_desc = umma_sdesc(smem_u32(s_q) + t * C::QTILE, 16, 1024, 2);
      const uint32_t o_col = tmem + C::O_COL + t * C::DP;
      const bool leader = elect_one();
      uint32_t fill = 0;                     // stages taken: K, V, K, V, ... in the order of the loads
      uint32_t pph = 0;                      // weights parities by score barrier
      uint32_t qph = 0, oph = 1;             // q_ready, o_free parities (the first o_free wait passes)
      uint32_t tph = t ^ 1;                  // turn parity (tile 0 goes first)
      auto wait_fill = [&](uint32_t f) {
        return warp_wait(&full[f % C::STAGES], (f / C::STAGES) & 1, kDetFull, abort_flag);
      };
      // scores from the K block of fill f, by score barrier sb
      auto issue_qk = [&](int sb, uint32_t f) {
        if (leader) {
          const uint64_t kd = k_desc + static_cast<uint64_t>((f % C::STAGES) * (C::STAGE / 16));
          const uint32_t d = tmem + C::S_COL + (sb ? 128 : 0);
#pragma unroll
          for (int j = 0; j < C::DP / 16; ++j) {
            const uint64_t off = ((j >> 2) * C::HALF + (j & 3) * 32) / 16;
            tc_mma_f16(d, q_desc + off, kd + off, idesc_s, j > 0 ? 1u : 0u);
          }
          tc_commit(&s_full[sb]);
          tc_commit(&empty[f % C::STAGES]);
        }
        __syncwarp();
      };
      for (uint32_t w = blockIdx.x; w < n_items && !abort_flag; w += gridDim.x) {
        const Item it = item_at(p, w);
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
        issue_qk(t, f0);
        int in_chunk = 0;
        for (int b = 0; b < nb; ++b) {
          const bool more = b + 1 < nb;
          const bool fresh = in_chunk == 0;      // a new chunk overwrites the accumulator
          if (++in_chunk == p.chunk_blocks) in_chunk = 0;
          const uint32_t fv = f0 + 2 * b + 1;
          if (!wait_fill(fv) || (more && !wait_fill(fv + 1))) break;
          if (dbl && more) issue_qk((b + 1) & 1 ? 2 : 0, fv + 1);   // into the other buffer
          const int valid = min(kBlock, it.tokens - b * kBlock);
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
          const int sb = dbl && (b & 1) ? 2 : t;
          const uint64_t vd = v_desc + static_cast<uint64_t>((fv % C::STAGES) * (C::STAGE / 16));
          const uint32_t pt = tmem + C::S_COL + (sb ? 128 : 0);
          // the first half of the weights, then the second
          if (!warp_wait(&p_half[sb], (pph >> sb) & 1, kDetProbs, abort_flag)) break;
          if (it.tiles == 2) {
            // the two issuers take turns, so that one tile's products run under the other's softmax
            // (left alone they fall into step, and both wait for each)
            if (!warp_wait(&turn[t], tph, kDetTurn, abort_flag)) break;
            tph ^= 1u;
          }
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < steps)
                mma_ts(o_col, pt + j * 8, vd + static_cast<uint64_t>(j * (2048 / 16)), idesc_o, (fresh && j == 0) ? 0u : 1u);
          }
          __syncwarp();
          if (!warp_wait(&p_ready[sb], (pph >> sb) & 1, kDetProbs, abort_flag)) break;
          pph ^= 1u << sb;
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int j = 4; j < 8; ++j)
              if (j < steps) mma_ts(o_col, pt + j * 8, vd + static_cast<uint64_t>(j * (2048 / 16)), idesc_o, 1u);
            tc_commit(&o_full[t]);
            tc_commit(&empty[fv % C::STAGES]);
          }
          __syncwarp();
          if (!dbl && more) issue_qk(t, fv + 1);
          if (it.tiles == 2 && leader) mbar_arrive(&turn[t ^ 1]);
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
    uint32_t sc[2] = {0, 0};                    // score phases consumed: own barrier, second buffer
    uint32_t ocnt = 0;                          // P.V completions of this tile so far
    // The tile's query rows into the swizzled K-major operand tile, asynchronously: neighbouring threads
    // take neighbouring chunks of a row ...
    const int tt = threadIdx.x & 127;
    constexpr int CPR = C::DP / 8;              // 16-byte chunks a row
    constexpr int QN = kRows * CPR / 128;       // chunks a thread
    auto q_at = [&](int i) {
      const int e = i * 128 + tt, row = e / CPR, c = e % CPR;
      return s_q + t * C::QTILE + (c >> 3) * C::HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    };
    auto fetch_q = [&](const Item& it) {
#pragma unroll 4
      for (int i = 0; i < QN; ++i) {
        const int e = i * 128 + tt, c = e % CPR;
        const uint32_t mrow = (it.pair * 2 + t) * kRows + e / CPR;
        const bool valid = mrow < static_cast<uint32_t>(p.rg) && c < D / 8;
        const uint32_t row = valid ? mrow / static_cast<uint32_t>(p.G) : 0, gh = valid ? mrow - row * p.G : 0;
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
      const Item it = item_at(p, w);
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
        const int second = dbl ? (b & 1) : 0;
        const int sb = second ? 2 : t;
        const bool first = in_chunk == 0;
        if (++in_chunk == p.chunk_blocks) in_chunk = 0;
        const int valid = min(kBlock, it.tokens - b * kBlock);
        if (!warp_wait(&s_full[sb], sc[second] & 1, kDetScores, abort_flag)) break;
        ++sc[second];
        tc_fence_after();
        const bool last = b + 1 == it.n_blocks;
        if (last) {   // all scores of this item are formed: q's place is free for the next one with this tile
          for (uint32_t wn = w + gridDim.x; wn < n_items && !q_loaded; wn += gridDim.x) {
            const Item next = item_at(p, wn);
            if (t < next.tiles) {
              fetch_q(next);
              q_loaded = true;
            }
          }
        }
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
              if (((i >> 1) & 3) >= 4 - C::FMA_OF_4) {   // by column alone, so by token
                e = exp2_fma(e);
              } else {
                e.x = exp2_hw(e.x);
                e.y = exp2_hw(e.y);
              }
              sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
              pk[i >> 1] = pack2<T>(e.x, e.y);
            }
            tmem_st_x16(s_t0 + c * 16, pk);
            if (c == 1) {
              tmem_st_wait();
              tc_fence_before();
              mbar_arrive(&p_half[sb]);
            }
          }
          tmem_st_wait();
          const float2 ps = add2(sum[0], sum[1]);
          l = __fadd_rn(l, __fadd_rn(ps.x, ps.y));
        } else {
          mbar_arrive(&p_half[sb]);
        }
        tc_fence_before();
        mbar_arrive(&p_ready[sb]);
        ++ocnt;
        if (q_loaded) q_here();
        if (in_chunk == 0 || last) {
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
            const bool valid_row = m0 + r < p.rg;
            const int n = it.kvh * p.rg + m0 + r;   // state row
            if (last && valid_row)
              *reinterpret_cast<float2*>(p.st_ml + 2 * (it.run * p.st_rows + n)) = make_float2(run_m, run_l);
            float* dst = p.st_o + (static_cast<int64_t>(it.run) * (D / 4) * p.st_rows + n) * 4;
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
                if (valid_row) {
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(dst + (c * 4 + i) * p.st_rows * 4) =
                        make_uint4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
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
  int own_max;              // states the own tokens may have: 1 (joined already) or the split limit
  int64_t st_rows, rg;      // hkv * rows * G, rows * G
  int G;
  void* out;
  int64_t o_sr, o_sh;
};

constexpr int kCombineCols = 32;   // columns a CTA takes of its 32 state rows, four a warp

template <typename T, int D>
__global__ void __launch_bounds__(kCombineCols * 8) combine_kernel(const CombineParams p) {
  constexpr int UN = 8;     // states in flight
  __shared__ __align__(16) T s_out[32][kCombineCols + 2];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const bool live = n < p.st_rows;
  const int quad = static_cast<int>(blockIdx.y) * (kCombineCols / 4) + warp;
  const uint32_t rg = static_cast<uint32_t>(p.rg), G = static_cast<uint32_t>(p.G);
  const uint32_t mrow = live ? static_cast<uint32_t>(n) % rg : 0;
  int n_own = 0;
  if (live && p.kv_lens) n_own = min(max((p.kv_lens[mrow / G] + own::kSplit - 1) / own::kSplit, 0), p.own_max);
  const int total = live ? p.n_runs + n_own : 0;
  const float* src = p.st_o + (static_cast<int64_t>(quad) * p.st_rows + n) * 4;
  const int64_t state = p.st_rows * D;
  float tm = -INFINITY, tl = 0.0f;          // the groups joined so far
  float gm = -INFINITY, gl = 0.0f;          // the open group
  float4 to = make_float4(0.0f, 0.0f, 0.0f, 0.0f), go = to;
  auto join4 = [](float4 v, float a, float4 vs, float b) {
    return make_float4(join(v.x, a, vs.x, b), join(v.y, a, vs.y, b), join(v.z, a, vs.z, b), join(v.w, a, vs.w, b));
  };
  int in_group = 0;
  for (int s0 = 0; s0 < total; s0 += UN) {
    float2 ml[UN];
    float4 o[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (s0 + u < total) {
        ml[u] = __ldcg(reinterpret_cast<const float2*>(p.st_ml + 2 * ((s0 + u) * p.st_rows + n)));
        o[u] = __ldcg(reinterpret_cast<const float4*>(src + (s0 + u) * state));
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int s = s0 + u;
      if (s < total) {
        float a, b;
        if (in_group == 0) {
          gm = ml[u].x;
          gl = ml[u].y;
          go = o[u];
        } else {
          gm = join_weights(gm, ml[u].x, a, b);
          gl = join(gl, a, ml[u].y, b);
          go = join4(go, a, o[u], b);
        }
        ++in_group;
        if (s < p.n_runs ? in_group == p.per_group || s + 1 == p.n_runs : s + 1 == total) {
          in_group = 0;
          if (s < p.per_group && s < p.n_runs) {   // the first group
            tm = gm;
            tl = gl;
            to = go;
          } else {
            tm = join_weights(tm, gm, a, b);
            tl = join(tl, a, gl, b);
            to = join4(to, a, go, b);
          }
        }
      }
    }
  }
  *reinterpret_cast<uint32_t*>(&s_out[lane][warp * 4]) = pack2<T>(__fdiv_rn(to.x, tl), __fdiv_rn(to.y, tl));
  *reinterpret_cast<uint32_t*>(&s_out[lane][warp * 4 + 2]) = pack2<T>(__fdiv_rn(to.z, tl), __fdiv_rn(to.w, tl));
  __syncthreads();
  T* out = static_cast<T*>(p.out) + blockIdx.y * kCombineCols + lane;
#pragma unroll
  for (int k = warp; k < 32; k += kCombineCols / 4) {
    const int64_t nk = static_cast<int64_t>(blockIdx.x) * 32 + k;
    if (nk < p.st_rows) {
      const uint32_t kh = static_cast<uint32_t>(nk) / rg, mk = static_cast<uint32_t>(nk) - kh * rg, rk = mk / G;
      out[rk * p.o_sr + (kh * G + mk - rk * G) * p.o_sh] = s_out[k][lane];
    }
  }
}

}  // namespace prefix
}  // namespace dk
