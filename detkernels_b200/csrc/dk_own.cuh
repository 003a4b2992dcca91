// A row's own tokens behind a shared prefix: split-KV decode attention that leaves softmax states.
//
// Fixed reduction structure: the row's tokens [0, len) in splits of kSplit = 64; inside a split
// steps of 32 tokens (16 for head_dim 128) in order with an online softmax (m, l, O), scores from
// mma.m16n8k16 (f32 accumulation), weights rounded to the input type for P.V (the MMA takes 16-bit operands)
// and summed as rounded, so that those of a row of few tokens still add up to one;
// split states joined in order.  Nothing depends on the batch, the tile a row sits in or the schedule.
//
// Work: a unit is (row tile of at most 16 query rows of one sequence, KV head, run of splits), one
// warp each, with no barrier wider than the warp: short sequences, which are what follows a shared
// prefix, leave many small units whose loads overlap each other.  The products are formed transposed
// (S^T = K q^T, O^T = V^T P^T: the tokens, then the head_dim, are the MMA's 16 rows and the query rows
// its 8 columns), so up to 8 query rows a tile cost half the MMAs and registers of the upright form;
// a column's bits do not depend on the others, so tiles of 16 rows (two column halves) give the same.
// K and V come through a ring of one-step stages (cp.async, zero filled past the sequence's end, so
// that whatever the cache holds there is never read); a warp's chain of dependent instructions a step bounds
// it, which longer steps shorten (256 rows of 16 heads of 64, 1-639 tokens behind 2048: 72 us against 82 in
// steps of 16) until their ring costs too many warps (512 rows of 32 heads of 128: 134 against 126).  A warp that owns all splits joins them in its
// shared memory, then with the prefix's states, and writes the output; otherwise every split leaves its
// state for combine_kernel.
#pragma once

#include <type_traits>

#include "dk_common.cuh"

namespace dk {
namespace own {

constexpr int kSplit = 64;
constexpr int kRows = 16;

enum : int {
  kDetLen = 0x210,   // a kv_len exceeds the cache capacity or max_kv_len
  kDetTile = 0x211,  // a row tile is malformed
  kDetPage = 0x212,  // a block table entry outside the block pool
};

// Whether a row tile lies inside the batch and the cache and fits a unit of `most` query rows.
__device__ __forceinline__ bool tile_fits(int r0, int nr, int seq, int G, int most, int n_rows, int n_seq) {
  return nr >= 1 && nr <= most && nr * G <= most && r0 >= 0 && r0 <= n_rows - nr && seq >= 0 && seq < n_seq;
}

// 2^x by the single hardware instruction; 2^-inf = 0, 2^0 = 1.
__device__ __forceinline__ float exp2_hw(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Weights (a, b) that join state (m, ..) with (ms, ..): the joined value is v * a + vs * b.
__device__ __forceinline__ float join_weights(float m, float ms, float& a, float& b) {
  const float mn = fmaxf(m, ms);
  const float ref = (mn == -INFINITY) ? 0.0f : mn;
  a = exp2_hw(__fsub_rn(m, ref));
  b = exp2_hw(__fsub_rn(ms, ref));
  return mn;
}
__device__ __forceinline__ float join(float v, float a, float vs, float b) { return __fmaf_rn(v, a, __fmul_rn(vs, b)); }
__device__ __forceinline__ float4 join4(float4 v, float a, float4 vs, float b) {
  return make_float4(join(v.x, a, vs.x, b), join(v.y, a, vs.y, b), join(v.z, a, vs.z, b), join(v.w, a, vs.w, b));
}

struct Params {
  const void *q, *k, *v;
  int64_t q_sr, q_sh;
  int64_t c_sn, c_sh, c_st;   // cache strides: sequence or block, head, token
  const int32_t* kv_lens;
  const int32_t* tiles;       // null: row r is a tile of sequence r
  int32_t n_tiles, n_rows, hq, hkv, G;
  int32_t n_seq, capacity;    // capacity: the longest length a row may have, at most max_splits splits
  const int32_t* block_table; // null: contiguous
  int64_t bt_stride;
  int32_t page, n_blocks;
  int32_t max_splits, spu, upt;   // splits a unit, units a (tile, head)
  float scale_log2;
  float* st_o;                // [max_splits][D / 4][st_rows][4], when out is null
  float* st_ml;               // [max_splits][st_rows][2]
  int64_t st_rows;            // hkv * rows * G: state row (kvh * rows + row) * G + head in the group
  // upt == 1: a unit owns all of its rows' splits, joins them with the prefix's states and writes the output
  void* out;
  int64_t o_sr, o_sh;
  const float* px_o;          // [n_runs][D / 4][st_rows][4]
  const float* px_ml;         // [n_runs][st_rows][2]
  int32_t n_runs, per_group;
};

template <int D>
struct Cfg {
  static constexpr int ROWB = D * 2;
  static constexpr int STEP = D == 128 ? 16 : 32;   // tokens a step
  static constexpr int TENSOR = STEP * ROWB;
  static constexpr int STAGE = 2 * TENSOR;
  static constexpr int STAGES = D == 128 ? 3 : 2;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int ROWF = D + 4;   // floats of a joined row in shared memory (conflict free either way)
  // the ring, then, for a warp that owns all splits, its 8 NB rows and their (m, l)
  static constexpr int smem(int nb, bool all) { return RING + (all ? 8 * nb * (ROWF + 2) * 4 : 0); }
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Whether either 16-bit value of a pair is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool non_finite(uint32_t v) {
  constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (v & e) == e || ((v >> 16) & e) == e;
}

// Byte offset of 16-byte chunk c of token row r in a stage tensor (conflict free for ldmatrix).
template <int D>
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
  const int swz = D >= 64 ? (r & 7) : ((r >> 1) & 3);
  return static_cast<uint32_t>(r * Cfg<D>::ROWB + ((c ^ swz) << 4));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {   // an 8 x 8 matrix of 16-bit values
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// NB: column halves (8 query rows each).
template <typename T, int D, int NB>
__global__ void __launch_bounds__(32, NB == 2 ? (D == 128 ? 9 : 10) : (D == 128 ? 12 : 16)) own_kernel(const Params p) {
  using C = Cfg<D>;
  constexpr int KC = D / 16, CPR = D / 8;
  constexpr int kStep = C::STEP, U = kStep / 16;
  constexpr int PER = kStep * CPR / 32;   // 16-byte chunks a lane copies of each tensor a step
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_launch_dependents();
  const int lane = threadIdx.x;
  int64_t w = blockIdx.x;
  const int kvh = static_cast<int>(w % p.hkv);
  w /= p.hkv;
  const int unit = static_cast<int>(w % p.upt);
  const int tile = static_cast<int>(w / p.upt);
  // every exit waits for the kernel before this one (see the launch)
  int r0 = tile, nr = 1, seq = tile;
  if (p.tiles) {
    r0 = p.tiles[3 * tile];
    nr = p.tiles[3 * tile + 1];
    seq = p.tiles[3 * tile + 2];
  }
  if (nr == 0) {   // padding of a tile list
    pdl_wait();
    return;
  }
  if (!tile_fits(r0, nr, seq, p.G, 8 * NB, p.n_rows, p.n_seq)) {
    if (lane == 0 && unit == 0 && kvh == 0) report_error(DK_ERR_DEVICE_CHECK, kDetTile);
    pdl_wait();
    return;
  }
  const int my_len = lane < nr ? p.kv_lens[r0 + lane] : 0;
  const bool bad = my_len < 0 || my_len > p.capacity;
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0 && unit == 0 && kvh == 0) report_error(DK_ERR_DEVICE_CHECK, kDetLen);
    pdl_wait();
    return;
  }
  const int max_len = __reduce_max_sync(0xffffffffu, my_len);
  const int min_len = __reduce_min_sync(0xffffffffu, lane < nr ? my_len : max_len);
  const bool all = p.upt == 1;
  const int t_begin = unit * p.spu * kSplit;
  const int t_end = t_begin + min(max_len - t_begin, p.spu * kSplit);   // (the sum of the two may leave 32 bits)
  if (t_begin >= t_end && !all) {
    pdl_wait();
    return;
  }
  const int g = lane >> 2, t4 = lane & 3;
  const int valid_rows = nr * p.G;
  // this lane's columns: query rows 8 h + 2 t4 + e of the tile, their tile rows and token ends
  int col_row[NB][2], end[NB][2];
#pragma unroll
  for (int h = 0; h < NB; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rho = 8 * h + 2 * t4 + e;
      col_row[h][e] = rho / p.G;
      const int len = __shfl_sync(0xffffffffu, my_len, min(col_row[h][e], 31));
      end[h][e] = rho < valid_rows ? len : 0;
    }

  // ---- loads: lane's chunks of a step, one page lookup a step (a page holds whole steps) ----
  const T* kb = static_cast<const T*>(p.k) + static_cast<int64_t>(kvh) * p.c_sh;
  const T* vb = static_cast<const T*>(p.v) + static_cast<int64_t>(kvh) * p.c_sh;
  const uint32_t ring_a = smem_u32(ring);
  constexpr int RPI = 32 / CPR > 0 ? 32 / CPR : 1;   // rows an instruction of the warp covers
  const int ld_r = lane / CPR, ld_c = lane % CPR;    // D = 128: 2 rows of 16 chunks an instruction
  int pg_first = -64, pg_mine = 0;                   // 32 table entries, one a lane
  const int n_steps = (t_end - t_begin + kStep - 1) / kStep;
  auto issue = [&](int st) {
    if (st < n_steps) {
      const int t0 = t_begin + st * kStep;
      int64_t slab = seq;
      int tok = t0;
      if (p.block_table) {
        const int pg = t0 / p.page;
        if (pg >= pg_first + 32 || pg < pg_first) {
          pg_first = pg;
          const int e = pg + lane;
          pg_mine = e * static_cast<int64_t>(p.page) < t_end
                        ? p.block_table[static_cast<int64_t>(seq) * p.bt_stride + e] : 0;
          if (pg_mine < 0 || pg_mine >= p.n_blocks) {
            report_error(DK_ERR_DEVICE_CHECK, kDetPage);
            pg_mine = 0;
          }
        }
        slab = __shfl_sync(0xffffffffu, pg_mine, pg - pg_first);
        tok = t0 - pg * p.page;
      }
      const int64_t off0 = slab * p.c_sn + static_cast<int64_t>(tok + ld_r) * p.c_st + ld_c * 8;
      const T* ks = kb + off0;
      const T* vs = vb + off0;
      const int64_t inc = RPI * p.c_st;
      const uint32_t dst = ring_a + (st % C::STAGES) * C::STAGE;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r = ld_r + i * RPI;
        const bool live = t0 + r < t_end;
        const uint32_t d = dst + chunk_off<D>(r, ld_c);
        cp_async16(d, live ? ks : kb, live);
        cp_async16(d + C::TENSOR, live ? vs : vb, live);
        ks += inc;
        vs += inc;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int st = 0; st < C::STAGES - 1; ++st) issue(st);

  // ---- query fragments: q^T, column g of each half ----
  uint32_t qb[NB][KC][2];
#pragma unroll
  for (int h = 0; h < NB; ++h) {
    const int rho = 8 * h + g, i = rho / p.G;
    const T* q = static_cast<const T*>(p.q) + static_cast<int64_t>(r0 + i) * p.q_sr +
                 static_cast<int64_t>(kvh * p.G + rho - i * p.G) * p.q_sh;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      qb[h][kc][0] = rho < valid_rows ? *reinterpret_cast<const uint32_t*>(q + kc * 16 + 2 * t4) : 0u;
      qb[h][kc][1] = rho < valid_rows ? *reinterpret_cast<const uint32_t*>(q + kc * 16 + 2 * t4 + 8) : 0u;
    }
  }
  const int mi = lane >> 3, ri = lane & 7;
  const int k_row = (mi & 1) * 8 + ri, k_c = mi >> 1;   // K as stored: token halves, then k halves
  const int v_row = (mi >> 1) * 8 + ri, v_c = mi & 1;   // V transposed: d halves, then token halves

  float o[NB][KC][4], m_r[NB][2], l_r[NB][2];
  float run_m[NB][2], run_l[NB][2];
  float* const run_o = reinterpret_cast<float*>(ring + C::RING);   // [8 NB][ROWF]
  float* const run_ml = run_o + 8 * NB * C::ROWF;                  // [8 NB][2]
#pragma unroll
  for (int h = 0; h < NB; ++h) {
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[h][j][e] = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m_r[h][e] = run_m[h][e] = -INFINITY;
      l_r[h][e] = run_l[h][e] = 0.0f;
    }
  }

  const int64_t n0 = (static_cast<int64_t>(kvh) * p.n_rows + r0) * p.G + 2 * t4;   // state row of column 2 t4
  auto store = [&](int64_t s, int h, int e, float m, float l) {
    const int64_t n = n0 + 8 * h + e;
    if (g == 0) *reinterpret_cast<float2*>(p.st_ml + 2 * (s * p.st_rows + n)) = make_float2(m, l);
    float* dst = p.st_o + ((s * (D / 4) + (g >> 2)) * p.st_rows + n) * 4 + (g & 3);
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      dst[static_cast<int64_t>(4 * j) * p.st_rows * 4] = o[h][j][e];
      dst[static_cast<int64_t>(4 * j + 2) * p.st_rows * 4] = o[h][j][2 + e];
    }
  };

  for (int st = 0; st < n_steps; ++st) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncwarp();
    issue(st + C::STAGES - 1);   // into the stage read in the previous step
    const uint32_t ka = ring_a + (st % C::STAGES) * C::STAGE, va = ka + C::TENSOR;
    const int t0 = t_begin + st * kStep;
    float sc[U][NB][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int h = 0; h < NB; ++h) sc[u][h][0] = sc[u][h][1] = sc[u][h][2] = sc[u][h][3] = 0.0f;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        uint32_t a[4];
        ldsm_x4(ka + chunk_off<D>(16 * u + k_row, 2 * kc + k_c), a);
#pragma unroll
        for (int h = 0; h < NB; ++h) mma<T>(sc[u][h], a, qb[h][kc][0], qb[h][kc][1]);
      }
    }
    // scores: sc[u][h][0..1] token t0 + 16 u + g, sc[u][h][2..3] token t0 + 16 u + g + 8, columns 2 t4 and 2 t4 + 1
    uint32_t pb[U][NB][2];
    bool same = true;
    float alpha[NB][2];
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      float x[U][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u][e] = (t0 + 16 * u + g < end[h][e]) ? __fmul_rn(sc[u][h][e], p.scale_log2) : -INFINITY;
          x[u][2 + e] = (t0 + 16 * u + g + 8 < end[h][e]) ? __fmul_rn(sc[u][h][2 + e], p.scale_log2) : -INFINITY;
          mx = fmaxf(mx, fmaxf(x[u][e], x[u][2 + e]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m_r[h][e], mx);
        const float ref = (mn == -INFINITY) ? 0.0f : mn;
        alpha[h][e] = exp2_hw(__fsub_rn(m_r[h][e], ref));
        same = same && alpha[h][e] == 1.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u][e] = exp2_hw(__fsub_rn(x[u][e], ref));
          x[u][2 + e] = exp2_hw(__fsub_rn(x[u][2 + e], ref));
        }
        m_r[h][e] = mn;
        l_r[h][e] = __fmul_rn(l_r[h][e], alpha[h][e]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t lo = pack2<T>(x[u][0], x[u][1]), hi = pack2<T>(x[u][2], x[u][3]);
        const float2 a = unpack2<T>(lo), b = unpack2<T>(hi);
        l_r[h][0] = __fadd_rn(l_r[h][0], __fadd_rn(a.x, b.x));
        l_r[h][1] = __fadd_rn(l_r[h][1], __fadd_rn(a.y, b.y));
        pb[u][h][0] = transpose8(lo);
        pb[u][h][1] = transpose8(hi);
      }
    }
    if (!same) {   // a factor of exactly 1 changes nothing
#pragma unroll
      for (int h = 0; h < NB; ++h)
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[h][j][e] = __fmul_rn(o[h][j][e], alpha[h][e & 1]);
    }
    // a row's weights beyond its end are 0, which a non-finite value there (a later row's token) must
    // not meet: then each row goes alone, longest first, over values cut at its own end
    bool alone = false;
    if (t0 + kStep > min_len && min_len < max_len) {
      bool wild = false;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r = ld_r + i * RPI;
        const uint4 x = *reinterpret_cast<const uint4*>(ring + (va - ring_a) + chunk_off<D>(r, ld_c));
        wild |= t0 + r >= min_len && (non_finite<T>(x.x) || non_finite<T>(x.y) || non_finite<T>(x.z) ||
                                      non_finite<T>(x.w));
      }
      alone = __any_sync(0xffffffffu, wild);
    }
    if (!alone) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          uint32_t a[4];
          ldsm_x4_t(va + chunk_off<D>(16 * u + v_row, 2 * j + v_c), a);
#pragma unroll
          for (int h = 0; h < NB; ++h) mma<T>(o[h][j], a, pb[u][h][0], pb[u][h][1]);
        }
    } else {
      int left = lane < nr ? my_len : -1;
      for (int k = 0; k < nr; ++k) {
        const int cut = __reduce_max_sync(0xffffffffu, left);
        const int row = __ffs(__ballot_sync(0xffffffffu, left == cut)) - 1;
        if (lane == row) left = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int r = ld_r + i * RPI;
          if (t0 + r >= cut)
            *reinterpret_cast<uint4*>(ring + (va - ring_a) + chunk_off<D>(r, ld_c)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          uint32_t a[U][4];
#pragma unroll
          for (int u = 0; u < U; ++u) ldsm_x4_t(va + chunk_off<D>(16 * u + v_row, 2 * j + v_c), a[u]);
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            float one[4] = {o[h][j][0], o[h][j][1], o[h][j][2], o[h][j][3]};
#pragma unroll
            for (int u = 0; u < U; ++u) mma<T>(one, a[u], pb[u][h][0], pb[u][h][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col_row[h][e & 1] == row) o[h][j][e] = one[e];
          }
        }
        __syncwarp();
      }
    }
    if ((st + 1) % (kSplit / kStep) == 0 || st + 1 == n_steps) {
      const int sp_begin = t0 / kSplit * kSplit;   // first token of the split that ends here
#pragma unroll
      for (int h = 0; h < NB; ++h) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float l = l_r[h][e];
          l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 4));
          l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 8));
          l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, 16));
          if (sp_begin < end[h][e]) {        // the row has tokens in this split
            float* const row = run_o + (8 * h + 2 * t4 + e) * C::ROWF + g;
            if (!all) {
              store(sp_begin / kSplit, h, e, m_r[h][e], l);
            } else if (sp_begin == 0) {
              run_m[h][e] = m_r[h][e];
              run_l[h][e] = l;
#pragma unroll
              for (int j = 0; j < KC; ++j) {
                row[16 * j] = o[h][j][e];
                row[16 * j + 8] = o[h][j][2 + e];
              }
            } else {
              float a, b;
              run_m[h][e] = join_weights(run_m[h][e], m_r[h][e], a, b);
              run_l[h][e] = join(run_l[h][e], a, l, b);
#pragma unroll
              for (int j = 0; j < KC; ++j) {
                row[16 * j] = join(row[16 * j], a, o[h][j][e], b);
                row[16 * j + 8] = join(row[16 * j + 8], a, o[h][j][2 + e], b);
              }
            }
          }
          m_r[h][e] = -INFINITY;
          l_r[h][e] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < KC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[h][j][e] = 0.0f;
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  pdl_wait();
  if (!all) return;
  // ---- join with the prefix's states and write the output: a lane takes row lane / 4 of a half and every
  // fourth column quad ----
  if (g == 0) {
#pragma unroll
    for (int h = 0; h < NB; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float2*>(run_ml + 2 * (8 * h + 2 * t4 + e)) = make_float2(run_m[h][e], run_l[h][e]);
  }
  __syncwarp();
  constexpr int QL = D / 16;   // quads a lane
#pragma unroll 1
  for (int h = 0; h < NB; ++h) {
    const int rho = 8 * h + g, i = rho / p.G;
    const int len = __shfl_sync(0xffffffffu, my_len, min(i, 31));
    if (rho >= valid_rows) continue;
    const int64_t n = (static_cast<int64_t>(kvh) * p.n_rows + r0) * p.G + rho;
    const float2* mls = reinterpret_cast<const float2*>(p.px_ml) + n;
    const float4* src = reinterpret_cast<const float4*>(p.px_o) + static_cast<int64_t>(t4) * p.st_rows + n;
    float tm = -INFINITY, tl = 0.0f, gm = -INFINITY, gl = 0.0f;
    float4 to[QL], go[QL];
    int in_group = 0;
    for (int s = 0; s < p.n_runs; ++s) {
      const float2 ml = __ldcg(mls + s * p.st_rows);
      float4 v[QL];
#pragma unroll
      for (int k = 0; k < QL; ++k) v[k] = __ldcg(src + (static_cast<int64_t>(s) * (D / 4) + 4 * k) * p.st_rows);
      float a = 0.0f, b = 1.0f;
      const bool head = in_group == 0;
      if (head) {
        gm = ml.x;
        gl = ml.y;
      } else {
        gm = join_weights(gm, ml.x, a, b);
        gl = join(gl, a, ml.y, b);
      }
#pragma unroll
      for (int k = 0; k < QL; ++k) go[k] = head ? v[k] : join4(go[k], a, v[k], b);
      if (++in_group == p.per_group || s + 1 == p.n_runs) {
        in_group = 0;
        const bool only = s < p.per_group;
        if (only) {
          tm = gm;
          tl = gl;
        } else {
          tm = join_weights(tm, gm, a, b);
          tl = join(tl, a, gl, b);
        }
#pragma unroll
        for (int k = 0; k < QL; ++k) to[k] = only ? go[k] : join4(to[k], a, go[k], b);
      }
    }
    float a = 1.0f, b = 0.0f;
    if (len > 0) {
      const float2 ml = *reinterpret_cast<const float2*>(run_ml + 2 * rho);
      join_weights(tm, ml.x, a, b);
      tl = join(tl, a, ml.y, b);
    }
    T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(r0 + i) * p.o_sr +
             static_cast<int64_t>(kvh * p.G + rho - i * p.G) * p.o_sh;
    const bool vec = (reinterpret_cast<uintptr_t>(dst) & 7u) == 0;
#pragma unroll
    for (int k = 0; k < QL; ++k) {
      const int d = 4 * (t4 + 4 * k);
      float4 v = to[k];
      if (len > 0) v = join4(v, a, *reinterpret_cast<const float4*>(run_o + rho * C::ROWF + d), b);
      const uint32_t lo = pack2<T>(__fdiv_rn(v.x, tl), __fdiv_rn(v.y, tl));
      const uint32_t hi = pack2<T>(__fdiv_rn(v.z, tl), __fdiv_rn(v.w, tl));
      if (vec) {
        *reinterpret_cast<uint2*>(dst + d) = make_uint2(lo, hi);
      } else {
        const T* e = reinterpret_cast<const T*>(&lo);
        dst[d] = e[0];
        dst[d + 1] = e[1];
        e = reinterpret_cast<const T*>(&hi);
        dst[d + 2] = e[0];
        dst[d + 3] = e[1];
      }
    }
  }
}

}  // namespace own
}  // namespace dk
