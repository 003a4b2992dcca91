// A row's own tokens behind a shared prefix: split-KV decode attention that leaves softmax states.
//
// Fixed reduction structure: the row's tokens [0, len) in splits of kSplit = 256; inside a split
// groups of 16 tokens in order with an online softmax (m, l, O), scores from mma.m16n8k16 (f32
// accumulation), weights rounded to the input type for P.V and summed as rounded; split states
// joined in order.  Nothing depends on the batch, the tile a row sits in or the schedule.
//
// Work: a unit is (row tile of at most 16 query rows of one sequence, KV head, run of splits), one
// warp each, with no barrier wider than the warp: short sequences, which are what follows a shared
// prefix, leave many small units whose loads overlap each other across the 14 (head_dim 64) or 9
// (128) warps an SM holds.  K and V come through a ring of 16-token stages (cp.async, zero filled
// past the sequence's end, so that whatever the cache holds there is never read).  A warp that owns
// all splits joins them in registers; otherwise every split leaves its state for combine_kernel.
#pragma once

#include <type_traits>

#include "dk_common.cuh"

namespace dk {
namespace own {

constexpr int kSplit = 256;
constexpr int kStep = 16;
constexpr int kRows = 16;

enum : int {
  kDetLen = 0x210,   // a kv_len exceeds the cache capacity or max_kv_len
  kDetTile = 0x211,  // a row tile is malformed
  kDetPage = 0x212,  // a block table entry outside the block pool
};

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

struct Params {
  const void *q, *k, *v;
  int64_t q_sr, q_sh;
  int64_t c_sn, c_sh, c_st;   // cache strides: sequence or block, head, token
  const int32_t* kv_lens;
  const int32_t* tiles;       // null: row r is a tile of sequence r
  int32_t n_tiles, n_rows, hq, hkv, G;
  int32_t n_seq, capacity;
  const int32_t* block_table; // null: contiguous
  int64_t bt_stride;
  int32_t page, n_blocks;
  int32_t max_splits, spu, upt;   // splits a unit, units a (tile, head)
  float scale_log2;
  float* st_o;                // [max_splits, or 1 when upt == 1][n_rows * hq][D]
  float* st_ml;               // [..][n_rows * hq][2]
  int64_t st_rows;
};

template <int D>
struct Cfg {
  static constexpr int ROWB = D * 2;
  static constexpr int TENSOR = kStep * ROWB;
  static constexpr int STAGE = 2 * TENSOR;
  static constexpr int STAGES = D == 128 ? 3 : (D == 64 ? 4 : 6);
  static constexpr int SMEM = STAGES * STAGE;
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

template <typename T, int D>
__global__ void __launch_bounds__(32) own_kernel(const Params p) {
  using C = Cfg<D>;
  constexpr int KC = D / 16, NT = D / 8, CPR = D / 8;
  constexpr int PER = kStep * CPR / 32;   // 16-byte chunks a lane copies of each tensor a step
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_launch_dependents();
  const int lane = threadIdx.x;
  int64_t w = blockIdx.x;
  const int kvh = static_cast<int>(w % p.hkv);
  w /= p.hkv;
  const int unit = static_cast<int>(w % p.upt);
  const int tile = static_cast<int>(w / p.upt);
  int r0 = tile, nr = 1, seq = tile;
  if (p.tiles) {
    r0 = p.tiles[3 * tile];
    nr = p.tiles[3 * tile + 1];
    seq = p.tiles[3 * tile + 2];
  }
  // every exit waits for the kernel before this one (see the launch)
  if (nr < 1 || nr * p.G > kRows || r0 < 0 || r0 + nr > p.n_rows || seq < 0 || seq >= p.n_seq) {
    if (lane == 0 && unit == 0 && kvh == 0) report_error(DK_ERR_DEVICE_CHECK, kDetTile);
    pdl_wait();
    return;
  }
  const int my_len = lane < nr ? p.kv_lens[r0 + lane] : 0;
  const bool bad = my_len < 0 || my_len > p.capacity || my_len > p.max_splits * kSplit;
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0 && unit == 0 && kvh == 0) report_error(DK_ERR_DEVICE_CHECK, kDetLen);
    pdl_wait();
    return;
  }
  const int max_len = __reduce_max_sync(0xffffffffu, my_len);
  const int min_len = __reduce_min_sync(0xffffffffu, lane < nr ? my_len : max_len);
  const int t_begin = unit * p.spu * kSplit;
  const int t_end = min(max_len, t_begin + p.spu * kSplit);
  if (t_begin >= t_end) {
    pdl_wait();
    return;
  }
  const int g = lane >> 2, t4 = lane & 3;
  const int valid_rows = nr * p.G;
  const int i0 = g / p.G, i1 = (g + 8) / p.G;      // tile rows of this lane's query rows
  const int len0 = __shfl_sync(0xffffffffu, my_len, min(i0, 31)), len1 = __shfl_sync(0xffffffffu, my_len, min(i1, 31));
  const bool v0 = g < valid_rows, v1 = g + 8 < valid_rows;
  const int end0 = v0 ? len0 : 0, end1 = v1 ? len1 : 0;

  // ---- loads: lane's chunks of a step, one page lookup a step (a page holds whole steps) ----
  const T* kb = static_cast<const T*>(p.k) + static_cast<int64_t>(kvh) * p.c_sh;
  const T* vb = static_cast<const T*>(p.v) + static_cast<int64_t>(kvh) * p.c_sh;
  const uint32_t ring_a = smem_u32(ring);
  int pg_first = -64, pg_mine = 0;                 // 32 table entries, one a lane
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
      const int64_t base = slab * p.c_sn + static_cast<int64_t>(tok) * p.c_st;
      const uint32_t dst = ring_a + (st % C::STAGES) * C::STAGE;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane + i * 32, r = e / CPR, c = e % CPR;
        const bool live = t0 + r < t_end;
        const int64_t off = live ? base + static_cast<int64_t>(r) * p.c_st + c * 8 : 0;
        const uint32_t d = dst + chunk_off<D>(r, c);
        cp_async16(d, kb + off, live);
        cp_async16(d + C::TENSOR, vb + off, live);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int st = 0; st < C::STAGES - 1; ++st) issue(st);

  // ---- query fragments ----
  uint32_t qa[KC][4];
  {
    const T* q = static_cast<const T*>(p.q);
    const T* q0 = q + static_cast<int64_t>(r0 + i0) * p.q_sr + static_cast<int64_t>(kvh * p.G + g - i0 * p.G) * p.q_sh;
    const T* q1 = q + static_cast<int64_t>(r0 + i1) * p.q_sr + static_cast<int64_t>(kvh * p.G + g + 8 - i1 * p.G) * p.q_sh;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      const int d = kc * 16 + 2 * t4;
      qa[kc][0] = v0 ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
      qa[kc][1] = v1 ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
      qa[kc][2] = v0 ? *reinterpret_cast<const uint32_t*>(q0 + d + 8) : 0u;
      qa[kc][3] = v1 ? *reinterpret_cast<const uint32_t*>(q1 + d + 8) : 0u;
    }
  }
  const int mi = lane >> 3, ri = lane & 7;
  const int k_row = (mi >> 1) * 8 + ri, k_c = mi & 1;   // K: two 8-token tiles, k halves
  const int v_row = (mi & 1) * 8 + ri, v_c = mi >> 1;   // V transposed: token halves, two 8-wide d tiles

  float o[NT][4], m_r[2], l_r[2];
  float run_o[NT][4], run_m[2], run_l[2];
  const bool direct = p.upt == 1;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = run_o[j][e] = 0.0f;
  m_r[0] = m_r[1] = run_m[0] = run_m[1] = -INFINITY;
  l_r[0] = l_r[1] = run_l[0] = run_l[1] = 0.0f;

  auto store = [&](int64_t s, int h, float m, float l, const float (&a)[NT][4]) {
    const int rho = g + 8 * h, i = h ? i1 : i0;
    const int64_t idx = s * p.st_rows + static_cast<int64_t>(r0 + i) * p.hq + kvh * p.G + (rho - i * p.G);
    if (t4 == 0) *reinterpret_cast<float2*>(p.st_ml + 2 * idx) = make_float2(m, l);
    float* dst = p.st_o + idx * D + 2 * t4;
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(dst + j * 8) = make_float2(a[j][2 * h], a[j][2 * h + 1]);
  };

  for (int st = 0; st < n_steps; ++st) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncwarp();
    issue(st + C::STAGES - 1);   // into the stage read in the previous step
    const uint32_t ka = ring_a + (st % C::STAGES) * C::STAGE, va = ka + C::TENSOR;
    const int t0 = t_begin + st * kStep;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      uint32_t b[4];
      ldsm_x4(ka + chunk_off<D>(k_row, 2 * kc + k_c), b);
      mma<T>(s0, qa[kc], b[0], b[1]);
      mma<T>(s1, qa[kc], b[2], b[3]);
    }
    const int tk = t0 + 2 * t4;
    uint32_t pa[4];
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[4] = {__fmul_rn(s0[2 * h], p.scale_log2), __fmul_rn(s0[2 * h + 1], p.scale_log2),
                    __fmul_rn(s1[2 * h], p.scale_log2), __fmul_rn(s1[2 * h + 1], p.scale_log2)};
      const int end = h ? end1 : end0;
      if (tk + 0 >= end) x[0] = -INFINITY;
      if (tk + 1 >= end) x[1] = -INFINITY;
      if (tk + 8 >= end) x[2] = -INFINITY;
      if (tk + 9 >= end) x[3] = -INFINITY;
      float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m_r[h], mx);
      const float ref = (mn == -INFINITY) ? 0.0f : mn;
      alpha[h] = exp2_hw(__fsub_rn(m_r[h], ref));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = exp2_hw(__fsub_rn(x[e], ref));
      pa[h] = pack2<T>(x[0], x[1]);
      pa[h + 2] = pack2<T>(x[2], x[3]);
      const float2 a = unpack2<T>(pa[h]), b = unpack2<T>(pa[h + 2]);
      l_r[h] = __fmaf_rn(l_r[h], alpha[h], __fadd_rn(__fadd_rn(a.x, a.y), __fadd_rn(b.x, b.y)));
      m_r[h] = mn;
    }
    if (alpha[0] != 1.0f || alpha[1] != 1.0f) {   // a factor of exactly 1 changes nothing
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        o[j][0] = __fmul_rn(o[j][0], alpha[0]);
        o[j][1] = __fmul_rn(o[j][1], alpha[0]);
        o[j][2] = __fmul_rn(o[j][2], alpha[1]);
        o[j][3] = __fmul_rn(o[j][3], alpha[1]);
      }
    }
    // a row's weights beyond its end are 0, which a non-finite value there (a later row's token) must
    // not meet: then each row goes alone, longest first, over values cut at its own end
    bool alone = false;
    if (t0 + kStep > min_len && min_len < max_len) {
      uint32_t wild = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane + i * 32, r = e / CPR, c = e % CPR;
        const uint4 x = *reinterpret_cast<const uint4*>(ring + (va - ring_a) + chunk_off<D>(r, c));
        wild |= t0 + r >= min_len && (non_finite<T>(x.x) || non_finite<T>(x.y) || non_finite<T>(x.z) ||
                                      non_finite<T>(x.w));
      }
      alone = __any_sync(0xffffffffu, wild != 0);
    }
    if (!alone) {
#pragma unroll
      for (int pc = 0; pc < D / 16; ++pc) {
        uint32_t b[4];
        ldsm_x4_t(va + chunk_off<D>(v_row, 2 * pc + v_c), b);
        mma<T>(o[2 * pc], pa, b[0], b[1]);
        mma<T>(o[2 * pc + 1], pa, b[2], b[3]);
      }
    } else {
      int left = lane < nr ? my_len : -1;
      for (int k = 0; k < nr; ++k) {
        const int cut = __reduce_max_sync(0xffffffffu, left);
        const int row = __ffs(__ballot_sync(0xffffffffu, left == cut)) - 1;
        if (lane == row) left = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int e = lane + i * 32, r = e / CPR, c = e % CPR;
          if (t0 + r >= cut) *reinterpret_cast<uint4*>(ring + (va - ring_a) + chunk_off<D>(r, c)) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
#pragma unroll
        for (int pc = 0; pc < D / 16; ++pc) {
          uint32_t b[4];
          ldsm_x4_t(va + chunk_off<D>(v_row, 2 * pc + v_c), b);
#pragma unroll
          for (int j = 2 * pc; j < 2 * pc + 2; ++j) {
            float one[4] = {o[j][0], o[j][1], o[j][2], o[j][3]};
            mma<T>(one, pa, b[2 * (j & 1)], b[2 * (j & 1) + 1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((e < 2 ? i0 : i1) == row) o[j][e] = one[e];
          }
        }
        __syncwarp();
      }
    }
    __syncwarp();
    if ((st + 1) % (kSplit / kStep) == 0 || st + 1 == n_steps) {
      const int sp_begin = t0 / kSplit * kSplit;   // first token of the split that ends here
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l_r[h] = __fadd_rn(l_r[h], __shfl_xor_sync(0xffffffffu, l_r[h], 1));
        l_r[h] = __fadd_rn(l_r[h], __shfl_xor_sync(0xffffffffu, l_r[h], 2));
        if (sp_begin < (h ? end1 : end0)) {        // the row has tokens in this split
          if (!direct) {
            store(sp_begin / kSplit, h, m_r[h], l_r[h], o);
          } else if (sp_begin == 0) {
            run_m[h] = m_r[h];
            run_l[h] = l_r[h];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              run_o[j][2 * h] = o[j][2 * h];
              run_o[j][2 * h + 1] = o[j][2 * h + 1];
            }
          } else {
            float a, b;
            run_m[h] = join_weights(run_m[h], m_r[h], a, b);
            run_l[h] = join(run_l[h], a, l_r[h], b);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              run_o[j][2 * h] = join(run_o[j][2 * h], a, o[j][2 * h], b);
              run_o[j][2 * h + 1] = join(run_o[j][2 * h + 1], a, o[j][2 * h + 1], b);
            }
          }
        }
        m_r[h] = -INFINITY;
        l_r[h] = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j][2 * h] = o[j][2 * h + 1] = 0.0f;
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (direct) {
    if (end0 > 0) store(0, 0, run_m[0], run_l[0], run_o);
    if (end1 > 0) store(0, 1, run_m[1], run_l[1], run_o);
  }
  pdl_wait();
}

}  // namespace own
}  // namespace dk
