// Per-head RMSNorm of queries and keys with the position rotation in the same pass, K and V stored
// into a KV cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w              (one head vector x of D elements, f32)
//   (a, b) -> (a cos - b sin, a sin + b cos)        for each pair of the first rd elements of y
//
// with pairs (i, i + rd / 2), or (2i, 2i + 1) when interleaved, and cos/sin of the row's position
// from an f32 table.  Everything stays in f32 until the one rounding of the store.  The sum of
// squares of a vector has a fixed order (a lane's elements in order, on the vector path even and odd ones apart, then
// a butterfly), so a row's bits depend on the path, which the call's layout decides, and not on the other rows.
//
// Memory bound: every vector is read and written once.  A group of lanes owns a vector in 16-byte
// chunks, lane l holding chunks l, l + L, l + 2L, ... with L = rd / 2 in chunks, so both elements of
// a pair sit in one lane.
#pragma once

#include "dk_common.cuh"

namespace dk {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxDim = 512;

enum : int {
  kDetPos = 0x610,    // a position outside the table
  kDetSlot = 0x611,   // a slot outside the cache
};

struct Params {
  const void *q, *k, *v;                 // [T, H | Hkv, D]; v null: no cache
  int64_t q_sr, q_sh, k_sr, k_sh, v_sr, v_sh;
  void *qo, *ko;                         // ko null: K goes to the cache only
  int64_t qo_sr, qo_sh, ko_sr, ko_sh;
  void *kc, *vc;                         // cache [n_slabs, Hkv, cap, D]
  int64_t c_sn, c_sh, c_st;
  int64_t cap, n_slabs;
  const int64_t* slots;
  const void* pos;                       // int32 or int64 [T]
  int pos64;
  const void *qw, *kw;
  int wdtype;
  const float* table;                    // [max_pos, rd]: cos then sin
  int64_t max_pos;
  int64_t n_rows;
  int H, Hkv, D, rd, interleaved;
  float eps, inv_d;                      // inv_d: 1 / D
  int nvec;                              // vectors a row: H + Hkv (+ Hkv with a cache)
  int lanes;                             // vector path: lanes that hold chunks (L)
  int glog;                              // log2 of the group's lane count
  int vpu;                               // vectors a warp walks (a multiple of the groups in it)
  int upr;                               // warps a row
};

template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
};

__device__ __forceinline__ float load_w(const void* w, int dtype, int i) {
  if (dtype == DK_F32) return static_cast<const float*>(w)[i];
  if (dtype == DK_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// A row's position and cache place; false when the position is outside the table.
struct Row {
  int64_t pos;
  int64_t cache;      // element offset of the row's token in head 0 of the cache, -1: not stored
};
__device__ __forceinline__ bool describe_row(const Params& p, int64_t t, bool report, Row& r) {
  r.pos = p.pos64 ? static_cast<const int64_t*>(p.pos)[t] : static_cast<const int32_t*>(p.pos)[t];
  r.cache = -1;
  if (r.pos < 0 || r.pos >= p.max_pos) {
    if (report) report_error(DK_ERR_DEVICE_CHECK, kDetPos);
    return false;
  }
  if (p.slots) {
    const int64_t s = p.slots[t];
    if (s >= 0) {
      const bool narrow = s <= 0xffffffffLL && p.cap <= 0xffffffffLL;
      const int64_t n = narrow ? static_cast<int64_t>(static_cast<uint32_t>(s) / static_cast<uint32_t>(p.cap)) : s / p.cap;
      if (n >= p.n_slabs) {
        if (report) report_error(DK_ERR_DEVICE_CHECK, kDetSlot);
      } else {
        r.cache = n * p.c_sn + (s - n * p.cap) * p.c_st;
      }
    }
  }
  return true;
}

// Where vector i of row t comes from and goes to (q heads, then k heads, then v heads).
template <typename T>
struct Place {
  const T* src;
  T* dst;       // null: nowhere
  T* dst2;      // a key's second destination (k_out beside the cache)
  int kind;     // 0 q, 1 k, 2 v
};
template <typename T>
__device__ __forceinline__ Place<T> place(const Params& p, const Row& row, int64_t t, int i) {
  Place<T> o;
  o.dst2 = nullptr;
  if (i < p.H) {
    o.kind = 0;
    o.src = static_cast<const T*>(p.q) + t * p.q_sr + i * p.q_sh;
    o.dst = static_cast<T*>(p.qo) + t * p.qo_sr + i * p.qo_sh;
  } else if (i < p.H + p.Hkv) {
    const int h = i - p.H;
    o.kind = 1;
    o.src = static_cast<const T*>(p.k) + t * p.k_sr + h * p.k_sh;
    o.dst = p.ko ? static_cast<T*>(p.ko) + t * p.ko_sr + h * p.ko_sh : nullptr;
    if (row.cache >= 0) o.dst2 = static_cast<T*>(p.kc) + row.cache + h * p.c_sh;
  } else {
    const int h = i - p.H - p.Hkv;
    o.kind = 2;
    o.src = static_cast<const T*>(p.v) + t * p.v_sr + h * p.v_sh;
    o.dst = row.cache >= 0 ? static_cast<T*>(p.vc) + row.cache + h * p.c_sh : nullptr;
  }
  return o;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& c, float* x);
template <>
__device__ __forceinline__ void unpack<float>(const uint4& c, float* x) {
  x[0] = __uint_as_float(c.x);
  x[1] = __uint_as_float(c.y);
  x[2] = __uint_as_float(c.z);
  x[3] = __uint_as_float(c.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& c, float* x) {
  const uint32_t u[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4& c, float* x) {
  const uint32_t u[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float* x);
template <>
__device__ __forceinline__ uint4 pack<float>(const float* x) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
template <>
__device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float* x) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <>
__device__ __forceinline__ uint4 pack<__half>(const float* x) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// Two f32 operations an instruction, each rounded by itself.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Vector path.  NC: chunks a lane holds (chunk l + j L, j < NC).  Rotated chunks: 0 and 1 (pairs
// between them) or, interleaved, those with index < rd / N (pairs inside a chunk).
//
// Warps walk units (a row, or part of one when rows are few) grid-stride, the next unit's position and
// slot in flight while one is rotated.  The weights stay in shared memory as f32 and the angles are read
// back from the cache a batch at a time, as 16-byte vectors.  Bound by the latency of its loads at the registers
// they leave: the 66,377-row prefill of 32 vectors of 64 a row (floor 86 us) took 161 us with both in registers
// through a type switch, 123 us with four vectors a lane in flight and the spills of that, and takes 113 us
// (5.0 TB/s) with two.  One resident set of 3 CTAs an SM walks all units; one CTA per 8 units took 15 % more.
// Half the arithmetic's instructions (f32x2) left the prefill as it was and took small batches from 4.0 to 3.2 us;
// fetching the next unit's vectors ahead cost more registers than it hid (142 us).
template <typename T, int NC, bool INTER>
__global__ void __launch_bounds__(kThreads, 3) vec_kernel(const Params p) {
  constexpr int N = Chunk<T>::N;
  constexpr int UB = NC <= 2 ? 2 : 1;   // vectors in flight per group
  constexpr int NA = INTER ? NC * N / 2 : N;   // angles a lane holds
  __shared__ __align__(16) float s_w[2][kMaxDim];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  for (int i = threadIdx.x; i < 2 * p.D; i += kThreads) {
    const int k = i >= p.D;
    if (k ? p.Hkv > 0 : p.H > 0) s_w[k][i - k * p.D] = load_w(k ? p.kw : p.qw, p.wdtype, i - k * p.D);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int gl = 1 << p.glog, gpw = 32 >> p.glog;
  const int l = lane & (gl - 1), gi = lane >> p.glog;
  const bool on = l < p.lanes;
  const int half = p.rd >> 1, cstep = p.lanes * N;   // elements between a lane's chunks
  const uint32_t units = static_cast<uint32_t>(p.n_rows) * p.upr;   // < 2^31 (the host checks)
  const uint32_t step = gridDim.x * (kThreads / 32);
  uint32_t unit = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  Row row{0, -1};
  bool good = unit < units && describe_row(p, unit / p.upr, lane == 0 && unit % p.upr == 0, row);
  for (; unit < units; unit += step) {
    const uint32_t t = unit / p.upr, part = unit - t * p.upr;
    const Row now = row;
    const bool go = good;
    const uint32_t next = unit + step;
    if (next < units) good = describe_row(p, next / p.upr, lane == 0 && next % p.upr == 0, row);
    if (!go) continue;   // (the whole warp: one row a unit)
    const int begin = static_cast<int>(part) * p.vpu;
    const int end = min(p.nvec, begin + p.vpu);
    // the row's tensors at this lane's first chunk
    const T* const qs = static_cast<const T*>(p.q) + t * p.q_sr + l * N;
    const T* const ks = static_cast<const T*>(p.k) + t * p.k_sr + l * N;
    const T* const vs = static_cast<const T*>(p.v) + t * p.v_sr + l * N;
    T* const qd = static_cast<T*>(p.qo) + t * p.qo_sr + l * N;
    T* const kd = static_cast<T*>(p.ko) + t * p.ko_sr + l * N;
    T* const kc = static_cast<T*>(p.kc) + now.cache + l * N;
    T* const vc = static_cast<T*>(p.vc) + now.cache + l * N;
    uint4 c[UB][NC];
    for (int i0 = begin; i0 < end; i0 += UB * gpw) {
      if (on) {
#pragma unroll
        for (int u = 0; u < UB; ++u) {
          const int i = i0 + gi + u * gpw;
          if (i < end) {
            const T* src = i < p.H ? qs + i * p.q_sh
                                   : (i < p.H + p.Hkv ? ks + (i - p.H) * p.k_sh : vs + (i - p.H - p.Hkv) * p.v_sh);
#pragma unroll
            for (int j = 0; j < NC; ++j) c[u][j] = __ldcs(reinterpret_cast<const uint4*>(src + j * cstep));
          }
        }
      }
      // this lane's angles: pairs of chunk 0 with chunk 1 share index i in [l N, l N + N); interleaved,
      // chunk j's pairs are i = (l + j L) N / 2 + [0, N / 2)  (re-read a batch from the cache: no registers held)
      F2 co[NA / 2], si[NA / 2], ns[NA / 2];   // ns: -sin
      if (on) {
        const float* cs = p.table + now.pos * p.rd;
        if constexpr (INTER) {
          // pair (a, b) -> (a, b) (cos, cos) + (b, a) (-sin, sin): both factors of two elements in one register pair
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const int at = (l + j * p.lanes) * (N / 2);
            const bool rot = at < half;   // a chunk is rotated as a whole
#pragma unroll
            for (int i = 0; i < N / 2; i += 2) {
              const float2 a = rot ? __ldg(reinterpret_cast<const float2*>(cs + at + i)) : make_float2(1.0f, 1.0f);
              const float2 b = rot ? __ldg(reinterpret_cast<const float2*>(cs + half + at + i)) : make_float2(0.0f, 0.0f);
              co[(j * (N / 2) + i) / 2] = f2(a.x, a.y);
              si[(j * (N / 2) + i) / 2] = f2(b.x, b.y);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; i += 4) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(cs + l * N + i));
            const float4 b = __ldg(reinterpret_cast<const float4*>(cs + half + l * N + i));
            co[i / 2] = f2(a.x, a.y), co[i / 2 + 1] = f2(a.z, a.w);
            si[i / 2] = f2(b.x, b.y), si[i / 2 + 1] = f2(b.z, b.w);
            ns[i / 2] = f2(-b.x, -b.y), ns[i / 2 + 1] = f2(-b.z, -b.w);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UB; ++u) {
        // every lane of the warp takes part in the shuffles
        const int i = i0 + gi + u * gpw;
        const bool live = on && i < end && i < p.H + p.Hkv;
        F2 x[NC][N / 2];
        float ss = 0.0f;
        if (live) {
          F2 sum = f2(0.0f, 0.0f);
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            float f[N];
            unpack<T>(c[u][j], f);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              x[j][e] = f2(f[2 * e], f[2 * e + 1]);
              sum = fma2(x[j][e], x[j][e], sum);
            }
          }
          const float2 parts = unpair(sum);
          ss = __fadd_rn(parts.x, parts.y);
        }
        for (int d = gl >> 1; d > 0; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, d));
        if (live) {
          const float rs = rsqrtf(__fmaf_rn(ss, p.inv_d, p.eps));
          const F2 rs2 = f2(rs, rs);
          const float* w = s_w[i >= p.H] + l * N;
#pragma unroll
          for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int e = 0; e < N; e += 4) {
              const float4 f = *reinterpret_cast<const float4*>(w + j * cstep + e);
              x[j][e / 2] = mul2(mul2(x[j][e / 2], rs2), f2(f.x, f.y));
              x[j][e / 2 + 1] = mul2(mul2(x[j][e / 2 + 1], rs2), f2(f.z, f.w));
            }
          if constexpr (INTER) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
              // a chunk that is not rotated keeps its values as they are: times (1, 0) a NaN would reach its neighbour
              const bool rot = (l + j * p.lanes) * (N / 2) < half;
#pragma unroll
              for (int e = 0; e < N / 2; ++e) {
                const float2 y = unpair(x[j][e]);
                const float2 c2 = unpair(co[(j * (N / 2) + e) / 2]), s2 = unpair(si[(j * (N / 2) + e) / 2]);
                const float cc = (e & 1) ? c2.y : c2.x, sn = (e & 1) ? s2.y : s2.x;
                const F2 turned = fma2(x[j][e], f2(cc, cc), mul2(f2(y.y, y.x), f2(-sn, sn)));
                if (rot) x[j][e] = turned;
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              const F2 a = x[0][e], b = x[1][e];
              x[0][e] = fma2(a, co[e], mul2(b, ns[e]));
              x[1][e] = fma2(a, si[e], mul2(b, co[e]));
            }
          }
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            float f[N];
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              const float2 y = unpair(x[j][e]);
              f[2 * e] = y.x;
              f[2 * e + 1] = y.y;
            }
            c[u][j] = pack<T>(f);
          }
        }
        if (on && i < end) {
          const int h = i < p.H ? i : (i < p.H + p.Hkv ? i - p.H : i - p.H - p.Hkv);
          T* dst = i < p.H ? qd + h * p.qo_sh : (now.cache >= 0 ? (i < p.H + p.Hkv ? kc : vc) + h * p.c_sh : nullptr);
          if (dst) {
#pragma unroll
            for (int j = 0; j < NC; ++j) *reinterpret_cast<uint4*>(dst + j * cstep) = c[u][j];
          }
          if (p.ko && i >= p.H && i < p.H + p.Hkv) {
#pragma unroll
            for (int j = 0; j < NC; ++j) *reinterpret_cast<uint4*>(kd + h * p.ko_sh + j * cstep) = c[u][j];
          }
        }
      }
    }
  }
}

// Any D <= kMaxDim, rotary width, stride and alignment: a warp per vector, staged in shared memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) any_kernel(const Params p) {
  __shared__ float s_x[kThreads / 32][kMaxDim];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* x = s_x[warp];
  const int64_t n = p.n_rows * p.nvec;
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + warp; w < n;
       w += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
    const int64_t t = w / p.nvec;
    const int i = static_cast<int>(w - t * p.nvec);
    Row row;
    if (!describe_row(p, t, lane == 0 && i == 0, row)) continue;
    const Place<T> pl = place<T>(p, row, t, i);
    float ss = 0.0f;
    for (int e = lane; e < p.D; e += 32) {
      const float f = to_f32<T>(pl.src[e]);
      x[e] = f;
      ss = __fmaf_rn(f, f, ss);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, d));
    __syncwarp();
    const float rs = rsqrtf(__fmaf_rn(ss, p.inv_d, p.eps));
    const float* cs = p.table + row.pos * p.rd;
    const int half = p.rd >> 1;
    const void* wt = pl.kind == 1 ? p.kw : p.qw;
    for (int e = lane; e < p.D; e += 32) {
      T out;
      if (pl.kind == 2) {
        out = pl.src[e];
      } else {
        float y = __fmul_rn(__fmul_rn(x[e], rs), load_w(wt, p.wdtype, e));
        if (e < p.rd) {
          const int pi = p.interleaved ? e >> 1 : (e < half ? e : e - half);
          const bool first = p.interleaved ? !(e & 1) : e < half;
          const int oe = p.interleaved ? e ^ 1 : (first ? e + half : e - half);
          const float o = __fmul_rn(__fmul_rn(x[oe], rs), load_w(wt, p.wdtype, oe));
          const float c = cs[pi], s = cs[half + pi];
          y = first ? __fmaf_rn(y, c, -__fmul_rn(o, s)) : __fmaf_rn(o, s, __fmul_rn(y, c));
        }
        out = from_f32<T>(y);
      }
      if (pl.dst) pl.dst[e] = out;
      if (pl.dst2) pl.dst2[e] = out;
    }
    __syncwarp();
  }
}

}  // namespace rope
}  // namespace dk
