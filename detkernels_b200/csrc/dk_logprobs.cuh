// Log probabilities of given tokens, the entropy and the most likely alternatives of rows of logits.
//
// With a row's logits x, any reference m and y = (x - m) log2 e, S = sum 2^y and T = sum y 2^y give log p(t) = x_t - m -
// log S and the entropy ln 2 (log2 S - T / S), and states (m, S, T) join by S' = f S, T' = f (T + g S), g = (m - m') log2 e,
// f = 2^g.  The difference is taken before the product, so that logits of any size (a type's lowest value among
// them) keep their distances.  One pass over the row, bound by its bytes.
//
// A row is cut into parts by the vocabulary's size alone, one CTA a part and the CTAs of a row a cluster: they join
// in the first one's shared memory, in order, so that there is neither scratch nor a second launch, and a row's bits
// follow from the row.  A thread holds up to 64 logits in registers (eights, 256 threads apart) against its own maximum.
// The alternatives are chosen from the same registers.  A bound below the k-th largest logit is had from the
// threads' maxima: in each of w warps the ceil(k / w)-th largest is at most it, and so is the least of these.  What
// lies above the bound (about twice k of 16384) is collected and ranked by counting; ties at the bound are taken in
// the order of their indices.  Where the bound is poor (logits in order), the k-th largest maximum itself is sought.
#pragma once

#include "dk_common.cuh"

namespace dk {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kVec = 8;                         // consecutive logits of a thread
constexpr int kIters = 8;                       // such vectors a thread holds
constexpr int kPart = kThreads * kVec * kIters; // logits a CTA holds
constexpr int kMaxParts = 8;                    // CTAs a row: a portable cluster
constexpr int kMaxK = 32;
constexpr int kCandidates = 2048;               // above the k-th largest maximum lie at most (k - 1) * 64 logits
constexpr int kPoor = 256;                      // a bound with more above it is worth improving
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
static_assert((kMaxK - 1) * kVec * kIters + kMaxK <= kCandidates, "candidates");

enum : int { kDetToken = 0x650 };               // a token outside the vocabulary (and not -1)

struct Params {
  const void* x;
  int64_t stride;
  int32_t n_vocab, parts, part;     // CTAs a row, logits a part (whole vectors)
  int32_t k;
  const int64_t* tokens;            // null: none asked for
  float* lp;
  float* entropy;                   // null: not asked for
  int64_t* top_ids;
  float* top_lp;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Whole numbers in the order of the values: NaN above all, -0 equal to 0, nothing is 0.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Eight logits as they lie in memory.
template <typename T>
struct Raw {
  static constexpr int W = kVec * sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ float2 pair(int i) const;   // logits 2 i and 2 i + 1
  __device__ __forceinline__ float at(int i) const {
    const float2 p = pair(i >> 1);
    return i & 1 ? p.y : p.x;
  }
  __device__ __forceinline__ float max() const;
};
template <>
__device__ __forceinline__ float2 Raw<float>::pair(int i) const {
  return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <>
__device__ __forceinline__ float2 Raw<__nv_bfloat16>::pair(int i) const {
  return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 Raw<__half>::pair(int i) const {
  return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
template <>
__device__ __forceinline__ float Raw<float>::max() const {
  float m = max_nan(__uint_as_float(w[0]), __uint_as_float(w[1]));
#pragma unroll
  for (int i = 2; i < 8; ++i) m = max_nan(m, __uint_as_float(w[i]));
  return m;
}
template <>
__device__ __forceinline__ float Raw<__nv_bfloat16>::max() const {
  uint32_t m = w[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
  return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
template <>
__device__ __forceinline__ float Raw<__half>::max() const {
  uint32_t m = w[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&m));
  return max_nan(v.x, v.y);
}
template <typename T>
__device__ __forceinline__ uint32_t nothing();   // a word of logits that are -infinity
template <>
__device__ __forceinline__ uint32_t nothing<float>() { return 0xff800000u; }
template <>
__device__ __forceinline__ uint32_t nothing<__nv_bfloat16>() { return 0xff80ff80u; }
template <>
__device__ __forceinline__ uint32_t nothing<__half>() { return 0xfc00fc00u; }

// The vector of logits [i, i + 8) of a row of n; what lies past n is -infinity.  A row that does not start on 16
// bytes is read in whole 16-byte words around the vector (each holds some of its logits), shifted into place.
template <typename T>
__device__ __forceinline__ void load(Raw<T>& r, const T* row, int i, int n, uint32_t shift) {
  constexpr int W = Raw<T>::W;
  if (i + kVec <= n) {
    const uint8_t* a = reinterpret_cast<const uint8_t*>(row + i) - shift;
    if (shift == 0) {
#pragma unroll
      for (int h = 0; h < W / 4; ++h) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(a) + h);
        r.w[4 * h] = v.x;
        r.w[4 * h + 1] = v.y;
        r.w[4 * h + 2] = v.z;
        r.w[4 * h + 3] = v.w;
      }
      return;
    }
    uint32_t t[W + 4];
#pragma unroll
    for (int h = 0; h <= W / 4; ++h) {
      const uint4 v = *(reinterpret_cast<const uint4*>(a) + h);
      t[4 * h] = v.x;
      t[4 * h + 1] = v.y;
      t[4 * h + 2] = v.z;
      t[4 * h + 3] = v.w;
    }
    if (shift & 8) {
#pragma unroll
      for (int j = 0; j < W + 2; ++j) t[j] = t[j + 2];
    }
    if (shift & 4) {
#pragma unroll
      for (int j = 0; j < W + 1; ++j) t[j] = t[j + 1];
    }
#pragma unroll
    for (int j = 0; j < W; ++j) r.w[j] = __funnelshift_r(t[j], t[j + 1], (shift & 3) * 8);
    return;
  }
#pragma unroll
  for (int j = 0; j < W; ++j) r.w[j] = nothing<T>();
  if (i < n) {
    constexpr int PER = 4 / sizeof(T);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (i + e < n) {
        uint32_t u;
        if constexpr (sizeof(T) == 4) {
          r.w[e] = *reinterpret_cast<const uint32_t*>(row + i + e);
        } else {
          u = *reinterpret_cast<const uint16_t*>(row + i + e);
          r.w[e / PER] = e & 1 ? (r.w[e / PER] & 0xffffu) | u << 16 : (r.w[e / PER] & 0xffff0000u) | u;
        }
      }
    }
  }
}

struct State {
  float m, s, t;
};
// b joins a.
__device__ __forceinline__ State joined(State a, State b) {
  const float m = max_nan(a.m, b.m);
  // a state of nothing (m of -infinity) has no weight, whatever the other's reference is
  const float ga = a.m == -INFINITY ? 0.0f : (a.m - m) * kLog2e, gb = b.m == -INFINITY ? 0.0f : (b.m - m) * kLog2e;
  const float fa = ex2(ga), fb = ex2(gb);
  const float ha = max_nan(ga, -200.0f), hb = max_nan(gb, -200.0f);   // f is 0 there
  return State{m, fmaf(fa, a.s, fb * b.s), fmaf(fa, fmaf(ha, a.s, a.t), fb * fmaf(hb, b.s, b.t))};
}

// Two f32 operations an instruction.
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
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

__device__ __forceinline__ uint32_t map_to_first(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

struct Shared {
  float red[3 * kWarps];
  uint32_t bound[kWarps];
  int scan[kWarps];
  int n_found;
  State state[kMaxParts];
  unsigned long long best[kMaxParts][kMaxK];   // the parts' alternatives, in the first CTA
  unsigned long long sorted[kMaxK];
};

// The places of `mine` ties in the order of the threads, and their total.
__device__ __forceinline__ int block_scan(int mine, int* warps, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) warps[warp] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += warps[i];
    total += warps[i];
  }
  __syncthreads();
  return before + v - mine;
}

template <typename T, bool TOPK>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? (TOPK ? 3 : 4) : 2) logprobs_kernel(const Params p) {
  __shared__ Shared sh;
  __shared__ unsigned long long found[TOPK ? kCandidates : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / p.parts;
  const int part = blockIdx.x - static_cast<int>(row) * p.parts;
  if (p.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA has begun
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const T* x = static_cast<const T*>(p.x) + row * p.stride;
  const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) & 15u);
  State st{-INFINITY, 0.0f, 0.0f};
  int held = 0;   // alternatives of earlier slabs, at the front of `found`
  // a part is one slab, but for vocabularies beyond kMaxParts of them
  for (int slab = part * p.part; slab < p.n_vocab; slab += p.parts * p.part) {
    const int end = min(p.n_vocab, slab + p.part);
    Raw<T> r[kIters];
#pragma unroll
    for (int i = 0; i < kIters; ++i) load<T>(r[i], x, slab + (i * kThreads + threadIdx.x) * kVec, end, shift);
    float m = r[0].max();
#pragma unroll
    for (int i = 1; i < kIters; ++i) m = max_nan(m, r[i].max());
    const float ref = m == -INFINITY ? 0.0f : m;
    const float2 off = make_float2(-ref, -ref), unit = make_float2(kLog2e, kLog2e);
    float2 s2 = make_float2(0.0f, 0.0f), t2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) {
        float2 y = mul2(add2(r[i].pair(e), off), unit);
        // an excluded logit (-infinity) has weight 0 and must not meet its infinite distance
        y.x = max_nan(y.x, -200.0f);
        y.y = max_nan(y.y, -200.0f);
        const float2 w = make_float2(ex2(y.x), ex2(y.y));
        s2 = add2(s2, w);
        t2 = fma2(y, w, t2);
      }
    }
    st = joined(st, State{m, s2.x + s2.y, t2.x + t2.y});
    if constexpr (TOPK) {
      const int nvec = (end - slab + kVec - 1) / kVec;
      const int base = slab + threadIdx.x * kVec;
      // the bound
      uint32_t mine = threadIdx.x < nvec ? key_of(m) : 0u;
      const uint32_t own = mine;
      const int full = min(kWarps, max(1, nvec / 32));   // warps with a logit in every lane
      uint32_t low = 0;
      for (int n = (p.k + full - 1) / full; n > 0; --n) {
        low = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t who = __ballot_sync(0xffffffffu, mine == low);
        if (lane == __ffs(who) - 1) mine = 0u;
      }
      if (lane == 0) sh.bound[warp] = low;
      if (threadIdx.x == 0) sh.n_found = held;
      __syncthreads();
      uint32_t bound = sh.bound[0];
      for (int w = 1; w < full; ++w) bound = min(bound, sh.bound[w]);
      auto collect = [&]() {   // everything above the bound
        if (own > bound) {
#pragma unroll
          for (int i = 0; i < kIters; ++i) {
            if (key_of(r[i].max()) > bound) {
              const int at = base + i * kThreads * kVec;
#pragma unroll
              for (int e = 0; e < kVec; ++e) {
                const uint32_t key = key_of(r[i].at(e));
                if (key > bound && at + e < end) {
                  const int f = atomicAdd(&sh.n_found, 1);
                  if (f < kCandidates)
                    found[f] = static_cast<unsigned long long>(key) << 32 | ~static_cast<uint32_t>(at + e);
                }
              }
            }
          }
        }
        __syncthreads();
      };
      collect();
      if (sh.n_found - held > kPoor) {
        // the k-th largest of the threads' maxima, bit by bit
        uint32_t best = 0;
        for (int b = 31; b >= 0; --b) {
          const uint32_t at = best | 1u << b;
          if (__syncthreads_count(own >= at) >= p.k) best = at;
        }
        if (best > bound) {
          bound = best;
          if (threadIdx.x == 0) sh.n_found = held;
          __syncthreads();
          collect();
        }
      }
      int n = sh.n_found;
      const int want = min(p.k, end - slab);
      if (n - held < want) {
        // ties at the bound, in the order of their indices
        int need = want - (n - held);
#pragma unroll
        for (int i = 0; i < kIters; ++i) {
          if (need > 0) {
            int ties = 0;
            const int at = base + i * kThreads * kVec;
#pragma unroll
            for (int e = 0; e < kVec; ++e) ties += key_of(r[i].at(e)) == bound && at + e < end;
            int total;
            int f = block_scan(ties, sh.scan, total);
#pragma unroll
            for (int e = 0; e < kVec; ++e)
              if (key_of(r[i].at(e)) == bound && at + e < end) {
                if (f < need) found[n + f] = static_cast<unsigned long long>(bound) << 32 | ~static_cast<uint32_t>(at + e);
                ++f;
              }
            n += min(total, need);
            need -= total;
          }
        }
        __syncthreads();
      }
      // the k largest of all, by counting (keys are distinct)
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long key = found[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += found[j] > key;
        if (above < p.k) sh.sorted[above] = key;
      }
      __syncthreads();
      held = min(p.k, n);
      if (threadIdx.x < held) found[threadIdx.x] = sh.sorted[threadIdx.x];
      __syncthreads();
    }
  }
  // threads, then parts
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    State o;
    o.m = __shfl_xor_sync(0xffffffffu, st.m, d);
    o.s = __shfl_xor_sync(0xffffffffu, st.s, d);
    o.t = __shfl_xor_sync(0xffffffffu, st.t, d);
    st = lane & d ? joined(o, st) : joined(st, o);
  }
  if (lane == 0) {
    sh.red[warp] = st.m;
    sh.red[kWarps + warp] = st.s;
    sh.red[2 * kWarps + warp] = st.t;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    st = State{sh.red[0], sh.red[kWarps], sh.red[2 * kWarps]};
#pragma unroll
    for (int i = 1; i < kWarps; ++i) st = joined(st, State{sh.red[i], sh.red[kWarps + i], sh.red[2 * kWarps + i]});
  }
  if (p.parts > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // the first CTA of the row has begun
    if (threadIdx.x == 0) {
      const uint32_t at = map_to_first(smem_u32(&sh.state[part]));
      st_cluster(at, st.m);
      st_cluster(at + 4, st.s);
      st_cluster(at + 8, st.t);
    }
    if (TOPK && threadIdx.x < p.k)
      st_cluster(map_to_first(smem_u32(&sh.best[part][threadIdx.x])), threadIdx.x < held ? found[threadIdx.x] : 0ull);
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (part != 0) {
      return;
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    st = sh.state[0];
    for (int i = 1; i < p.parts; ++i) st = joined(st, sh.state[i]);
  } else {
    if (threadIdx.x == 0) sh.state[0] = st;
    __syncthreads();
    st = sh.state[0];
  }
  const float log_s = log2f(st.s);
  auto log_p = [&](float v) { return fmaf(-kLn2, log_s, v - st.m); };
  if (threadIdx.x == 0) {
    if (p.tokens) {
      const int64_t tok = p.tokens[row];
      float lp = 0.0f;   // -1 asks for nothing
      if (tok >= 0 && tok < p.n_vocab) {
        lp = log_p(to_f32<T>(x[tok]));
      } else if (tok != -1) {
        report_error(DK_ERR_DEVICE_CHECK, kDetToken);
        lp = __uint_as_float(0x7fffffffu);
      }
      p.lp[row] = lp;
    }
    if (p.entropy) p.entropy[row] = kLn2 * (log_s - st.t / st.s);
  }
  if constexpr (TOPK) {
    auto give = [&](int at, unsigned long long key) {
      p.top_ids[row * p.k + at] = static_cast<int64_t>(~static_cast<uint32_t>(key));
      p.top_lp[row * p.k + at] = log_p(value_of(static_cast<uint32_t>(key >> 32)));
    };
    if (p.parts == 1) {
      if (threadIdx.x < held) give(threadIdx.x, found[threadIdx.x]);
    } else {
      const int n = p.parts * p.k;   // at most 256
      if (threadIdx.x < n) {
        const unsigned long long key = sh.best[threadIdx.x / p.k][threadIdx.x % p.k];
        int above = 0;
        for (int a = 0; a < p.parts; ++a)
          for (int j = 0; j < p.k; ++j) above += sh.best[a][j] > key;
        if (key != 0 && above < p.k) give(above, key);
      }
    }
  }
}

}  // namespace logprobs
}  // namespace dk
