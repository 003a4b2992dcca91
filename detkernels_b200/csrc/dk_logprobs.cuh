// Log probabilities of given tokens, the entropy and the most likely alternatives of rows of logits.
//
// With a row's logits x, any reference m and y = (x - m) log2 e, S = sum 2^y and T = sum y 2^y give log p(t) = x_t - m -
// log S and the entropy ln 2 (log2 S - T / S), and states (m, S, T) join by S' = f S, T' = f (T + g S), g = (m - m') log2 e,
// f = 2^g.  The difference is taken before the product, so that logits of any size (a type's lowest value among
// them) keep their distances.  One pass over the row, bound by its bytes.
//
// A row is cut into passes of 16 KB, and the passes of long rows into eight parts, by the vocabulary's size alone.  In a
// pass a warp takes 2 KB side by side, a thread four 16-byte vectors of them, against its own maximum; it joins its passes,
// then its parts, in order, and the lanes, then the warps, are joined last.  So few rows may give each part a CTA of its own
// (a cluster, whose first CTA gathers the threads' states in its shared memory), and many rows a CTA each, which goes through
// all parts: the same bits, with neither scratch nor a second launch.  Passes come into a ring in shared memory by bulk
// copies, which keep more of them in flight than registers would, and at any alignment of a row: the copy takes the whole
// 16-byte words around it, and a thread shifts its vectors into place.
//
// The alternatives are chosen from the same stage.  A bound below the k-th largest logit of the first pass is had from the
// threads' maxima: in each of w warps the ceil(k / w)-th largest is at most it, and so is the least of these (of warps whose
// threads all have their logits: a lane with fewer has a lower maximum, and 3 us were lost to a poor bound).  What reaches the
// bound (about twice k) is collected and ranked by counting, equal ones by their indices.  From then on the k-th largest
// so far is the bound, and only what lies above it is collected; a pass costs one barrier.  Where a bound is poor (logits in
// order), the k-th largest of the pass's maxima is sought and takes its place; the pass then gives k alternatives by itself,
// ties in the order of their indices.
//
// Measured, in a graph, logits out of L2: 4096 rows of 50,001 bf16 94 us (4.4 TB/s; the exponential unit is 56 % busy, the
// issue slots 61 %: without exponentials 79 us, with a quarter of the sums 69); 1531 of 32,000 f32 with 5 alternatives
// 55 us (3.6 TB/s, barriers), without any 38 (5.1); 8 of 32,000 bf16 with 20 alternatives 7.9 us (latency), without 3.8.
// Logits of -infinity or the type's lowest value make their warp form its sums twice (below): one in 1000 of them 159 us in
// place of 94, 63 for 55 and 8.6 for 8.2, nearly all 177, 96 and 17; -1e9 in their place costs the sums nothing.
#pragma once

#include "dk_common.cuh"

namespace dk {
namespace logprobs {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kIters = 4;                       // 16-byte vectors of a pass that a thread takes
constexpr int kMaxParts = 8;                    // a portable cluster
constexpr int kMaxK = 32;
constexpr int kCandidates = 1160;               // above the k-th largest maximum lie at most (k - 1) * 32 logits
constexpr int kPoor = 256;                      // a bound with more above it is worth improving
constexpr int kMany = 128;                      // candidates worth ranking before the row's end
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
static_assert((kMaxK - 1) * 32 + 2 * kMaxK + 16 + kMaxK < kCandidates, "candidates");   // so many, those before, and ties

enum : int {
  kDetToken = 0x650,   // a token outside the vocabulary (and not -1)
  kDetFull = 0x651,
};

struct Params {
  const void* x;
  int64_t stride, n_rows;
  int32_t n_vocab, parts, part;     // parts a row, logits a part (whole passes)
  int32_t split;                    // a CTA a part, else a row
  int32_t stages;                   // of the ring
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

// A vector of logits as it lies in memory.
template <typename T>
struct Raw {
  static constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  // kNone: nothing but -infinity; kFar: logits of weight 0 beside any above kFloor
  static constexpr uint32_t kFar = sizeof(T) == 4 ? 0xf149f2cau : std::is_same<T, __half>::value ? 0xfbfffbffu : 0xf14af14au;
  static constexpr float kFloor = std::is_same<T, __half>::value ? -6e4f : -1e29f;
  uint32_t w[4];
  __device__ __forceinline__ float2 pair(int i) const;   // logits 2 i and 2 i + 1
  __device__ __forceinline__ float at(int i) const {
    const float2 p = pair(i >> 1);
    return i & 1 ? p.y : p.x;
  }
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
// The larger ones of two words' logits, and the largest of a word's.
template <typename T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t max_word<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
}
template <>
__device__ __forceinline__ uint32_t max_word<__nv_bfloat16>(uint32_t a, uint32_t b) {
  asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
template <>
__device__ __forceinline__ uint32_t max_word<__half>(uint32_t a, uint32_t b) {
  asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
template <typename T>
__device__ __forceinline__ float max_of(uint32_t a);
template <>
__device__ __forceinline__ float max_of<float>(uint32_t a) { return __uint_as_float(a); }
template <>
__device__ __forceinline__ float max_of<__nv_bfloat16>(uint32_t a) {
  return max_nan(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
}
template <>
__device__ __forceinline__ float max_of<__half>(uint32_t a) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a));
  return max_nan(v.x, v.y);
}

// A vector from the 16-byte word in which it starts and the next one; Q: whole 32-bit words, bits: and bits behind its start.
template <typename T, int Q>
__device__ __forceinline__ Raw<T> shifted(const uint4& a, const uint4& b, uint32_t bits) {
  const uint32_t t[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  Raw<T> r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.w[j] = __funnelshift_r(t[Q + j], t[(Q + j + 1) & 7], bits);
  return r;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Vectors v, v + 32, ... of a warp's stage whose row starts `shift` bytes behind a 16-byte word (the same for the whole row).
template <typename T, bool ALIGNED, int N>
__device__ __forceinline__ void vectors_at(Raw<T> (&r)[N], const uint8_t* stage, int v, uint32_t shift) {
  const uint4* at = reinterpret_cast<const uint4*>(stage) + v;
  auto all = [&](auto q) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = shifted<T, q>(at[i * 32], at[i * 32 + 1], (shift & 3) * 8);
  };
  if (ALIGNED || shift == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint4 a = at[i * 32];
      r[i] = Raw<T>{{a.x, a.y, a.z, a.w}};
    }
  } else {
    switch (shift >> 2) {
      case 0: all(std::integral_constant<int, 0>()); break;
      case 1: all(std::integral_constant<int, 1>()); break;
      case 2: all(std::integral_constant<int, 2>()); break;
      default: all(std::integral_constant<int, 3>()); break;
    }
  }
}
// Of the vector's logits only the first n are the row's, the others become `none`.
template <typename T>
__device__ __forceinline__ void cut(Raw<T>& r, int n, uint32_t none = Raw<T>::kNone) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r.w[e] = e < n ? r.w[e] : none;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r.w[e] = 2 * e + 1 < n ? r.w[e] : 2 * e < n ? (r.w[e] & 0xffffu) | (none & 0xffff0000u) : none;
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
  float top[2][kWarps], s[2][kWarps], t[2][kWarps];   // by row parity: the warps' states
  uint32_t bound[kWarps];
  int scan[kWarps];
  int n_found[3];   // by pass: what is being counted, what is read, what is 0
  __align__(16) unsigned long long best[kMaxParts * kMaxK];   // the parts' alternatives (k of each), in the first CTA of a split row
  unsigned long long sorted[kMaxK];
};

// A pass, its stage of the ring, and CTAs an SM.
template <typename T, bool TOPK>
struct Cfg {
  static constexpr int VEC = 16 / sizeof(T), ITERS = kIters;   // logits a vector, vectors a thread
  static constexpr int SEG = 32 * ITERS * VEC;                 // logits of a pass that are a warp's
  static constexpr int PASS = kWarps * SEG;
  static constexpr int STAGE = PASS * sizeof(T) + 128;         // the words around a pass
  static constexpr int STAGES = 8;                             // at most
  static constexpr int CTAS = 4;
  static constexpr int STATES = 3 * kMaxParts * kThreads * 4;  // behind the ring of a split row: its parts' threads' states
  static constexpr int STATIC = sizeof(Shared) + (TOPK ? kCandidates * 8 : 8) + STAGES * 8 + 128;
};

// The sum of the lanes before this one, and of all.
__device__ __forceinline__ int warp_scan(int mine, int& total) {
  const int lane = threadIdx.x & 31;
  int v = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  total = __shfl_sync(0xffffffffu, v, 31);
  return v - mine;
}

// How many of n keys are larger.
__device__ __forceinline__ int count_above(const unsigned long long* keys, int n, unsigned long long key) {
  int above = 0;
#pragma unroll 4
  for (int j = 0; j + 1 < n; j += 2) {
    const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + j);
    above += (two.x > key) + (two.y > key);
  }
  return above + (n & 1 && keys[n - 1] > key);
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T, bool TOPK, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, Cfg<T, TOPK>::CTAS) logprobs_kernel(const Params p) {
  using C = Cfg<T, TOPK>;
  constexpr int VEC = C::VEC, ITERS = C::ITERS, SEG = C::SEG, kPass = C::PASS;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ Shared sh;
  __shared__ __align__(16) unsigned long long found[TOPK ? kCandidates : 1];
  __shared__ __align__(8) uint64_t full[C::STAGES];
  float(*threads)[kMaxParts][kThreads] = reinterpret_cast<float(*)[kMaxParts][kThreads]>(ring + p.stages * C::STAGE);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  if (p.split) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA has begun
  if (tid < 3) sh.n_found[tid] = 0;
  if (tid < C::STAGES) {
    mbar_init(&full[tid], 1);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  if (tid == 0) pdl_launch_dependents();
  // the passes that this CTA goes through: [j0, j0 + nj) of rows row0, row0 + row_step, ...
  const uint32_t n_rows = static_cast<uint32_t>(p.n_rows), row_step = p.split ? n_rows : gridDim.x;
  const uint32_t row0 = p.split ? blockIdx.x / static_cast<uint32_t>(p.parts) : blockIdx.x;
  const int first_part = p.split ? static_cast<int>(blockIdx.x - row0 * p.parts) : 0;
  const int per = p.part / kPass, j0 = first_part * per, to_end = (p.n_vocab + kPass - 1) / kPass - j0;
  const int nj = p.split ? min(to_end, per) : to_end;
  constexpr int kSize = static_cast<int>(sizeof(T));
  const int64_t row_bytes = static_cast<int64_t>(row_step) * p.stride * kSize;
  const uint8_t* x_bytes = static_cast<const uint8_t*>(p.x) + row0 * p.stride * kSize;
  bool abort_flag = false;
  const int from = j0 * kPass;                         // the CTA's first logit of a row
  // The next pass that is not on its way (warp 0), with the words around it.
  const uint8_t* ahead = x_bytes + static_cast<int64_t>(from) * kSize;
  int ahead_left = p.n_vocab - from, ahead_n = nj;     // logits from there to the row's end; passes to go
  uint32_t ahead_rows = row0 < n_rows ? (n_rows - row0 + row_step - 1) / row_step : 0;
  auto issue = [&](int stage) {
    if (ahead_rows == 0) return;
    const uint32_t before = ALIGNED ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ahead) & 15u);
    const uint32_t bytes = (before + static_cast<uint32_t>(min(kPass, ahead_left) * kSize) + 15u) & ~15u;
    if (elect_one()) {
      mbar_arrive_expect_tx(&full[stage], bytes);
      bulk_load_1d(ring + stage * C::STAGE, ahead - before, bytes, &full[stage]);
    }
    __syncwarp();
    ahead += kPass * kSize;
    ahead_left -= kPass;
    if (--ahead_n == 0) {
      ahead_n = nj;
      ahead_left += nj * kPass;
      ahead += row_bytes - static_cast<int64_t>(nj) * (kPass * kSize);
      --ahead_rows;
    }
  };
  if (warp == 0)
    for (int s = 0; s < p.stages; ++s) issue(s);
  int slot = 0;         // of the count of found ones
  int held = 0;         // alternatives so far, at the front of `found`
  int n = 0;            // and candidates behind them
  uint32_t bound = 0;   // below the k-th largest logit; once there are k of them, the k-th itself
  int flip = 0;         // row parity
  int stage = 0;
  uint32_t phase = 0;
  for (uint32_t row = row0; row < n_rows; row += row_step, x_bytes += row_bytes) {
    const uint32_t shift = ALIGNED ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x_bytes) & 15u);
    float asked = 0.0f;   // thread 0: the logit of the row's token, fetched long before it is used
    if (tid == 0 && first_part == 0 && p.tokens) {
      const int64_t tok = p.tokens[row];
      if (tok >= 0 && tok < p.n_vocab) asked = to_f32<T>(reinterpret_cast<const T*>(x_bytes)[tok]);
    }
    State st{-INFINITY, 0.0f, 0.0f}, in_part{-INFINITY, 0.0f, 0.0f};
    int left = p.n_vocab - from - warp * SEG;   // logits from the warp's first of the pass on
    int in = per;                      // passes to go in the part
    if (TOPK) held = n = 0;
    for (int j = 0; j < nj; ++j, left -= kPass) {
      const uint8_t* here = ring + stage * C::STAGE + warp * (SEG * kSize);
      mbar_wait(&full[stage], phase, kDetFull, abort_flag);
      State now{-INFINITY, 0.0f, 0.0f};
      if (left > 0) {
        Raw<T> r[ITERS];
        vectors_at<T, ALIGNED>(r, here, lane, shift);
        if (left < SEG) {
#pragma unroll
          for (int i = 0; i < ITERS; ++i) cut(r[i], left - (i * 32 + lane) * VEC);
        }
        uint32_t mw = Raw<T>::kNone;
#pragma unroll
        for (int i = 0; i < ITERS; ++i)
          mw = max_word<T>(mw, max_word<T>(max_word<T>(r[i].w[0], r[i].w[1]), max_word<T>(r[i].w[2], r[i].w[3])));
        now.m = max_of<T>(mw);
        const float ref = now.m == -INFINITY ? 0.0f : now.m, c = __fmul_rn(ref, kLog2e);
        const float2 unit = make_float2(kLog2e, kLog2e);
        float2 s2[2], t2[2];
        auto add = [&](float2 y, int e) {
          const float2 w = make_float2(ex2(y.x), ex2(y.y));
          s2[e & 1] = add2(s2[e & 1], w);
          t2[e & 1] = fma2(y, w, t2[e & 1]);
        };
        auto sum_up = [&]() {
          s2[0] = add2(s2[0], s2[1]);
          t2[0] = add2(t2[0], t2[1]);
          now.s = s2[0].x + s2[0].y;
          now.t = t2[0].x + t2[0].y;
        };
        // (what is not the row's is -infinity no more, which would cost the second pass below)
        if (left < SEG) {
#pragma unroll
          for (int i = 0; i < ITERS; ++i) cut(r[i], left - (i * 32 + lane) * VEC, Raw<T>::kFar);
        }
        // y = x log2 e - c, c = m log2 e rounded: one operation for two logits.  What c is off by is put right in the sums.
        s2[0] = s2[1] = t2[0] = t2[1] = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < ITERS; ++i)
#pragma unroll
          for (int e = 0; e < VEC / 2; ++e) add(fma2(r[i].pair(e), unit, make_float2(-c, -c)), e);
        sum_up();
        const float d = fmaf(-ref, kLog2e, c), f = ex2(d);   // (x - m) log2 e = y + d
        now.t = f * fmaf(d, now.s, now.t);
        now.s = f * now.s;
        // An excluded logit (-infinity, or as far away) has weight 0 and must not meet its infinite distance, and a product may
        // be beyond f32: once more, differences first, with distances that end where weights have long been 0.  So, too, where
        // c is off by much (logits from 7e8 on: c's last place is 128 there): from 126 on the maximum's own weight 2^-d would
        // be 0, and the sums' roundings count d times in T.
        if (!(fabsf(now.t) < INFINITY) || fabsf(d) > 32.0f || (left < SEG && now.m <= Raw<T>::kFloor && now.m != -INFINITY)) {
          s2[0] = s2[1] = t2[0] = t2[1] = make_float2(0.0f, 0.0f);
#pragma unroll 1
          for (int i = 0; i < ITERS; ++i) {
            Raw<T> v[1];
            vectors_at<T, ALIGNED>(v, here, i * 32 + lane, shift);
            cut(v[0], left - (i * 32 + lane) * VEC);
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) {
              const float2 y = mul2(add2(v[0].pair(e), make_float2(-ref, -ref)), unit);
              add(make_float2(max_nan(y.x, -200.0f), max_nan(y.y, -200.0f)), e);
            }
          }
          sum_up();
        }
      }
      const float m = now.m;
      in_part = in == per ? now : joined(in_part, now);
      if (--in == 0 || j + 1 == nj) {
        st = j < per ? in_part : joined(st, in_part);
        in = per;
      }
      if constexpr (TOPK) {
        const int begin = (j0 + j) * kPass, end = min(p.n_vocab, begin + kPass);
        const int nvec = (end - begin + VEC - 1) / VEC;
        const uint32_t own = warp * (SEG / VEC) + lane < nvec ? key_of(m) : 0u;
        if (held < p.k) {
          // the bound from the threads' maxima
          uint32_t mine = own;
          const int warps = max(1, nvec / (SEG / VEC));   // whose threads all have as many logits
          uint32_t low = 0;
          for (int a = (p.k + warps - 1) / warps; a > 0; --a) {
            low = __reduce_max_sync(0xffffffffu, mine);
            const uint32_t who = __ballot_sync(0xffffffffu, mine == low);
            if (lane == __ffs(who) - 1) mine = 0u;
          }
          if (lane == 0) sh.bound[warp] = low;
          __syncthreads();
          bound = sh.bound[0];
          for (int w = 1; w < warps; ++w) bound = min(bound, sh.bound[w]);
        }
        // Everything above `lim`, behind the n that there are; how many.  A warp takes its threads with a larger maximum some at
        // a time, a lane a logit: one place in the list is asked for all that they have.
        auto collect = [&](uint32_t lim) {
          constexpr int OWN = ITERS * VEC, AT_ONCE = 32 / OWN, Q = 4 / AT_ONCE;   // a thread's logits, threads at once, times
          uint32_t who = __ballot_sync(0xffffffffu, own > lim);
          const T* logits = reinterpret_cast<const T*>(here + shift);
          const int off = lane % OWN / VEC * (32 * VEC) + lane % VEC;
          while (who) {
            uint32_t key[Q], hits[Q];
            int at[Q];
            int n_hits = 0;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              int thread = who ? __ffs(who) - 1 : -1;
              who &= who - 1;
              if (AT_ONCE == 2) {
                const int other = who ? __ffs(who) - 1 : -1;
                who &= who - 1;
                if (lane >= OWN) thread = other;
              }
              at[q] = thread >= 0 ? thread * VEC + off : left;
              key[q] = at[q] < left ? key_of(to_f32<T>(logits[at[q]])) : 0u;
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              hits[q] = __ballot_sync(0xffffffffu, key[q] > lim);
              n_hits += __popc(hits[q]);
            }
            int f = 0;
            if (lane == 0) f = atomicAdd(&sh.n_found[slot], n_hits);
            f = n + __shfl_sync(0xffffffffu, f, 0);
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              const int to = f + __popc(hits[q] & ((1u << lane) - 1));
              if ((hits[q] >> lane & 1u) && to < kCandidates)
                found[to] = static_cast<unsigned long long>(key[q]) << 32 | ~static_cast<uint32_t>(begin + warp * SEG + at[q]);
              f += __popc(hits[q]);
            }
          }
          __syncthreads();
          return sh.n_found[slot];
        };
        // A bound from this pass's logits: at it, too, they may be alternatives.  (Every logit's key is above 0.)
        bool fresh = held < p.k;
        int got = collect(fresh && bound > 0 ? bound - 1 : bound);
        bool ties = false;
        if (got > kPoor) {
          // the k-th largest of the threads' maxima, bit by bit
          uint32_t best = 0;
          for (int b = 31; b >= 0; --b) {
            const uint32_t to = best | 1u << b;
            if (__syncthreads_count(own >= to) >= p.k) best = to;
          }
          if (fresh || best > bound) {
            bound = max(bound, best);
            fresh = ties = true;
            if (tid == 0) sh.n_found[slot] = 0;
            __syncthreads();
            got = collect(bound);
          }
        }
        n += got;
        slot = slot == 2 ? 0 : slot + 1;
        if (tid == 0) sh.n_found[slot == 2 ? 0 : slot + 1] = 0;   // read by all before this pass's barrier, counted in after the next
        if (ties) {
          // those at the bound, in the order of their indices, until the pass has given k
          const int need = min(p.k, end - begin) - got;
          if (need > 0) {
            auto tie = [&](int i, int e) {   // the logit itself: a tie, or -1
              const int at = (i * 32 + lane) * VEC + e;
              return at < left && key_of(to_f32<T>(reinterpret_cast<const T*>(here + shift)[at])) == bound ? at : -1;
            };
            int mine = 0;
#pragma unroll 1
            for (int i = 0; i < ITERS; ++i)
#pragma unroll
              for (int e = 0; e < VEC; ++e) mine += tie(i, e) >= 0;
            const int all = __reduce_add_sync(0xffffffffu, mine);
            if (lane == 0) sh.scan[warp] = all;
            __syncthreads();
            int total = 0, f = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              if (w < warp) f += sh.scan[w];
              total += sh.scan[w];
            }
#pragma unroll 1
            for (int i = 0; i < ITERS && f < need; ++i) {
              int ties = 0, sum;
#pragma unroll
              for (int e = 0; e < VEC; ++e) ties += tie(i, e) >= 0;
              int g = f + warp_scan(ties, sum);
              f += sum;
              if (ties == 0) continue;
#pragma unroll 1
              for (int e = 0; e < VEC && g < need; ++e) {
                const int at = tie(i, e);
                if (at >= 0) found[n + g++] = static_cast<unsigned long long>(bound) << 32 | ~static_cast<uint32_t>(begin + warp * SEG + at);
              }
            }
            n += min(total, need);
          }
        }
        if (fresh || n > min(kMany, 2 * p.k + 16) || (j + 1 == nj && n > held)) {
          // the k largest so far, by counting (keys are distinct)
          if (ties) __syncthreads();
          for (int i = tid; i < n; i += kThreads) {
            const unsigned long long key = found[i];
            const int above = count_above(found, n, key);
            if (above < p.k) sh.sorted[above] = key;
          }
          __syncthreads();
          held = min(p.k, n);   // (k of the first pass on, but for a row that has no more)
          if (tid < held) found[tid] = sh.sorted[tid];
          if (held == p.k) bound = static_cast<uint32_t>(sh.sorted[p.k - 1] >> 32);   // an equal logit behind it comes later
          n = held;
        }
      }
      if (!TOPK) __syncthreads();   // the stage has been read
      if (warp == 0) issue(stage);
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (p.split) {
      const int part = first_part;
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // the first CTA of the row has begun
      st_cluster(map_to_first(smem_u32(&threads[0][part][tid])), st.m);
      st_cluster(map_to_first(smem_u32(&threads[1][part][tid])), st.s);
      st_cluster(map_to_first(smem_u32(&threads[2][part][tid])), st.t);
      if (TOPK && tid < p.k) st_cluster(map_to_first(smem_u32(&sh.best[part * p.k + tid])), tid < held ? sh.sorted[tid] : 0ull);
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      if (part != 0) return;   // a split row is all that its CTAs do
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      for (int q = 0; q < p.parts; ++q) {
        const State o{threads[0][q][tid], threads[1][q][tid], threads[2][q][tid]};
        st = q == 0 ? o : joined(st, o);
      }
    }
    // the lanes against their warp's maximum, then the warps against the row's
    auto rebased = [](State a, float to) {
      const float g = a.m == -INFINITY ? 0.0f : (a.m - to) * kLog2e, f = ex2(g);
      return State{to, f * a.s, f * fmaf(max_nan(g, -200.0f), a.s, a.t)};
    };
    st = rebased(st, warp_max_nan(st.m));
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      st.s += __shfl_xor_sync(0xffffffffu, st.s, d);
      st.t += __shfl_xor_sync(0xffffffffu, st.t, d);
    }
    if (lane == 0) {
      sh.top[flip][warp] = st.m;
      sh.s[flip][warp] = st.s;
      sh.t[flip][warp] = st.t;
    }
    __syncthreads();
    if (warp == 0 || p.split) {
      float top = sh.top[flip][0], s = 0.0f, t = 0.0f;
#pragma unroll
      for (int i = 1; i < kWarps; ++i) top = max_nan(top, sh.top[flip][i]);
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const State o = rebased(State{sh.top[flip][i], sh.s[flip][i], sh.t[flip][i]}, top);
        s += o.s;
        t += o.t;
      }
      const float log_s = log2f(s);
      auto log_p = [&](float v) { return fmaf(-kLn2, log_s, v - top); };
      if (tid == 0 && p.entropy) p.entropy[row] = kLn2 * (log_s - t / s);
      if (tid == 0 && p.tokens) {
        const int64_t tok = p.tokens[row];
        float lp = 0.0f;   // -1 asks for nothing
        if (tok >= 0 && tok < p.n_vocab) {
          lp = log_p(asked);
        } else if (tok != -1) {
          report_error(DK_ERR_DEVICE_CHECK, kDetToken);
          lp = __uint_as_float(0x7fffffffu);
        }
        p.lp[row] = lp;
      }
      if constexpr (TOPK) {
        auto give = [&](int to, unsigned long long key) {
          const int64_t at = static_cast<int64_t>(row) * p.k + to;
          p.top_ids[at] = static_cast<int64_t>(~static_cast<uint32_t>(key));
          p.top_lp[at] = log_p(value_of(static_cast<uint32_t>(key >> 32)));
        };
        if (!p.split) {
          if (lane < held) give(lane, sh.sorted[lane]);   // (the next row's come behind more barriers)
        } else {
          const int all = p.parts * p.k;   // at most 256
          if (tid < all) {
            const unsigned long long key = sh.best[tid];
            const int above = count_above(sh.best, all, key);
            if (key != 0 && above < p.k) give(above, key);
          }
        }
      }
    }
    flip ^= 1;
  }
}

}  // namespace logprobs
}  // namespace dk
