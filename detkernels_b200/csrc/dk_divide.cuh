// Divisions by a number that the host knows, as multiplications, after Granlund and Montgomery ("Division by
// invariant integers using multiplication").  Plain C++ as well, so that they can be checked without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define DK_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define DK_HOST_DEVICE inline
#endif

namespace dk {

// Any 32-bit n: with l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1,
// n / d = (t + ((n - t) >> 1)) >> (l - 1), t the high half of m n; d = 1 is n itself.
struct Divisor {
  uint32_t d, m, sh1, sh2;
};
inline Divisor divisor(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  const uint64_t m = ((((1ull << l) - d) << 32) / d) + 1;
  return Divisor{d, static_cast<uint32_t>(m), l < 1 ? l : 1, l > 1 ? l - 1 : 0};
}
DK_HOST_DEVICE uint32_t div_by(uint32_t n, const Divisor& v) {
  const uint32_t t = static_cast<uint32_t>((static_cast<uint64_t>(v.m) * n) >> 32);
  return (t + ((n - t) >> v.sh1)) >> v.sh2;
}
DK_HOST_DEVICE uint32_t ceil_div32(uint32_t a, const Divisor& v) {
  const uint32_t q = div_by(a, v);
  return q + (a != q * v.d);
}

// n < 2^31, in one wide product: m = ceil(2^(31 + l) / d) exceeds 2^(31 + l) / d by e / d with e < d <= 2^l, so that
// n m / 2^(31 + l) exceeds n / d by less than 1 / d.
struct Divisor31 {
  uint32_t m, shift;
};
inline Divisor31 divisor31(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return Divisor31{static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}
DK_HOST_DEVICE uint32_t div_by(uint32_t n, const Divisor31& v) {
  return static_cast<uint32_t>((static_cast<uint64_t>(n) * v.m) >> v.shift);
}

}  // namespace dk
