// What the kernels of a batch of sequences in HBM share: 8-bit elements, entries of integer tensors
// of either type, a token's place in its pages.
#pragma once
#include <string.h>

#include "model_math.hpp"

namespace da {

// OCP e4m3: 4 exponent and 3 mantissa bits, largest 448, no infinities.
struct E4M3 {
  static constexpr int kBytes = 1;
};
constexpr float kE4m3Max = 448.f;

__device__ __forceinline__ float clamp_e4m3(float x) {
  return x != x ? x : fminf(fmaxf(x, -kE4m3Max), kE4m3Max);   // (NaN stays)
}
// Four values, round to nearest even, as the bytes of a dword.
__device__ __forceinline__ uint32_t pack_e4m3(const float *f) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(f[0]), clamp_e4m3(f[1]), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(f[2]), clamp_e4m3(f[3]), w, true);
  return (uint32_t)w;
}

// Entry i of an int32 or int64 tensor (the branch is the same for every lane).
__device__ __forceinline__ int64_t load_index(const void *p, int wide, int64_t i) {
  return wide ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// n / d for 0 <= n < 2^31 by one multiplication: with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1 the quotient is (mulhi(m, n) + n) >> l.
struct Divisor {
  uint32_t mul;
  int32_t shift;
  int32_t d;
};
inline Divisor divisor_of(int32_t d) {
  int l = 0;
  while (((int64_t)1 << l) < d) ++l;
  const uint64_t m = ((((uint64_t)1 << l) - (uint64_t)d) << 32) / (uint64_t)d + 1;
  return Divisor{(uint32_t)m, l, d};
}
__device__ __forceinline__ int divide(int n, const Divisor &by) {
  return (int)((__umulhi(by.mul, (uint32_t)n) + (uint32_t)n) >> by.shift);
}

}  // namespace da
