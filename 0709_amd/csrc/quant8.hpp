// The two 8-bit value types of quantised caches, e4m3 (OCP fp8) and int8:
// conversions between their codes and fp32.
#pragma once

#include "common.hpp"

namespace atlas {

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int CACHE>
struct Quant8;

template <>
struct Quant8<ATLAS_CACHE_E4M3> {
  // four codes -> four values
  static __device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    f[0] = lo[0];
    f[1] = lo[1];
    f[2] = hi[0];
    f[3] = hi[1];
  }
  // The conversion rounds to nearest even and makes NaN of what lies past 448;
  // values are clamped before it.  NaN passes the comparisons and stays.
  static __device__ __forceinline__ float clamp(float x) { return x > 448.f ? 448.f : (x < -448.f ? -448.f : x); }
  static __device__ __forceinline__ uint32_t encode4(const float (&f)[4]) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp(f[0]), clamp(f[1]), 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(clamp(f[2]), clamp(f[3]), w, true));
  }
  // exponent e of the least 2^e with amax <= 448 * 2^e, 448 = 0.875 * 2^9
  static constexpr int kBits = 9;
  static constexpr uint32_t kTopMantissa = 0x600000;  // 0.875 = 1.75 / 2
};

template <>
struct Quant8<ATLAS_CACHE_INT8> {
  static __device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = float(int(w << (24 - 8 * i)) >> 24);
  }
  static __device__ __forceinline__ uint32_t encode4(const float (&f)[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = __builtin_amdgcn_fmed3f(f[i], -127.f, 127.f);
      const int v = f[i] == f[i] ? int(__builtin_rintf(c)) : 0;
      w |= (uint32_t(v) & 0xffu) << (8 * i);
    }
    return w;
  }
  static constexpr int kBits = 7;
  static constexpr uint32_t kTopMantissa = 0x7e0000;  // 127 / 128 = (127 / 64) / 2
};

// Exponent of the least power of two 2^e with amax <= top * 2^e, -126 for a
// block of zeros (or of values below every scale); amax is finite.
template <int CACHE>
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int x = int(bits >> 23) - 126;  // amax = m * 2^x, 0.5 <= m < 1 (subnormals: at most 2^-126, clamped below)
  const int e = x - Quant8<CACHE>::kBits + ((bits & 0x7fffffu) > Quant8<CACHE>::kTopMantissa ? 1 : 0);
  return e < -126 ? -126 : e;
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

}  // namespace atlas
