// Row blocks of the fp8 linear in registers: loads, the block's maximum, its power-of-two scale and codes.
#pragma once

#include <cuda_fp8.h>

#include "fp8_args.cuh"

namespace moss {
namespace fp8 {

template <int kKind>
struct Raw {  // 8 values
  uint32_t w[kKind == kF32 ? 8 : 4];
};

// Exponent p of the row scale: the least with amax <= 448 * 2^p = 1.75 * 2^(p + 8).
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  return static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

template <int kKind>
__device__ __forceinline__ Raw<kKind> load_raw(const void* x, int64_t at) {
  Raw<kKind> r;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + at * (kKind == kF32 ? 4 : 2));
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r)) / 16; ++i) {
    const uint4 v = __ldg(p + i);
    r.w[4 * i] = v.x;
    r.w[4 * i + 1] = v.y;
    r.w[4 * i + 2] = v.z;
    r.w[4 * i + 3] = v.w;
  }
  return r;
}
template <int kKind>
__device__ __forceinline__ float amax_of(const Raw<kKind>& r) {
  if constexpr (kKind == kF32) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(__uint_as_float(r.w[i])));
    return m;
  } else if constexpr (kKind == kBF16) {
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&r.w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&r.w[i])));
    return max_nan(__low2float(m), __high2float(m));
  } else {
    __half2 m = __habs2(*reinterpret_cast<const __half2*>(&r.w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&r.w[i])));
    return max_nan(__low2float(m), __high2float(m));
  }
}
template <int kKind>
__device__ __forceinline__ void values_of(const Raw<kKind>& r, float (&v)[8]) {
  if constexpr (kKind == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kKind == kBF16) {
        v[2 * i] = __uint_as_float(r.w[i] << 16);
        v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}

// Codes of the 8 values of one lane for a block whose largest magnitude is `amax`, and the block's scale.
__device__ __forceinline__ uint2 block_codes(const float (&v)[8], float amax, float& scale) {
  // a block with an infinity or a NaN has no scale: NaN, and so has every product with it
  const bool finite = amax < __uint_as_float(0x7f800000u);
  const int p = finite ? scale_exponent(amax) : 0;
  const float inv = pow2(-p);
  uint2 q;
  q.x = codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  q.y = codes4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
  scale = finite ? pow2(p) : __uint_as_float(0x7fffffffu);
  return q;
}
// Over the 16 lanes that hold one row's block.
__device__ __forceinline__ float half_warp_max(float amax) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  return amax;
}

}  // namespace fp8
}  // namespace moss
