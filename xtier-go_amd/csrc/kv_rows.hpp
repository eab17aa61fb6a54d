// What the kernels that move rows into and out of KV caches share: pieces of rows as FP32, and the largest magnitude of a
// block over the lanes that share it.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "rowops.hpp"

namespace xtg::hip {

// N consecutive elements of a row as FP32 (N: 1, 2, 4 or a multiple of 8, aligned alike).
template <int N>
__device__ inline void load_row4(const float* p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = *p;
    return;
  }
  if constexpr (N == 2) {
    const float2 a = *reinterpret_cast<const float2*>(p);
    x[0] = a.x, x[1] = a.y;
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const float4 a = *reinterpret_cast<const float4*>(p + e);
    x[e] = a.x, x[e + 1] = a.y, x[e + 2] = a.z, x[e + 3] = a.w;
  }
}
template <int N>
__device__ inline void load_row4(const __bf16* p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = (float)*p;
    return;
  }
  if constexpr (N == 2) {
    const uint32_t a = *reinterpret_cast<const uint32_t*>(p);
    x[0] = __uint_as_float(a << 16), x[1] = __uint_as_float(a & 0xffff0000u);
    return;
  }
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 8) {
      const uint4 a = *reinterpret_cast<const uint4*>(p + e);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) x[e + 2 * c] = __uint_as_float(w[c] << 16), x[e + 2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const uint2 a = *reinterpret_cast<const uint2*>(p + e);
    x[e] = __uint_as_float(a.x << 16), x[e + 1] = __uint_as_float(a.x & 0xffff0000u);
    x[e + 2] = __uint_as_float(a.y << 16), x[e + 3] = __uint_as_float(a.y & 0xffff0000u);
  }
}

template <int N>
__device__ inline void store_row4(float* p, const float (&x)[N]) {
  if constexpr (N == 1) {
    *p = x[0];
    return;
  }
  if constexpr (N == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
}
// Rounded to nearest even (an FP8 row's values; NVFP4 and BF16 rows' are exact).
template <int N>
__device__ inline void store_row4(__bf16* p, const float (&x)[N]) {
  if constexpr (N == 1) {
    *p = (__bf16)x[0];
    return;
  }
  if constexpr (N == 2) {
    const __bf16 b[2] = {(__bf16)x[0], (__bf16)x[1]};
    *reinterpret_cast<uint32_t*>(p) = __builtin_bit_cast(uint32_t, b);
    return;
  }
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 8) {
      const __bf16 b[8] = {(__bf16)x[e], (__bf16)x[e + 1], (__bf16)x[e + 2], (__bf16)x[e + 3],
                           (__bf16)x[e + 4], (__bf16)x[e + 5], (__bf16)x[e + 6], (__bf16)x[e + 7]};
      *reinterpret_cast<uint4*>(p + e) = __builtin_bit_cast(uint4, b);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const __bf16 b[4] = {(__bf16)x[e], (__bf16)x[e + 1], (__bf16)x[e + 2], (__bf16)x[e + 3]};
    *reinterpret_cast<uint2*>(p + e) = __builtin_bit_cast(uint2, b);
  }
}

// 8 E4M3 codes' values times a scale.
__device__ inline void fp8_values(uint2 w, float s, float (&x)[8]) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
  const auto c = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true);
  x[0] = a[0] * s, x[1] = a[1] * s, x[2] = b[0] * s, x[3] = b[1] * s;
  x[4] = c[0] * s, x[5] = c[1] * s, x[6] = d[0] * s, x[7] = d[1] * s;
}

// The larger of the magnitudes' bits: that of a value that is not finite is above every finite one's.
__device__ inline uint32_t max_bits(uint32_t m, float x) { return max(m, __float_as_uint(x) & 0x7fffffffu); }
constexpr uint32_t kInfBits = 0x7f800000u;

template <int CTRL>
__device__ inline uint32_t dpp_max(uint32_t v) {
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, false)));
}

// The block's maximum over the lanes that share it: LANES neighbours.
template <int LANES>
__device__ inline uint32_t over_block(uint32_t m) {
  if constexpr (LANES >= 2) m = dpp_max<kDppXor1>(m);
  if constexpr (LANES >= 4) m = dpp_max<kDppXor2>(m);
  if constexpr (LANES >= 8) m = dpp_max<kDppHalfMirror>(m);
  if constexpr (LANES >= 16) m = dpp_max<kDppMirror>(m);
  return m;
}

}  // namespace xtg::hip
