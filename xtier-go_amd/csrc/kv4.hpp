// The NVFP4 KV cache: its device layout, and its arithmetic as the store, the read-back and the attention share it.
//
// For each (slot, KV head) and each 16 dims of K and of V: one E4M3 scale s and 16 E2M1 codes c; the value is
// c * s * global, where the cache's two globals (K's and V's) are powers of two. A lane's codes and scales are what it
// holds of a matrix operand of 16-bit values:
//   K codes: per head, per 16-slot block, per chunk of 128 dims (64-dim heads: one of 64), 64 lanes of 16 (8) bytes;
//     lane (g, i) has slot i of the block and the chunk's dims 32 g .. +32 (16 g .. +16), even dims in the low nibbles.
//     Bytes 4 c .. +4 are the lane's A entry of product step c of v_mfma_f32_16x16x32 (keys x dims).
//   K scales: in the same order, 2 (1) bytes a lane: the layout of the NVFP4 weights' tiles.
//   V codes: per head, per tile of 32 slots, per 4 dims of a lane, 64 lanes of 16 bytes; lane (g, i) has dims
//     i ND + dd, dd = 0 .. ND - 1 (ND = head_dim / 16), and of each one word: nibble e is the code of slot
//     4 g + e (e < 4) or 16 + 4 g + e - 4. A word is the lane's A entry (dims x keys) of the P.V product whose B entry
//     is what the lane holds of the score tile. A lane's dims are one scale block's, or part of one.
//   V scales: per head, per tile: [g][scale block][8 slots e], so a lane reads the 8 scales of its slots at once.
// The slots of a word belong to different positions: a store rewrites the nibbles of its own rows only.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "nvfp4.hpp"

namespace xtg::hip {

// The byte of a code in a head-major K or V array, and which nibble of it (0: the low one).
struct Code4 {
  size_t byte;
  int high;
};

__host__ __device__ inline Code4 k4_code(int h, int slot, int dim, int slots_pad, int d) {
  const int chunk = d < 128 ? d : 128, lane_dims = chunk / 4, b = slot >> 4, i = slot & 15;
  const int g = (dim % chunk) / lane_dims, w = dim % lane_dims;
  return {size_t(h) * size_t(slots_pad) * size_t(d / 2) + size_t(b) * size_t(8 * d) + size_t(dim / chunk * 8 * chunk) +
              size_t((g * 16 + i) * (lane_dims / 2) + w / 2),
          w & 1};
}

__host__ __device__ inline size_t k4_scale(int h, int slot, int dim, int slots_pad, int d) {
  const int chunk = d < 128 ? d : 128, lane_dims = chunk / 4, b = slot >> 4, i = slot & 15;
  const int g = (dim % chunk) / lane_dims, w = dim % lane_dims;
  return size_t(h) * size_t(slots_pad) * size_t(d / 16) + size_t(b) * size_t(d) + size_t(dim / chunk * chunk) +
         size_t((g * 16 + i) * (lane_dims / 16) + w / 16);
}

__host__ __device__ inline Code4 v4_code(int h, int slot, int dim, int slots_pad, int d) {
  const int nd = d / 16, t = slot >> 5, kk = slot & 31, g = (kk & 15) >> 2, e = (kk >> 4) * 4 + (kk & 3);
  const int i = dim / nd, dd = dim % nd;
  return {size_t(h) * size_t(slots_pad) * size_t(d / 2) + size_t(t) * size_t(16 * d) + size_t((dd / 4) * 1024) +
              size_t((g * 16 + i) * 16 + (dd % 4) * 4 + e / 2),
          e & 1};
}

__host__ __device__ inline size_t v4_scale(int h, int slot, int dim, int slots_pad, int d) {
  const int t = slot >> 5, kk = slot & 31, g = (kk & 15) >> 2, e = (kk >> 4) * 4 + (kk & 3);
  return size_t(h) * size_t(slots_pad) * size_t(d / 16) + size_t(t) * size_t(2 * d) +
         size_t((g * (d / 16) + dim / 16) * 8 + e);
}

// A code's value without its scale, and an E4M3 scale's (0x7f: NaN, a row that is not finite).
__host__ __device__ inline float e2m1_value(int code) {
  const int m = code & 7;   // 0, 0.5, 1, 1.5, 2, 3, 4, 6
  const float a = m < 4 ? 0.5f * float(m) : m < 6 ? float(m - 2) : float(2 * m - 8);
  return code & 8 ? -a : a;
}

__host__ __device__ inline float e4m3_scale_value(uint8_t s) {
  if ((s & 0x7f) == 0x7f) return __builtin_nanf("");
  const int e = s >> 3, m = s & 7;   // scales are not negative
  return e == 0 ? float(m) * 0.001953125f : __builtin_ldexpf(1.f + float(m) / 8.f, e - 7);
}

// The E4M3 code of the scale of a block whose largest magnitude (over the global) is amax, finite: the nearest value
// to amax / 6, ties to even, at most 448, at least 2^-9 where amax > 0. The quotient is rounded to odd first (its last
// bit set wherever it is not exact), so that the second rounding is that of the exact quotient.
__device__ inline uint32_t block_scale_code(float amax) {
  if (amax >= 2688.f) return 0x7eu;
  const float y = amax / 6.f;
  const float r = fmaf(-y, 6.f, amax);
  uint32_t a = __float_as_uint(y);
  if (r != 0.f && !(a & 1u)) a = r > 0.f ? a | 1u : a - 1u;
  if (a < 0x3c800000u) {                       // below 2^-6: whole steps of 2^-9
    const float t = __uint_as_float(a) * 512.f, lo = floorf(t), frac = t - lo;
    uint32_t n = uint32_t(lo);
    n += frac > 0.5f || (frac == 0.5f && (n & 1u)) ? 1u : 0u;
    return n == 0u && amax > 0.f ? 1u : n;
  }
  const uint32_t u = a + 0x7ffffu + ((a >> 20) & 1u);
  const uint32_t code = (((u >> 23) - 120u) << 3) | ((u >> 20) & 7u);
  return code > 0x7eu ? 0x7eu : code;
}

// The E2M1 code of x in a block of scale s (its global included): the nearest of 0, 0.5, .., 6 times s, ties to the
// even code, from comparisons with the midpoints, which are exact in FP32.
__device__ inline uint32_t e2m1_code(float x, float s) {
  const float a = fabsf(x);
  uint32_t n = a > 0.25f * s;
  n += a >= 0.75f * s;
  n += a > 1.25f * s;
  n += a >= 1.75f * s;
  n += a > 2.5f * s;
  n += a >= 3.5f * s;
  n += a > 5.f * s;
  n = s > 0.f ? n : 0u;
  return n | (x < 0.f ? 8u : 0u);
}

}  // namespace xtg::hip
