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

// The quantisation of a block of 16 whose largest magnitude over the global (a power of two, ginv its inverse) is amax: the scale is the
// E4M3 value nearest to amax / 6, ties to even, at most 448, at least 2^-9 where amax > 0; a code is the E2M1 value
// nearest to x / scale, at most 6. Both quotients are rounded to FP32 first, which the second rounding does not see: a
// quotient by b 2^q (1 <= b < 2) that is not a midpoint m of the second grid is off it by an ulp of its numerator over
// b 2^q or more, which is over half an ulp of m, so it never rounds onto m. Numerators are held to 6 * 448 and 6 * scale
// first, exact products: a quotient that passes FP32 would be an infinity, whose correction is NaN.
struct BlockScale {
  uint32_t code;     // E4M3
  float s, inv;      // its value with the global, and the inverse (0 for a block of zeros)
};

// x / s for inv = 1 / s: the product is off by an ulp or two, one step makes it the nearest.
__device__ inline float quotient(float x, float s, float inv) {
  const float y = x * inv;
  return fmaf(fmaf(-y, s, x), inv, y);
}

// A value over its block's scale, held to what the codes hold.
__device__ inline float over_scale(float x, const BlockScale& s) {
  return quotient(__builtin_amdgcn_fmed3f(x, -6.f * s.s, 6.f * s.s), s.s, s.inv);
}

__device__ inline BlockScale block_scale(float amax, float global, float ginv) {
  BlockScale r;
  const float y = fmaxf(quotient(fminf(amax, 2688.f), 6.f, 1.f / 6.f), amax > 0.f ? 0.001953125f : 0.f);
  r.code = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false)) & 0xffu;
  const float s = __builtin_amdgcn_cvt_f32_fp8(int(r.code), 0);
  const float i = __builtin_amdgcn_rcpf(s);
  r.s = s * global;
  r.inv = s > 0.f ? fmaf(fmaf(-s, i, 1.f), i, i) * ginv : 0.f;
  return r;
}

}  // namespace xtg::hip
