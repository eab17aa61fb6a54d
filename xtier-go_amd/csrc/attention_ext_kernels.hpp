// Kernels of attention with capped, biased and masked scores over a cache of any dtype.
//
// out = sum_p w_p v_p / sum_p w_p with w_p = 2^(s_p - m) over the keys p that a row sees, in one pass over them: m is a
// running maximum of the scores (in base-2 units), and what has been summed is rescaled when it moves. Both products
// are matrix ops with the keys as rows, S^T = K Q^T and O^T = V^T P^T: a lane holds the scores of one q-col (a row of
// the call and one of the q heads of a KV head), and the weights that it computes from them are the B operand of the
// second product as they are. A row sees the positions lo <= p < hi, so a mask is one unsigned comparison.
//
// Operands have 16 bits: BF16 for BF16 and FP8 caches and the call's own keys, f16 for NVFP4 caches, whose values
// (E2M1 code times E4M3 scale) f16 holds exactly and whose weights then keep 11 bits; q, BF16, is exact in both (in f16
// times a power of two for each q-col, elements under 2^-25 of its largest to within 2^-33 of that). Weights beside BF16
// values keep 8 bits: one type for both operands, which f16's range rules out for V, and a second term of each weight would
// be half again as many matrix ops. An output is then off by up to 2^-8 of its weighted |v|, of the size of the rounding
// of a BF16 output. Scores, sums and accumulators are FP32.
//
//   ext_few_kernel: up to some hundred q-cols (kFewCols; a decode or verify step, a short turn). Each wave takes 32-slot
//     tiles of its own straight from the cache's operand layout into registers; work-groups split the tiles of a KV head,
//     and more of them take the call's own keys. One row is bound by the cache's bytes (32768 NVFP4 keys of 8 heads of 128
//     dims: 11.1 us for 38 MB, 3.4 TB/s), more rows by the vector ALUs (a tile is dequantised for every 32 q-cols).
//   ext_rows_kernel: more q-cols (a prompt chunk). Four waves of 32 q-cols share tiles through LDS: each is dequantised
//     once per work-group. The call's own keys are packed as BF16 tiles first (ext_pack_kernel). Bound by what a SIMD issues:
//     the matrix ops of its two waves (38 % of the time at 2.1 GHz) and their vector ALU work (48 %: exponentials, masks,
//     dequantisation) hardly overlap, while LDS is busy for 29 %. 512 rows over 16384 NVFP4 keys, 32 / 8 heads of 128 dims:
//     154 us, 0.9 PFLOP/s; 1500 capped rows over 2500 keys, 16 / 4 heads of 256 dims: 96 us, 0.50.
//   ext_merge_kernel: joins the records of a q-col in their order.
//
// Values that are not finite: a score that is masked is replaced, so a key's only reach the q-cols that see it. Not so a
// value's, times a weight of zero. NVFP4 caches hold such rows as NaN keys (kv4.hip) and their V scales are taken as zero.
// With the others a q-col whose sum of weights is finite and whose accumulator is not is computed again key by key, by
// whichever kernel writes it (slow_col). So is one without a sum that may see a key: scores of minus infinity alone are NaN.
#pragma once

#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attention_ext.hpp"
#include "common.hpp"
#include "kv4.hpp"

namespace xtg::hip {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Weights are 2^(s - m + 7), and m moves only when a score passes it by more than 8: weights stay below f16's 2^16,
// and those of 2^-21 of the largest still have all their bits.
constexpr float kUp = 7.f, kSlack = 8.f;

__device__ inline f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <int T>
struct OperandOf {
  using type = bf16x8;
};
template <>
struct OperandOf<kNvfp4> {
  using type = f16x8;
};

// 8 elements of a row as BF16 (FP32 rows are rounded).
__device__ inline bf16x8 row8(const void* p, size_t at, int bf16) {
  if (bf16) return *reinterpret_cast<const bf16x8*>(static_cast<const __bf16*>(p) + at);
  const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
  const float4 a = f[0], b = f[1];
  return bf16x8{(__bf16)a.x, (__bf16)a.y, (__bf16)a.z, (__bf16)a.w, (__bf16)b.x, (__bf16)b.y, (__bf16)b.z, (__bf16)b.w};
}

// N chunks of 8 elements of a row, chunk c at at(c); zeros where it is not live (then row 0 is read). The type is asked
// once: a branch a chunk would put each load behind the last one's.
template <int N, class A>
__device__ inline void row_chunks(const void* p, int bf16, bool live, A at, bf16x8 (&x)[N]) {
  if (bf16) {
#pragma unroll
    for (int c = 0; c < N; ++c) x[c] = *reinterpret_cast<const bf16x8*>(static_cast<const __bf16*>(p) + at(c));
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) x[c] = row8(p, at(c), 0);
  }
  if (!live) {
#pragma unroll
    for (int c = 0; c < N; ++c) x[c] = bf16x8{};
  }
}

// The q-col's N operand chunks. SCALED: times a power of two that brings the largest magnitude over the q-col's lanes (`join`)
// to 2^8 .. 2^9, for f16; for FP8 caches (BF16 operands) only where the wave has a magnitude of 2^65 or more, since codes'
// products are multiplied by their key's scale afterwards and could pass FP32 before it (scaling all of them cost 45 rows
// over 4000 keys 5 %). Else as they are. Returns the power of two that a product has to be multiplied by.
template <bool SCALED, int N, class X8, class J>
__device__ inline int to_operand(const bf16x8 (&x)[N], X8 (&q)[N], J join) {
  bool scaled = SCALED;
  if constexpr (SCALED && std::is_same_v<X8, bf16x8>) {
    uint32_t both = 0;   // the two highest bits of an exponent
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const uint4 w = __builtin_bit_cast(uint4, x[c]);
      both |= (w.x & w.x << 1) | (w.y & w.y << 1) | (w.z & w.z << 1) | (w.w & w.w << 1);
    }
    scaled = __ballot(both & 0x40004000u) != 0;
  }
  if (SCALED && scaled) {
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint((float)x[c][e]) & 0x7fffffffu);
    m = __float_as_uint(join(__uint_as_float(m & 0xff800000u)));   // powers of two, or infinity: ordered as floats
    constexpr int kLeast = std::is_same_v<X8, f16x8> ? -126 : 0;   // (2^-ex is finite; FP8: never up)
    const int ex = m == 0u || m >= 0x7f800000u ? 0 : max(int(m >> 23) - 127 - 8, kLeast);
    const float down = ldexpf(1.f, -ex);
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) q[c][e] = (float)x[c][e] * down;
    return ex;
  }
  if constexpr (std::is_same_v<X8, bf16x8>) {
#pragma unroll
    for (int c = 0; c < N; ++c) q[c] = x[c];
  }
  return 0;
}

// 8 E4M3 codes as BF16, exactly.
__device__ inline bf16x8 fp8_operand(uint32_t w0, uint32_t w1) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, false);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, false);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 E2M1 codes times four pairs of scales (V: pairs of keys).
__device__ inline f16x8 dequant8_pairs(uint32_t word, const f16x2 (&s)[4]) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 0) * s[0];
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 1) * s[1];
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 2) * s[2];
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, 1.0f, 3) * s[3];
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 E4M3 scales of V as pairs in f16 (exact), NaN as zero.
__device__ inline void v_scales(uint2 w, f16x2 (&s)[4]) {
  const f16x2 zero = {(_Float16)0.f, (_Float16)0.f};
  auto pair = [&](auto x) { return __builtin_elementwise_max(__builtin_bit_cast(f16x2, x), zero); };
  s[0] = pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.f, false));
  s[1] = pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.f, true));
  s[2] = pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.f, false));
  s[3] = pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.f, true));
}

// The positions that a row sees: lo <= p < lo + len.
struct Span {
  int lo;
  uint32_t len;
  int t;   // the row's own position
};
__device__ inline Span row_span(const ExtArgs& a, int row) {
  Span s;
  s.t = a.pos0 + row;
  s.lo = max(max(0, a.first ? a.first[row] : 0), a.window > 0 ? s.t - a.window + 1 : 0);
  const int hi = a.end ? a.end[row] : s.t + 1;
  s.len = hi > s.lo ? uint32_t(hi - s.lo) : 0u;
  return s;
}
// The same of the cached keys.
__device__ inline Span cached_span(const ExtArgs& a, Span s) {
  if (s.lo >= a.cached_end) s.len = 0;
  else s.len = min(s.len, uint32_t(a.cached_end - s.lo));
  return s;
}

// What turns a product q.k into a score in base-2 units.
struct Score {
  float f;             // times this (the scale, or with a cap what the exponential takes)
  float top, slope;    // cap * log2(e); the head's slope * log2(e)
};
// Score::f for operands whose product times global * 2^ex is q.k (a power of two too). Exponents are added as integers: those of
// a small cap, a global and a q-col pass FP32 together. (It stays finite and above zero: times an infinity one, times zero
// none.)
__device__ inline float score_factor(const ExtArgs& a, float global, int ex) {
  return fminf(fmaxf(ldexpf(a.factor * global, a.factor_exp + ex), FLT_MIN), FLT_MAX);
}
__device__ inline Score score_of(const ExtArgs& a, int head, float global, int ex) {
  Score s;
  s.f = score_factor(a, global, ex);
  s.top = fmaxf(a.softcap * kLog2e, FLT_MIN);
  s.slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
  return s;
}
// What a call does to its scores, a bit each; kernels are made for each of the four.
constexpr int kCap = 1, kBias = 2;
// cap * tanh(x / cap) = cap * (1 - 2 / (e^(2 x / cap) + 1)), minus the bias.
template <int MOD>
__device__ inline float changed(const Score& s, float qk, int dist) {
  float y = qk * s.f;
  if (MOD & kCap) y = fmaf(-2.f * s.top, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y) + 1.f), s.top);
  if (MOD & kBias) y = fmaf(-s.slope, fabsf(float(dist)), y);
  return y;
}

// A score in two steps: begun for every key (masked(): where it is not seen), and from the best of them for the maximum
// (best: the score is monotone in it) or inside the exponential, finish(x, minus) = score - minus in one operation.
template <int MOD>
__device__ inline float begin(const Score& s, float qk, int dist) {
  if (MOD == kCap) return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(qk * s.f) + 1.f);
  return MOD ? changed<MOD>(s, qk, dist) : qk;
}
template <int MOD>
__device__ inline float masked() { return MOD == kCap ? INFINITY : -INFINITY; }
template <int MOD>
__device__ inline float best(float a, float b) { return MOD == kCap ? fminf(a, b) : fmaxf(a, b); }
template <int MOD>
__device__ inline float finish(const Score& s, float x, float minus) {
  return MOD == kCap ? fmaf(-2.f * s.top, x, s.top - minus) : MOD ? x - minus : fmaf(x, s.f, -minus);
}
// From here on a plain score's product is rounded before the maximum, which is rounded, is subtracted: in one operation the
// best key's exponent is off by up to half an ulp of the maximum, 1/4 below and more than weights have range for from 2^28 on.
constexpr float kLarge = 8388608.f;   // 2^23

__device__ inline bool not_finite(float x) { return !(fabsf(x) <= FLT_MAX); }

// A kernel's ExtArgs, its first argument, read again: what of them only a rare path behind the loops needs does not stay in
// registers through these.
__device__ inline ExtArgs args_again() {
  auto from = (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(from));
  struct Words {
    uint32_t w[sizeof(ExtArgs) / 4];
  } words;
#pragma unroll
  for (size_t x = 0; x < sizeof(ExtArgs) / 4; ++x) words.w[x] = from[x];
  return __builtin_bit_cast(ExtArgs, words);
}

// A sum of no weights in a row that sees some positions: nothing is there, or all of its scores are minus infinity.
__device__ inline bool no_sum(float l, int row) { return l == 0.f && row_span(args_again(), row).len > 0; }

// ------------------------------------------------------------------------------------------- a q-col key by key

template <int D, int T>
__device__ inline float cached_value(const ExtArgs& a, bool v, int h, int slot, int dim) {
  const uint8_t* c = v ? a.cv : a.ck;
  const void* s = v ? a.vs : a.ks;
  const int pad = a.slots_pad;
  if constexpr (T == kBf16) {
    const uint16_t x = reinterpret_cast<const uint16_t*>(
        c)[v ? kv_v_index(h, slot, dim, pad, D) : kv_k_index(h, slot, dim, pad, D)];
    return __uint_as_float(uint32_t(x) << 16);
  } else if constexpr (T == kFp8) {
    const int code = c[v ? kv_v8_index(h, slot, dim, pad, D) : kv_k8_index(h, slot, dim, pad, D)];
    return __builtin_amdgcn_cvt_f32_fp8(code, 0) * static_cast<const float*>(s)[size_t(h) * size_t(pad) + size_t(slot)];
  } else {
    const Code4 at = v ? v4_code(h, slot, dim, pad, D) : k4_code(h, slot, dim, pad, D);
    const uint8_t sc = static_cast<const uint8_t*>(s)[v ? v4_scale(h, slot, dim, pad, D) : k4_scale(h, slot, dim, pad, D)];
    return e2m1_value(c[at.byte] >> (4 * at.high) & 15) * e4m3_scale_value(sc) * (v ? a.vglobal : a.kglobal);
  }
}

__device__ inline float row_value(const void* p, size_t at, int bf16) {
  return bf16 ? (float)static_cast<const __bf16*>(p)[at] : (float)(__bf16) static_cast<const float*>(p)[at];
}

// One q-col by a work-group of 256 threads: 256 keys at a time, a score each thread, then a dim each thread; values of
// keys that the row does not see are not read. Scores of minus infinity alone leave no sum, and NaN; keys that the row does
// not see, or that are not there, zeros. lds: 272 + D floats.
template <int D, int T>
__device__ inline void slow_col(const ExtArgs& a, int h, int kv_heads, int row, int head, float* lds) {
  float *q = lds, *w = lds + D, *red = lds + D + 256;
  const int tid = int(threadIdx.x);
  const Span all = row_span(a, row), cached = cached_span(a, all);
  const Score sc = score_of(a, head, 1.f, 0);
  const size_t at = (size_t(row) * size_t(a.heads) + size_t(head)) * D + size_t(tid);
  __syncthreads();
  if (tid < D) q[tid] = row_value(a.q, at, a.bf16);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc = 0.f;   // (m: -inf until a key is seen, -FLT_MAX at least from then on)
  for (int k0 = 0; k0 < a.slots_pad + a.own; k0 += 256) {
    // (a linear cache's slots are positions; the work-group's threads have one row)
    if (!a.ring && k0 + 256 <= a.slots_pad && (k0 + 256 <= all.lo || k0 - all.lo >= int(cached.len))) continue;
    const int key = k0 + tid, j = key - a.slots_pad;   // own key j
    int pos = -1;
    if (j < 0)
      pos = a.slot_pos[key];
    else if (j < a.own)
      pos = a.pos0 + j;
    const bool seen = uint32_t(pos - all.lo) < (j < 0 ? cached.len : all.len);   // (the spans begin alike)
    float s = -INFINITY;
    if (seen) {
      s = 0.f;
      for (int x = 0; x < D; ++x)
        s += q[x] * (j < 0 ? cached_value<D, T>(a, false, h, key, x)
                           : row_value(a.k, (size_t(j) * size_t(kv_heads) + size_t(h)) * D + size_t(x), a.bf16));
      if (a.scale < 0.f) s = -s;
      s = a.softcap > 0.f ? changed<kCap | kBias>(sc, s, all.t - pos) : changed<kBias>(sc, s, all.t - pos);
    }
    const float top = block_max<256>(seen ? fmaxf(s, -FLT_MAX) : -INFINITY, red), m_new = fmaxf(m, top);
    if (top == -INFINITY) continue;
    const float p = __builtin_amdgcn_exp2f(s - m_new), corr = __builtin_amdgcn_exp2f(m - m_new);
    w[tid] = seen ? p : -1.f;   // -1: not seen
    l = l * corr + block_sum<256>(p, red);
    m = m_new;
    acc *= corr;
    __syncthreads();
    if (tid < D)
      for (int x = 0; x < 256; ++x) {
        if (w[x] < 0.f) continue;
        const int kx = k0 + x, jx = kx - a.slots_pad;
        acc += w[x] * (jx < 0 ? cached_value<D, T>(a, true, h, kx, tid)
                              : row_value(a.v, (size_t(jx) * size_t(kv_heads) + size_t(h)) * D + size_t(tid), a.bf16));
      }
    __syncthreads();
  }
  if (tid < D) {
    const float y = l == 0.f ? m == -INFINITY ? 0.f : NAN : acc / l;
    if (a.bf16)
      static_cast<__bf16*>(a.out)[at] = (__bf16)y;
    else
      static_cast<float*>(a.out)[at] = y;
  }
}

// The largest and smallest of a wave's values (every lane gets them).
__device__ inline void wave_extremes(int& top, int& least) {
  auto step = [&](int a, int b) { top = max(top, a), least = min(least, b); };
  step(__builtin_amdgcn_update_dpp(0, top, kDppXor1, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, least, kDppXor1, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, top, kDppXor2, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, least, kDppXor2, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, top, kDppHalfMirror, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, least, kDppHalfMirror, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, top, kDppMirror, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, least, kDppMirror, 0xF, 0xF, false));
  auto a = __builtin_amdgcn_permlane16_swap(uint32_t(top), uint32_t(top), false, false);
  auto b = __builtin_amdgcn_permlane16_swap(uint32_t(least), uint32_t(least), false, false);
  top = max(int(a[0]), int(a[1])), least = min(int(b[0]), int(b[1]));
  a = __builtin_amdgcn_permlane32_swap(uint32_t(top), uint32_t(top), false, false);
  b = __builtin_amdgcn_permlane32_swap(uint32_t(least), uint32_t(least), false, false);
  top = max(int(a[0]), int(a[1])), least = min(int(b[0]), int(b[1]));
}

// ------------------------------------------------------------------------------------------------- few q-cols

// A wave's tile of 32 slots: the keys of a lane's scores are slots 4 g + e and 16 + 4 g + e - 4. k(b, st), v(dd): the
// operands; dim(dd, r): the dim of row r of product dd.
template <int D, int T>
struct Tile;

template <int D>
struct Tile<D, kBf16> {
  uint4 kw[2][D / 32], vw[D / 16];
  static constexpr bool kScaled = false;
  __device__ static int q_dim(int st, int g) { return 32 * st + 8 * g; }
  __device__ static int dim(int dd, int r) { return 16 * dd + r; }
  __device__ void load_k(const ExtArgs& a, int h, int t, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.ck) + (size_t(h) * size_t(a.slots_pad) + size_t(32 * t)) * (D / 8) + lane;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) kw[b][c] = p[(b * (D / 32) + c) * 64];
  }
  __device__ void load_v(const ExtArgs& a, int h, int t, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.cv) + (size_t(h) * size_t(a.slots_pad) + size_t(32 * t)) * (D / 8) + lane;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd) vw[dd] = p[dd * 64];
  }
  __device__ bf16x8 k(int b, int st) const { return __builtin_bit_cast(bf16x8, kw[b][st]); }
  __device__ void begin_v() {}
  __device__ bf16x8 v(int dd) const { return __builtin_bit_cast(bf16x8, vw[dd]); }
};

template <int D>
struct Tile<D, kFp8> {
  uint4 kw[2][D / 64], vw[D / 32];
  float ks[8], vs[8];   // a key whose V scale is not finite is NaN itself, and the scale zero
  static constexpr bool kScaled = true;
  __device__ static int q_dim(int st, int g) { return 32 * st + 8 * g; }
  __device__ static int dim(int dd, int r) { return 16 * dd + r; }
  __device__ void load_k(const ExtArgs& a, int h, int t, int lane) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(32 * t);
    const uint4* p = reinterpret_cast<const uint4*>(a.ck) + at * (D / 16) + lane;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) kw[b][c] = p[(b * (D / 64) + c) * 64];
    load8(ks, static_cast<const float*>(a.ks) + at + 4 * (lane >> 4));
    load8(vs, static_cast<const float*>(a.vs) + at + 4 * (lane >> 4));
  }
  __device__ static void load8(float (&x)[8], const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 16);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  __device__ void load_v(const ExtArgs& a, int h, int t, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.cv) + (size_t(h) * size_t(a.slots_pad) + size_t(32 * t)) * (D / 16) + lane;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) vw[c] = p[c * 64];
  }
  __device__ bf16x8 k(int b, int st) const {
    const uint4 w = kw[b][st >> 1];
    return st & 1 ? fp8_operand(w.z, w.w) : fp8_operand(w.x, w.y);
  }
  __device__ void begin_v() {}
  __device__ bf16x8 v(int dd) const {
    const uint4 w = vw[dd >> 1];
    return dd & 1 ? fp8_operand(w.z, w.w) : fp8_operand(w.x, w.y);
  }
};

template <int D>
struct Tile<D, kNvfp4> {
  static constexpr int CH = D < 128 ? D : 128, LD = CH / 4, SPC = CH / 32;   // a lane's dims of a chunk, steps a chunk
  uint32_t kw[2][D / 32], vw[D / 16], ks[2][D / CH];
  uint2 vs;
  f16x2 vp[4];
  static constexpr bool kScaled = false;
  __device__ static int q_dim(int st, int g) { return st / SPC * CH + g * LD + 8 * (st % SPC); }
  __device__ static int dim(int dd, int r) { return r * (D / 16) + dd; }
  __device__ void load_k(const ExtArgs& a, int h, int t, int lane) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(32 * t);
    const uint8_t* p = a.ck + at * (D / 2);
    const uint8_t* s = static_cast<const uint8_t*>(a.ks) + at * (D / 16);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / CH; ++c) {
        const int i = b * (D / CH) + c;
        if constexpr (D >= 128) {
          const uint4 w = reinterpret_cast<const uint4*>(p)[i * 64 + lane];
          kw[b][4 * c] = w.x, kw[b][4 * c + 1] = w.y, kw[b][4 * c + 2] = w.z, kw[b][4 * c + 3] = w.w;
          ks[b][c] = reinterpret_cast<const uint16_t*>(s)[i * 64 + lane];
        } else {
          const uint2 w = reinterpret_cast<const uint2*>(p)[i * 64 + lane];
          kw[b][0] = w.x, kw[b][1] = w.y;
          ks[b][0] = s[i * 64 + lane];
        }
      }
  }
  __device__ void load_v(const ExtArgs& a, int h, int t, int lane) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(32 * t);
    const uint4* p = reinterpret_cast<const uint4*>(a.cv + at * (D / 2)) + lane;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = p[c * 64];
      vw[4 * c] = w.x, vw[4 * c + 1] = w.y, vw[4 * c + 2] = w.z, vw[4 * c + 3] = w.w;
    }
    const int block = (lane & 15) * (D / 16) / 16;
    vs = reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.vs) + at * (D / 16))[(lane >> 4) * (D / 16) + block];
  }
  __device__ f16x8 k(int b, int st) const { return dequant8(kw[b][st], scale_pair(ks[b][st / SPC], st % SPC / 2)); }
  __device__ void begin_v() { v_scales(vs, vp); }
  __device__ f16x8 v(int dd) const { return dequant8_pairs(vw[dd], vp); }
};

// 32 of the call's own keys, as its rows are, values in the order of T's tiles; keys past the last are zeros (and not
// seen).
template <int D, int T>
struct OwnTile {
  bf16x8 kw[2][D / 32], vw[D / 16];
  static constexpr bool kScaled = false;
  __device__ static int q_dim(int st, int g) { return 32 * st + 8 * g; }
  const ExtArgs& a;
  const int h, kv_heads, t, lane;
  __device__ OwnTile(const ExtArgs& a, int h, int kv_heads, int t, int lane) : a(a), h(h), kv_heads(kv_heads), t(t), lane(lane) {
    const int g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int j = 32 * t + 16 * b + i;
      const size_t at = (size_t(j < a.own ? j : 0) * size_t(kv_heads) + size_t(h)) * D + size_t(8 * g);
      row_chunks(a.k, a.bf16, j < a.own, [&](int c) { return at + size_t(32 * c); }, kw[b]);
    }
  }
  __device__ bf16x8 k(int b, int st) const { return kw[b][st]; }
  __device__ void begin_v() {
    const int g = lane >> 4, i = lane & 15;
    auto take = [&](auto* p) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = 32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e);
        const size_t at = (size_t(j < a.own ? j : 0) * size_t(kv_heads) + size_t(h)) * D;
#pragma unroll
        for (int dd = 0; dd < D / 16; ++dd) vw[dd][e] = j < a.own ? (__bf16)p[at + size_t(Tile<D, T>::dim(dd, i))] : (__bf16)0.f;
      }
    };
    if (a.bf16)
      take(static_cast<const __bf16*>(a.v));
    else
      take(static_cast<const float*>(a.v));
  }
  __device__ bf16x8 v(int dd) const { return vw[dd]; }
};

// The state of a lane's q-col in each block of 16: the maximum (the same in the col's 4 lanes), the lane's own part of the
// sum, and the accumulator: rows 4 g + r of product dd.
template <int D, int QB>
struct FewState {
  float m[QB], l[QB];
  f32x4 acc[QB][D / 16];
};

// One tile. next_k loads the next tile's keys once this one's are used, next_v its values: each load has about half a
// tile's work to land behind.
template <int D, int QB, int MOD, class TILE, class X8, class NK, class NV>
__device__ inline void few_tile(const ExtArgs& a, TILE& T, const X8 (&q)[QB][D / 32], const Span (&span)[QB],
                                const Score (&sc)[QB], FewState<D, QB>& st, int4 p0, int4 p1, NK&& next_k, NV&& next_v) {
  const int pos[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
  f32x4 s[QB][2];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) s[qb][0] = s[qb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const X8 k = T.k(b, c);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[qb][b] = mfma16(k, q[qb][c], s[qb][b]);
    }
  float ks[8], vs[8];
  if constexpr (TILE::kScaled) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool bad = not_finite(T.vs[e]);
      ks[e] = bad ? NAN : T.ks[e];
      vs[e] = bad ? 0.f : T.vs[e];
    }
  }
  next_k();
  X8 w[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    float y[8];
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = s[qb][e >> 2][e & 3];
      if constexpr (TILE::kScaled) x *= ks[e];
      x = changed<MOD>(sc[qb], x, span[qb].t - pos[e]);
      y[e] = uint32_t(pos[e] - span[qb].lo) < span[qb].len ? x : -INFINITY;
      mx = fmaxf(mx, y[e]);
    }
    mx = xor32_max(xor16_max(mx));
    if (__ballot(mx > st.m[qb] + kSlack)) {   // (a maximum of -inf: any score)
      const float m = mx > st.m[qb] + kSlack ? mx : st.m[qb];
      const float corr = __builtin_amdgcn_exp2f(st.m[qb] - (m == -INFINITY ? 0.f : m));
      st.m[qb] = m;
      st.l[qb] *= corr;
#pragma unroll
      for (int dd = 0; dd < D / 16; ++dd) st.acc[qb][dd] *= corr;
    }
    const float ref = (st.m[qb] == -INFINITY ? 0.f : st.m[qb]) - kUp;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float p = __builtin_amdgcn_exp2f(y[e] - ref);
      st.l[qb] += p;
      if constexpr (TILE::kScaled) p *= vs[e];
      w[qb][e] = p;
    }
  }
  T.begin_v();
#pragma unroll
  for (int dd = 0; dd < D / 16; ++dd) {
    const X8 v = T.v(dd);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) st.acc[qb][dd] = mfma16(v, w[qb], st.acc[qb][dd]);
  }
  next_v();
}

// The row of a q-col.
__device__ inline int few_row(const ExtArgs& a, int col) { return int(uint32_t(col) * a.group_inv >> 16); }

// The q-cols' rows, spans and score factors of a work-group; then their operands of T's type. The rows' loads go out
// before the first tile's, and are waited for behind them.
template <int D, int QB, class TILE>
struct FewQueries {
  bf16x8 x[QB][D / 32];
  Span span[QB];
  Score sc[QB];
  __device__ void load(const ExtArgs& a, int h, int col0, int lane) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int col = col0 + qb * 16 + (lane & 15), row = few_row(a, col), head = h * a.group + col - row * a.group;
      const bool live = row < a.n_q;
      const size_t at = live ? (size_t(row) * size_t(a.heads) + size_t(head)) * D : 0;
      row_chunks(a.q, a.bf16, live, [&](int c) { return at + size_t(TILE::q_dim(c, lane >> 4)); }, x[qb]);
      span[qb] = live ? row_span(a, row) : Span{0, 0u, 0};
      sc[qb] = score_of(a, live ? head : 0, 1.f, 0);
    }
  }
  template <bool SCALED, class X8>
  __device__ void operand(const ExtArgs& a, float global, X8 (&q)[QB][D / 32]) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (a.scale < 0.f) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) x[qb][c] = -x[qb][c];
      }
      sc[qb].f = score_factor(a, global, to_operand<SCALED>(x[qb], q[qb], [](float v) { return xor32_max(xor16_max(v)); }));
    }
  }
};

template <int D, int QB>
constexpr size_t few_lds() { return size_t(kExtWaves) * QB * (2 * 16 + D * 16) * sizeof(float); }

template <int D, int QB, int T, int MOD>
__global__ void __launch_bounds__(kExtWaves * 64, QB * D > 256 ? 1 : 2) ext_few_kernel(ExtArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  float* lds = reinterpret_cast<float*>(smem);
  __shared__ uint32_t again;   // q-cols to be computed again
  constexpr int ND = D / 16;
  const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6, g = lane >> 4, i = lane & 15;
  const int h = int(blockIdx.x), kv_heads = int(gridDim.x), split = int(gridDim.y) - 1 - int(blockIdx.y);
  const int col0 = int(blockIdx.z) * QB * 16;   // the work-group's first q-col
  const bool own = split >= a.splits;   // the work-groups past the cache's, queued first: the call's own keys
  FewState<D, QB> st;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    st.m[qb] = -INFINITY, st.l[qb] = 0.f;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (own) {
    bf16x8 q[QB][D / 32];
    FewQueries<D, QB, OwnTile<D, T>> rows;
    rows.load(a, h, col0, lane);
    rows.template operand<false>(a, 1.f, q);
    const int t = (split - a.splits) * kExtWaves + wave, p = a.pos0 + 32 * t;   // (p + 32 can pass 2^31)
    bool any = false;   // a q-col that sees one of the tile's keys
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      any |= rows.span[qb].len > 0 && rows.span[qb].lo - 32 < p && int(rows.span[qb].len) > p - rows.span[qb].lo;
    if (32 * t < a.own && __ballot(any)) {
      OwnTile<D, T> tile(a, h, kv_heads, t, lane);
      auto at = [&](int e) { return 32 * t + 4 * g + e < a.own ? p + 4 * g + e : -1; };
      few_tile<D, QB, MOD>(a, tile, q, rows.span, rows.sc, st, make_int4(at(0), at(1), at(2), at(3)),
                           make_int4(at(16), at(17), at(18), at(19)), [] {}, [] {});
    }
  } else {
    using X8 = typename OperandOf<T>::type;
    const int t_begin = a.tile_lo + int((long long)a.tiles * split / a.splits);
    const int t_end = a.tile_lo + int((long long)a.tiles * (split + 1) / a.splits);
    X8 q[QB][D / 32];
    FewQueries<D, QB, Tile<D, T>> rows;
    rows.load(a, h, col0, lane);
    Tile<D, T> tile;
    int t = t_begin + wave;
    if (!a.ring && (a.first || a.window > 0)) {   // tiles before the first position that a q-col sees
      int lo = INT_MAX, none = 0;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) lo = rows.span[qb].len ? min(lo, rows.span[qb].lo) : lo;
      wave_extremes(none, lo);
      const int skip = (min(__builtin_amdgcn_readfirstlane(lo) / 32, t_end) - t + kExtWaves - 1) / kExtWaves;
      if (skip > 0) t += skip * kExtWaves;
    }
    const int4* sp = reinterpret_cast<const int4*>(a.slot_pos) + g;
    if (t < t_end) {
      tile.load_k(a, h, t, lane);
      int4 p0 = sp[t * 8], p1 = sp[t * 8 + 4];
      tile.load_v(a, h, t, lane);
      rows.template operand<T != kBf16>(a, T == kNvfp4 ? a.kglobal : 1.f, q);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) rows.span[qb] = cached_span(a, rows.span[qb]);
      for (; t < t_end; t += kExtWaves) {
        const int n = min(t + kExtWaves, t_end - 1);   // past the end: loaded again, and not used
        const int4 c0 = p0, c1 = p1;
        few_tile<D, QB, MOD>(
            a, tile, q, rows.span, rows.sc, st, c0, c1,
            [&] {
              tile.load_k(a, h, n, lane);
              p0 = sp[n * 8], p1 = sp[n * 8 + 4];
            },
            [&] { tile.load_v(a, h, n, lane); });
      }
    }
    if (T == kNvfp4 && a.vglobal != 1.f) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] *= a.vglobal;
    }
  }

  if (threadIdx.x == 0) again = 0;

  // the waves' states joined: the maxima and sums, then the accumulators, each wave a part of the sums
  float* ml = lds;                                   // [wave][QB * 16][2]
  float* part = lds + kExtWaves * QB * 2 * 16;       // [wave][QB][products][64 lanes][4]
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float l = xor32_sum(xor16_sum(st.l[qb]));
    if (g == 0) {
      ml[(wave * QB * 16 + qb * 16 + i) * 2] = st.m[qb];
      ml[(wave * QB * 16 + qb * 16 + i) * 2 + 1] = l;
    }
  }
  __syncthreads();
  float m_all[QB], l_all[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kExtWaves; ++w) m = fmaxf(m, ml[(w * QB * 16 + qb * 16 + i) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kExtWaves; ++w)
      l += ml[(w * QB * 16 + qb * 16 + i) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * QB * 16 + qb * 16 + i) * 2] - ref);
    const float corr = __builtin_amdgcn_exp2f(st.m[qb] - ref);
    m_all[qb] = m;
    l_all[qb] = l;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] *= corr;
  }
  const size_t rec = ((size_t(blockIdx.z) * size_t(kv_heads) + size_t(h)) * size_t(a.records) + size_t(split)) * size_t(a.cols);
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int dd = 0; dd < ND; ++dd)
      *reinterpret_cast<f32x4*>(part + (((wave * QB + qb) * ND + dd) * 64 + lane) * 4) = st.acc[qb][dd];
  __syncthreads();
  {
#pragma unroll
    for (int x = 0; x < QB * ND; x += kExtWaves) {
      const int qd = x + wave, qb = qd / ND, dd = qd % ND;
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kExtWaves; ++w) y += *reinterpret_cast<const f32x4*>(part + ((w * QB * ND + qd) * 64 + lane) * 4);
      const int mine = qb * 16 + i, col = col0 + mine, row = few_row(a, col);
      if (row >= a.n_q) continue;
      float l = l_all[0];
      if constexpr (QB == 2) l = qb ? l_all[1] : l;
      if (a.records == 1) {
        bool bad = no_sum(l, row);
#pragma unroll
        for (int r = 0; r < 4; ++r) bad |= !not_finite(l) && not_finite(y[r]);
        if (bad) atomicOr(&again, 1u << mine);
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int dim = Tile<D, T>::dim(dd, 4 * g + r);
          const size_t at = (size_t(row) * size_t(a.heads) + size_t(h * a.group + col - row * a.group)) * D + size_t(dim);
          if (a.bf16)
            static_cast<__bf16*>(a.out)[at] = (__bf16)(y[r] * inv);
          else
            static_cast<float*>(a.out)[at] = y[r] * inv;
        }
      } else {
        *reinterpret_cast<f32x4*>(a.acc + (rec + size_t(mine)) * D + size_t(16 * dd + 4 * g)) = y;
      }
    }
  }
  if (a.records == 1) {
    __syncthreads();
    for (uint32_t bits = again; bits; bits &= bits - 1) {
      const int col = col0 + __builtin_ctz(bits), row = few_row(a, col);
      slow_col<D, T>(args_again(), h, kv_heads, row, h * a.group + col - row * a.group, lds);
    }
    return;
  }
  if (wave == 0 && g < QB) {
    const int col = g * 16 + i;
    float m = m_all[0], l = l_all[0];
    if constexpr (QB == 2) m = g ? m_all[1] : m, l = g ? l_all[1] : l;
    if (col < a.cols) {
      a.ml[(rec + size_t(col)) * 2] = m;
      a.ml[(rec + size_t(col)) * 2 + 1] = l;
    }
  }
}

// -------------------------------------------------------------------------------------------------- own keys

// The call's own keys and values as tiles of 32 in the order of a BF16 cache's (attention.hip), V's dims in the order of
// T's tiles; zeros past the last. One thread for a K entry (8 dims of a key) or 8 V entries (8 keys of 8 dims).
template <int D, int T>
__global__ void __launch_bounds__(256) ext_pack_kernel(const void* __restrict__ k, const void* __restrict__ v, int bf16,
                                                       int n, int kv_heads, int tiles, uint4* __restrict__ pk,
                                                       uint4* __restrict__ pv) {
  constexpr int KE = 32 * D / 8, VE = 4 * D / 8;   // threads of a tile's K and V
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long tile = at / (KE + VE);
  if (tile >= (long long)tiles * kv_heads) return;
  const int x = int(at % (KE + VE)), t = int(tile / kv_heads), h = int(tile % kv_heads);
  const size_t base = (size_t(h) * size_t(tiles) + size_t(t)) * (32 * D / 8);
  if (x < KE) {
    const int key = x / (D / 8), c8 = x % (D / 8), j = 32 * t + key;
    const bf16x8 y = j < n ? row8(k, (size_t(j) * size_t(kv_heads) + size_t(h)) * D + size_t(8 * c8), bf16) : bf16x8{};
    pk[base + size_t(((key >> 4) * (D / 32) + (c8 >> 2)) * 64 + (c8 & 3) * 16 + (key & 15))] = __builtin_bit_cast(uint4, y);
    return;
  }
  const int g = (x - KE) / (D / 8), c8 = (x - KE) % (D / 8);
  bf16x8 y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int j = 32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e);
    y[e] = j < n ? row8(v, (size_t(j) * size_t(kv_heads) + size_t(h)) * D + size_t(8 * c8), bf16) : bf16x8{};
  }
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const int dim = 8 * c8 + d, dd = T == kNvfp4 ? dim % (D / 16) : dim / 16, i = T == kNvfp4 ? dim / (D / 16) : dim % 16;
    const bf16x8 z = {y[0][d], y[1][d], y[2][d], y[3][d], y[4][d], y[5][d], y[6][d], y[7][d]};
    pv[base + size_t(dd * 64 + g * 16 + i)] = __builtin_bit_cast(uint4, z);
  }
}

// --------------------------------------------------------------------------------------------------- many q-cols

// A tile of TK keys in LDS: K as [32-key block][16-dim step][64 lanes] entries of 8 dims, V as [32-row block][key step]
// [64 lanes] entries of 8 keys: A operands of v_mfma_f32_32x32x16. Lane (half, i) of a K entry has key i and dims
// 8 half .. +8 of the step, of a V entry row i and keys 8 a + 4 half + e, 16 + 8 a + 4 half + e (e = 0 .. 3) of step
// a = 0, 1 of a 32-key block: what the lane's scores are of. A cache's entries are these too, in another order.
// Two buffers of each, with the tiles' positions, FP8 scales and first and last position.
template <int D>
struct Rows {
  static constexpr int TK = D == 256 ? 32 : 64;
  static constexpr int KB = TK / 32, NS = D / 16, NB = D / 32, KS = TK / 16;
  static constexpr int kEntries = TK * D / 8;           // of K, and of V
  static constexpr int PER = kEntries / 256;            // entries a thread stages
  static constexpr int kInfo = 3 * TK + 4;              // ints of a tile's positions, scales and extremes
  static constexpr size_t kLds = size_t(kEntries) * 64 + size_t(kInfo) * 8 + 2048 + (D == 256 ? 2 * 4096 : 0);
  // (and room to turn the output; for heads of 256 dims, for two chunks of q)
};

// What a thread stages of a tile: loads in flight (raw), then entries written to LDS. A cache of an odd number of 32-slot
// tiles ends in the middle of a 64-key tile (`half`): its other half is zeros.
template <int D, int T>
struct Stage;

// BF16: entries as they are. Also the packed own keys.
template <int D>
struct Stage<D, kBf16> {
  using R = Rows<D>;
  uint4 k[R::PER], v[R::PER];
  __device__ static void load(uint4 (&x)[R::PER], const uint4* c, int h, int pad, int tile, bool half) {
    const size_t at = (size_t(h) * size_t(pad) + size_t(tile) * R::TK) * (D / 8) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < R::PER; ++u) x[u] = half && 2 * u >= R::PER ? make_uint4(0, 0, 0, 0) : c[at + u * 256];
  }
  __device__ void load_k(const uint4* ck, int h, int pad, int tile, bool half) { load(k, ck, h, pad, tile, half); }
  __device__ void load_v(const uint4* cv, int h, int pad, int tile, bool half) { load(v, cv, h, pad, tile, half); }
  // The tile straight into its place in LDS: 64 entries a wave's load, a lane's the one that comes to its part of them.
  __device__ static void direct(const uint4* c, int h, int pad, int tile, uint4* to, bool v) {
    const uint4* from = c + (size_t(h) * size_t(pad) + size_t(tile) * R::TK) * (D / 8);
    const int lane = int(threadIdx.x) & 63, half = lane >> 5, i = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
#pragma unroll
    for (int u = 0; u < R::PER; ++u) {
      const int row = u * 4 + wave;   // of 64 entries
      int x;
      if (v) {
        const int dd = row / R::KS * 2 + (i >> 4), ks = row % R::KS;
        x = (ks >> 1) * 4 * D + dd * 64 + ((ks & 1) * 2 + half) * 16 + (i & 15);
      } else {
        const int b = row / R::NS * 2 + (i >> 4), st = row % R::NS;
        x = b * 2 * D + (st >> 1) * 64 + ((st & 1) * 2 + half) * 16 + (i & 15);
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + x),
                                       (__attribute__((address_space(3))) void*)(to + row * 64), 16, 0, 0);
    }
  }
  // entry x of a BF16 tile of TK keys to its place
  __device__ static int k_place(int x) {
    const int b = x / (2 * D), c = x / 64 % (D / 32), g = x >> 4 & 3, i = x & 15;
    return ((b >> 1) * R::NS + 2 * c + (g >> 1)) * 64 + (g & 1) * 32 + (b & 1) * 16 + i;
  }
  __device__ static int v_place(int x) {
    const int t = x / (4 * D), dd = x / 64 % (D / 16), g = x >> 4 & 3, i = x & 15;
    return ((dd >> 1) * R::KS + 2 * t + (g >> 1)) * 64 + (g & 1) * 32 + (dd & 1) * 16 + i;
  }
  __device__ void store_k(uint4* lk) const {
#pragma unroll
    for (int u = 0; u < R::PER; ++u) lk[k_place(int(threadIdx.x) + u * 256)] = k[u];
  }
  __device__ void store_v(uint4* lv) const {
#pragma unroll
    for (int u = 0; u < R::PER; ++u) lv[v_place(int(threadIdx.x) + u * 256)] = v[u];
  }
};

// FP8: a 16-byte load is two entries' codes.
template <int D>
struct Stage<D, kFp8> {
  using R = Rows<D>;
  using B = Stage<D, kBf16>;
  uint4 k[R::PER / 2], v[R::PER / 2];
  __device__ static void load(uint4 (&x)[R::PER / 2], const uint4* c, int h, int pad, int tile, bool half) {
    const size_t at = (size_t(h) * size_t(pad) + size_t(tile) * R::TK) * (D / 16) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < R::PER / 2; ++u) {
      const bool past = half && int(threadIdx.x) + u * 256 >= R::kEntries / 4;
      x[u] = past ? make_uint4(0, 0, 0, 0) : c[at + u * 256];
    }
  }
  __device__ void load_k(const uint4* ck, int h, int pad, int tile, bool half) { load(k, ck, h, pad, tile, half); }
  __device__ void load_v(const uint4* cv, int h, int pad, int tile, bool half) { load(v, cv, h, pad, tile, half); }
  __device__ static int first(int u) {   // of BF16's entries
    const int x = int(threadIdx.x) + u * 256;
    return (x >> 6) * 128 + (x & 63);
  }
  __device__ void store_k(uint4* lk) const {
#pragma unroll
    for (int u = 0; u < R::PER / 2; ++u) {
      lk[B::k_place(first(u))] = __builtin_bit_cast(uint4, fp8_operand(k[u].x, k[u].y));
      lk[B::k_place(first(u) + 64)] = __builtin_bit_cast(uint4, fp8_operand(k[u].z, k[u].w));
    }
  }
  __device__ void store_v(uint4* lv) const {
#pragma unroll
    for (int u = 0; u < R::PER / 2; ++u) {
      lv[B::v_place(first(u))] = __builtin_bit_cast(uint4, fp8_operand(v[u].x, v[u].y));
      lv[B::v_place(first(u) + 64)] = __builtin_bit_cast(uint4, fp8_operand(v[u].z, v[u].w));
    }
  }
};

// NVFP4: a thread's codes are PER entries of K, which share a key, and PER of V, which share their keys' scales.
template <int D>
struct Stage<D, kNvfp4> {
  using R = Rows<D>;
  uint32_t k[R::PER], v[R::PER], ks;
  uint2 vs;
  __device__ void load_k(const ExtArgs& a, int h, int tile, bool half) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(tile) * R::TK;
    const int tid = int(threadIdx.x);
#pragma unroll
    for (int u = 0; u < R::PER; ++u) k[u] = 0;
    ks = 0;
    if (half && tid >= 128) return;
    take(k, a.ck + at * (D / 2), tid);
    const uint8_t* s = static_cast<const uint8_t*>(a.ks) + at * (D / 16);
    ks = D == 64 ? s[tid] : reinterpret_cast<const uint16_t*>(s)[tid];
  }
  // V: a wave has half a 32-slot tile's words (256 dims: a quarter)
  __device__ void load_v(const ExtArgs& a, int h, int tile, bool half) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(tile) * R::TK;
    const int tid = int(threadIdx.x), lane = tid & 63, part = tid >> 6, t = D == 256 ? 0 : part >> 1;
#pragma unroll
    for (int u = 0; u < R::PER; ++u) v[u] = 0;
    vs = make_uint2(0, 0);
    if (half && tid >= 128) return;
    take_v(a.cv + at * (D / 2), part, lane);
    const uint2* sv = reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.vs) + at * (D / 16));
    vs = sv[t * (D / 4) + (lane >> 4) * (D / 16) + (lane & 15) * (D / 16) / 16];
  }
  __device__ void take(uint32_t (&w)[R::PER], const uint8_t* p, int tid) {
    if constexpr (R::PER == 4) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[tid];
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
      const uint2 x = reinterpret_cast<const uint2*>(p)[tid];
      w[0] = x.x, w[1] = x.y;
    }
  }
  // words of products first_dd(part) .. of a lane
  __device__ void take_v(const uint8_t* p, int part, int lane) {
    if constexpr (R::PER == 4) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[part * 64 + lane];   // [tile][4 products][lane]
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {   // 64 dims: one 16-byte group a tile, half of it a wave
      const uint2 x = reinterpret_cast<const uint2*>(p)[((part >> 1) * 64 + lane) * 2 + (part & 1)];
      v[0] = x.x, v[1] = x.y;
    }
  }
  __device__ void store_k(uint4* lk) const {
    const int tid = int(threadIdx.x), lane = tid & 63, part = tid >> 6, g = lane >> 4, i = lane & 15;
    // D = 64, 128: 16-slot block `part`; 256: block part / 2, chunk part % 2
    const int b = D == 256 ? part >> 1 : part, chunk = D == 256 ? part & 1 : 0;
#pragma unroll
    for (int c = 0; c < R::PER; ++c) {
      const int dim8 = chunk * 16 + g * R::PER + c;   // dims 8 dim8 .. +8
      lk[((b >> 1) * R::NS + (dim8 >> 1)) * 64 + (dim8 & 1) * 32 + (b & 1) * 16 + i] =
          __builtin_bit_cast(uint4, dequant8(k[c], scale_pair(ks, c >> 1)));
    }
  }
  __device__ void store_v(uint4* lv) const {
    const int tid = int(threadIdx.x), lane = tid & 63, part = tid >> 6, g = lane >> 4, i = lane & 15;
    f16x2 s[4];
    v_scales(vs, s);
    const int t = D == 256 ? 0 : part >> 1, dd0 = (D == 256 ? part : part & 1) * R::PER;
#pragma unroll
    for (int c = 0; c < R::PER; ++c) {
      const int dd = dd0 + c;
      lv[((dd >> 1) * R::KS + 2 * t + (g >> 1)) * 64 + (g & 1) * 32 + (dd & 1) * 16 + i] =
          __builtin_bit_cast(uint4, dequant8_pairs(v[c], s));
    }
  }
};

// The tiles of TK keys that a work-group goes over (its split's part): of the cache (a linear one's slots are positions),
// then of the call's own keys, from the first to the last that one of its q-cols sees. lo_top, hi_low: positions from
// the one to below the other are seen by all of the wave's q-cols.
struct KeyTiles {
  int c_first, c_end, o_first, o_end, lo_top, hi_low;
};
template <int TK, int WAVES, int COLS>
__device__ inline KeyTiles key_tiles(const ExtArgs& a, Span all, int (&bounds)[WAVES][2], int wave, int lane, int split) {
  int lo = all.len ? all.lo : INT_MAX, hi = all.len ? all.lo + int(all.len) : 0;
  int lo_top = all.len ? all.lo : INT_MAX, hi_low = hi;
#pragma unroll
  for (int x = 1; x < COLS; x <<= 1) {
    lo = min(lo, __shfl_xor(lo, x));
    hi = max(hi, __shfl_xor(hi, x));
    lo_top = max(lo_top, __shfl_xor(lo_top, x));
    hi_low = min(hi_low, __shfl_xor(hi_low, x));
  }
  if (lane == 0) bounds[wave][0] = lo, bounds[wave][1] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) lo = min(lo, bounds[w][0]), hi = max(hi, bounds[w][1]);
  int c_lo = 0, c_n = 0, o_lo = 0, o_n = 0;
  if (hi > lo) {
    const int s_lo = a.ring ? 0 : min(lo, a.tiles), s_hi = a.ring ? a.tiles : min(min(hi, a.cached_end), a.tiles);
    if (s_hi > s_lo && lo < a.cached_end) c_lo = s_lo / TK, c_n = (s_hi + TK - 1) / TK - c_lo;
    const int j_lo = max(0, lo - a.pos0), j_hi = min(a.own, hi - a.pos0);
    if (j_hi > j_lo) o_lo = j_lo / TK, o_n = (j_hi + TK - 1) / TK - o_lo;
  }
  const int n = c_n + o_n, first = int((long long)n * split / a.splits), last = int((long long)n * (split + 1) / a.splits);
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return {uniform(c_lo + min(first, c_n)), uniform(c_lo + min(last, c_n)), uniform(o_lo + max(first, c_n) - c_n),
          uniform(o_lo + max(last, c_n) - c_n), uniform(lo_top), uniform(hi_low)};
}

template <int D, int T, int MOD>
__global__ void __launch_bounds__(kExtWaves * 64, 2) ext_rows_kernel(ExtArgs a, int kv_heads) {
  using R = Rows<D>;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ int bounds[kExtWaves][2];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int h = int(blockIdx.x) % kv_heads, block = (int(gridDim.x) - 1 - int(blockIdx.x)) / kv_heads;   // later rows,
  const int split = int(blockIdx.y);                                                                  // which see most, first
  const int col = block * 128 + wave * 32 + (lane & 31), row = col / a.group, head = h * a.group + col % a.group;
  const bool live = row < a.n_q;

  const Span all = live ? row_span(a, row) : Span{0, 0u, 0};
  const KeyTiles n = key_tiles<R::TK, kExtWaves, 32>(a, all, bounds, wave, lane, split);

  float m = -INFINITY, l = 0.f;
  f32x16 acc[R::NB];
#pragma unroll
  for (int d = 0; d < R::NB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  const size_t q_at = (size_t(row) * size_t(a.heads) + size_t(head)) * D + size_t(8 * half);

  uint4* const kbuf = reinterpret_cast<uint4*>(smem);             // two buffers each
  uint4* const vbuf = kbuf + 2 * R::kEntries;
  int* const info = reinterpret_cast<int*>(smem + size_t(R::kEntries) * 64);

  // The tiles f .. e - 1 of one kind (S: the type of its stages), the next one's loads in flight behind each. (Making the
  // scores of one tile and the products of another while a third's weights are computed was no faster, nor reading LDS
  // further ahead, nor priorities or a delay between the two work-groups of a CU.)
  auto run = [&](auto src, auto operand, int f, int e, Span span, int span_hi_low, float global) {
    constexpr int S = decltype(src)::value;
    constexpr bool OWN = decltype(operand)::value;
    using X8 = typename OperandOf<S>::type;
    if (f >= e) return;
    X8 q[R::NS];
    constexpr int QL = D == 256 && S != kBf16 ? 2 : 0;   // chunks of q in LDS, for the same reason
    X8* const ql = reinterpret_cast<X8*>(smem + R::kLds - 4096 * QL) + wave * 64 + lane;
    Score sc;
    float sc_f = 1.f;   // Score::f of the tile's plain scores (1: they have been multiplied)
    bf16x8 x[R::NS];
    row_chunks(a.q, a.bf16, live, [&](int c) { return (live ? q_at : size_t(8 * half)) + size_t(16 * c); }, x);
    Stage<D, S> stage;
    int pos = -1;
    float ks = 0.f, vs = 0.f;
    auto half_tile = [&](int t) { return !OWN && R::TK == 64 && t * 64 + 32 == a.slots_pad; };
    // BF16 tiles of 256 dims, whose stages do not fit beside q and the accumulators, go from memory to LDS directly (with
    // registers spilled, each of their reloads waited for the tile's loads: 115 us, now 93, of the case above; heads of 128
    // dims, whose stages fit, took 39.5 us so and 40.7 directly)
    constexpr bool kDirect = D == 256 && S == kBf16;
    const int rows_pad = OWN ? (a.own + 63) / 64 * 64 : a.slots_pad;
    auto load_k = [&](int t) {
      if constexpr (kDirect) {   // (past the last: nothing)
        if (t < e)
          stage.direct(OWN ? a.pk : reinterpret_cast<const uint4*>(a.ck), h, rows_pad, t, kbuf + ((t - f) & 1) * R::kEntries, false);
      }
      t = min(t, e - 1);   // past the last: loaded again, and not used
      pos = -1;
      if constexpr (OWN) {
        if constexpr (!kDirect) stage.load_k(a.pk, h, rows_pad, t, false);
        if (tid < R::TK && t * R::TK + tid < a.own) pos = a.pos0 + t * R::TK + tid;
      } else {
        if constexpr (S == kNvfp4)
          stage.load_k(a, h, t, half_tile(t));
        else if constexpr (!kDirect)
          stage.load_k(reinterpret_cast<const uint4*>(a.ck), h, a.slots_pad, t, half_tile(t));
        if (tid < (half_tile(t) ? 32 : R::TK)) {
          pos = a.slot_pos[t * R::TK + tid];
          if constexpr (S == kFp8) {
            const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(t * R::TK + tid);
            ks = static_cast<const float*>(a.ks)[at];
            vs = static_cast<const float*>(a.vs)[at];
          }
        }
      }
    };
    auto load_v = [&](int t) {
      if constexpr (kDirect) {
        if (t < e)
          stage.direct(OWN ? a.pv : reinterpret_cast<const uint4*>(a.cv), h, rows_pad, t, vbuf + ((t - f) & 1) * R::kEntries, true);
        return;
      }
      t = min(t, e - 1);
      if constexpr (OWN)
        stage.load_v(a.pv, h, rows_pad, t, false);
      else if constexpr (S == kNvfp4)
        stage.load_v(a, h, t, half_tile(t));
      else
        stage.load_v(reinterpret_cast<const uint4*>(a.cv), h, a.slots_pad, t, half_tile(t));
    };
    auto store_k = [&](int t) {
      if constexpr (!kDirect) stage.store_k(kbuf + ((t - f) & 1) * R::kEntries);
      int* lp = info + ((t - f) & 1) * R::kInfo;
      if (wave == 0) {   // the tile's last and first positions, -1 with a slot that has none
        int top = pos, least = tid < R::TK ? pos : INT_MAX;
        wave_extremes(top, least);
        if (tid == 0) lp[3 * R::TK] = top, lp[3 * R::TK + 1] = least;
        if (tid < R::TK) {
          lp[tid] = pos;
          if constexpr (S == kFp8) {   // a key whose V scale is not finite is NaN itself, and the scale zero
            reinterpret_cast<float*>(lp)[R::TK + tid] = not_finite(vs) ? NAN : ks;
            reinterpret_cast<float*>(lp)[2 * R::TK + tid] = not_finite(vs) ? 0.f : vs;
          }
        }
      }
    };
    auto store_v = [&](int t) {
      if constexpr (kDirect)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the tile's loads into LDS, before the barrier behind
      else
        stage.store_v(vbuf + ((t - f) & 1) * R::kEntries);
    };
    auto scores = [&](int t, f32x16 (&s)[R::KB]) {
      const X8* lk = reinterpret_cast<const X8*>(kbuf + ((t - f) & 1) * R::kEntries);
#pragma unroll
      for (int b = 0; b < R::KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
      for (int c = 0; c < R::NS; ++c)
#pragma unroll
        for (int b = 0; b < R::KB; ++b) s[b] = mfma32(lk[(b * R::NS + c) * 64 + lane], c < R::NS - QL ? q[c] : ql[(c - R::NS + QL) * 256], s[b]);
    };
    X8 w[R::KS];
    auto products = [&](int t) {
      const X8* lv = reinterpret_cast<const X8*>(vbuf + ((t - f) & 1) * R::kEntries);
#pragma unroll
      for (int k = 0; k < R::KS; ++k)
#pragma unroll
        for (int d = 0; d < R::NB; ++d) acc[d] = mfma32(lv[(d * R::KS + k) * 64 + lane], w[k], acc[d]);
    };

    // scores begun (masked) in y, m moved if they pass it; then their weights
    auto softmax_begin = [&](int t, const f32x16 (&s)[R::KB], float (&y)[R::KB][16]) {
      const int* lp = info + ((t - f) & 1) * R::kInfo;
      // row 8 j + r' of block b (r = 4 j + r') is key 32 b + 8 j + 4 half + r'
      const int4* lp4 = reinterpret_cast<const int4*>(lp) + half;
      const float4* lf4 = reinterpret_cast<const float4*>(lp) + half;
#pragma unroll
      for (int b = 0; b < R::KB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          int p[4] = {0, 0, 0, 0};
          float k4[4] = {1.f, 1.f, 1.f, 1.f};
          if constexpr ((MOD & kBias) != 0) {
            const int4 p4 = lp4[b * 8 + j * 2];
            p[0] = p4.x, p[1] = p4.y, p[2] = p4.z, p[3] = p4.w;
          }
          if constexpr (S == kFp8) {
            const float4 z = lf4[R::TK / 4 + b * 8 + j * 2];
            k4[0] = z.x, k4[1] = z.y, k4[2] = z.z, k4[3] = z.w;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            y[b][4 * j + r] = begin<MOD>(sc, S == kFp8 ? s[b][4 * j + r] * k4[r] : s[b][4 * j + r], span.t - p[r]);
        }
      // the tile's positions against what the wave's q-cols see: all, or a mask
      const int top = __builtin_amdgcn_readfirstlane(lp[3 * R::TK]), least = __builtin_amdgcn_readfirstlane(lp[3 * R::TK + 1]);
      if (least < n.lo_top || top >= span_hi_low) {
#pragma unroll
        for (int b = 0; b < R::KB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int4 p4 = lp4[b * 8 + j * 2];
            const int p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (uint32_t(p[r] - span.lo) >= span.len) y[b][4 * j + r] = masked<MOD>();
          }
      }
      float mx = masked<MOD>();
#pragma unroll
      for (int b = 0; b < R::KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = best<MOD>(mx, y[b][r]);
      mx = xor32_max(finish<MOD>(sc, mx, 0.f));
      if constexpr (MOD == 0) {
        sc_f = sc.f;
        if (__ballot(fabsf(mx) >= kLarge && fabsf(mx) <= FLT_MAX)) {
          sc_f = 1.f;
#pragma unroll
          for (int b = 0; b < R::KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) y[b][r] *= sc.f;
        }
      }
      if (__ballot(mx > m + kSlack)) {
        const float to = mx > m + kSlack ? mx : m;
        const float corr = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f : to));
        m = to;
        l *= corr;
#pragma unroll
        for (int d = 0; d < R::NB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= corr;
      }
    };
    auto softmax_end = [&](int t, const float (&y)[R::KB][16]) {
      const float4* lf4 = reinterpret_cast<const float4*>(info + ((t - f) & 1) * R::kInfo) + half;
      const float ref = (m == -INFINITY ? 0.f : m) - kUp;
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < R::KB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v4[4] = {1.f, 1.f, 1.f, 1.f};
          if constexpr (S == kFp8) {
            const float4 z = lf4[2 * R::TK / 4 + b * 8 + j * 2];
            v4[0] = z.x, v4[1] = z.y, v4[2] = z.z, v4[3] = z.w;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float p = __builtin_amdgcn_exp2f(MOD ? finish<MOD>(sc, y[b][4 * j + r], ref) : fmaf(y[b][4 * j + r], sc_f, -ref));
            sum += p;
            if constexpr (S == kFp8) p *= v4[r];
            w[2 * b + (j & 1)][(j >> 1) * 4 + r] = p;
          }
        }
      l += sum;
    };

    if constexpr (kDirect) __syncthreads();
    load_k(f);
    load_v(f);
    if constexpr (!kDirect) __syncthreads();   // the buffers may still be read by what ran before
    store_k(f);
    if (a.scale < 0.f) {
#pragma unroll
      for (int c = 0; c < R::NS; ++c) x[c] = -x[c];
    }
    const int ex = to_operand<S != kBf16>(x, q, [](float y) { return xor32_max(y); });
    sc = score_of(a, live ? head : 0, global, ex);
#pragma unroll
    for (int c = 0; c < QL; ++c) ql[c * 256] = q[R::NS - QL + c];
    f32x16 s[R::KB];
    float y[R::KB][16];
    store_v(f);
    __syncthreads();
    for (int t = f; t < e; ++t) {
      load_k(t + 1);
      load_v(t + 1);
      scores(t, s);
      softmax_begin(t, s, y);
      softmax_end(t, y);
      products(t);
      store_k(t + 1);
      store_v(t + 1);
      __syncthreads();
    }
  };
  run(std::integral_constant<int, T>{}, std::false_type{}, n.c_first, n.c_end, cached_span(a, all),
      min(n.hi_low, a.cached_end), T == kNvfp4 ? a.kglobal : 1.f);
  if (T == kNvfp4 && a.vglobal != 1.f) {
#pragma unroll
    for (int d = 0; d < R::NB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= a.vglobal;
  }
  run(std::integral_constant<int, kBf16>{}, std::true_type{}, n.o_first, n.o_end, all, n.hi_low, 1.f);

  l = xor32_sum(l);
  if (a.splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bool bad = false;
#pragma unroll
    for (int d = 0; d < R::NB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) bad |= live && not_finite(acc[d][r]);
    const long long out = live ? (long long)((size_t(row) * size_t(a.heads) + size_t(head)) * D) : -1;
    __syncthreads();   // the last tile's buffer, and bounds
    // a lane has a q-col's values 512 bytes or more from its neighbour's: they are turned in LDS, a wave its own 32 rows
    auto write = [&](auto* to) {
      using X = std::remove_pointer_t<decltype(to)>;
      constexpr int DP = sizeof(X) == 4 && D > 128 ? 128 : D, PITCH = DP + 16 / int(sizeof(X));   // dims of a pass
      static_assert(kExtWaves * 32 * PITCH * sizeof(X) <= R::kLds, "the tiles' buffers hold the rows");
      X* mine = reinterpret_cast<X*>(smem) + wave * 32 * PITCH;
#pragma unroll
      for (int p = 0; p < D; p += DP) {
        if (p) __syncthreads();
#pragma unroll
        for (int d = 0; d < R::NB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int v = 32 * d + 8 * (r >> 2) + (r & 3);   // and 4 half
            const int low = Tile<D, T>::dim(v >> 4, v & 15), step = Tile<D, T>::dim(0, 4) - Tile<D, T>::dim(0, 0);
            if (low < p || low >= p + DP) continue;   // (with half = 1 on the same side)
            mine[(lane & 31) * PITCH + low - p + half * step] = X(acc[d][r] * inv);
          }
        __syncthreads();
        constexpr int CH = DP * int(sizeof(X)) / 16, PER = 64 / CH;   // 16-byte pieces of a row; rows at a time
#pragma unroll
        for (int c = 0; c < 32; c += PER) {
          const int of = c + lane / CH, piece = lane % CH;
          const int lo32 = __shfl(int(uint32_t(out)), of), hi32 = __shfl(int(out >> 32), of);
          if (hi32 < 0) continue;
          const size_t at = (size_t(uint32_t(hi32)) << 32 | size_t(uint32_t(lo32))) + size_t(p);
          reinterpret_cast<uint4*>(to + at)[piece] = reinterpret_cast<const uint4*>(mine + of * PITCH)[piece];
        }
      }
    };
    if (a.bf16)
      write(static_cast<__bf16*>(a.out));
    else
      write(static_cast<float*>(a.out));
    const uint64_t any = __ballot((bad && !not_finite(l)) || (live && no_sum(l, row)));
    if (lane == 0) bounds[wave][0] = int(uint32_t(any) | uint32_t(any >> 32));
    __syncthreads();
    for (int w = 0; w < kExtWaves; ++w)
      for (uint32_t bits = uint32_t(bounds[w][0]); bits; bits &= bits - 1) {
        const int c = block * 128 + w * 32 + __builtin_ctz(bits);
        slow_col<D, T>(args_again(), h, kv_heads, c / a.group, h * a.group + c % a.group, reinterpret_cast<float*>(smem));
      }
    return;
  }
  if (!live) return;
  const size_t rec = ((size_t(block) * size_t(kv_heads) + size_t(h)) * size_t(a.splits) + size_t(split)) * 128 +
                     size_t(wave * 32 + (lane & 31));
#pragma unroll
  for (int d = 0; d < R::NB; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<f32x4*>(a.acc + rec * D + size_t(32 * d + 8 * j + 4 * half)) =
          f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
  if (half == 0) a.ml[rec * 2] = m, a.ml[rec * 2 + 1] = l;
}

// ---------------------------------------------------------------------------------------------------- merge

// A q-col's records: their weights 2^(m - largest m) first, then the sums, D / 4 lanes to a record's accumulator and G
// groups of lanes with the records s = group, group + G, .., whose sums are added in order. A batch of B accumulators is
// loaded before the weights are known: few q-cols' records are a matter of latency. G = 1 (up to 16 records): a work-group
// has several q-cols; 1440 of 9 records of 128 dims took 3.9 us so and 6.5 with a work-group each.
template <int D, int T, int G, int B>
__global__ void __launch_bounds__(256) ext_merge_kernel(ExtArgs a, int kv_heads, int total) {
  constexpr int L = D / 4, PER = 256 / (L * G);   // lanes a record; q-cols of a work-group
  __shared__ float4 part[G > 1 ? PER * G * L : 1];
  __shared__ float slow[272 + D], all_m[4], all_l[4];
  __shared__ int again[PER];
  const int tid = int(threadIdx.x), x = tid % L, grp = tid / L % G, mine = tid / (L * G);
  const int id = int(blockIdx.x) * PER + mine;   // q-col of the call: row * heads + head
  const bool live = id < total;
  const int row = live ? id / a.heads : 0, head = live ? id % a.heads : 0, h = head / a.group, c = row * a.group + head % a.group;
  if (x == 0 && grp == 0) again[mine] = 0;
  // record s's accumulator, maximum and sum
  const size_t rec0 = (size_t(c / a.cols) * size_t(kv_heads) + size_t(h)) * size_t(a.records) * size_t(a.cols) + size_t(c % a.cols);
  const float* acc = a.acc + rec0 * D + size_t(4 * x);
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + rec0;
  float4 v[B];
  float2 w[B];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int s = s0 + k * G;
      w[k] = s < a.records ? ml[size_t(s) * size_t(a.cols)] : make_float2(-INFINITY, 0.f);
      v[k] = s < a.records ? *reinterpret_cast<const float4*>(acc + size_t(s) * size_t(a.cols) * D) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  load(grp);
  // the largest maximum and the sum at it: a thread a record where a work-group has one q-col, else every thread all
  float m = -INFINITY, l = 0.f;
  if constexpr (G > 1) {
    for (int s = tid; s < a.records; s += 256) m = fmaxf(m, ml[size_t(s) * size_t(a.cols)].x);
    m = wave_max(m);
    if ((tid & 63) == 0) all_m[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(all_m[0], all_m[1]), fmaxf(all_m[2], all_m[3]));
  } else {
#pragma unroll
    for (int k = 0; k < B; ++k) m = fmaxf(m, w[k].x);   // (G = 1: all of them, B or fewer)
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = grp; s0 < a.records; s0 += B * G) {
    if (s0 != grp) load(s0);
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const float f = __builtin_amdgcn_exp2f(w[k].x - ref);
      l += w[k].y * f;
      if (f != 0.f)   // (a record whose maximum is far below, or that saw nothing, adds nothing)
        y.x += v[k].x * f, y.y += v[k].y * f, y.z += v[k].z * f, y.w += v[k].w * f;
    }
  }
  if constexpr (G > 1) {
    part[tid] = y;
    l = x == 0 ? l : 0.f;   // a group's sum once; the groups' over the work-group
    l = wave_sum(l);
    if ((tid & 63) == 0) all_l[tid >> 6] = l;
    __syncthreads();
    l = all_l[0] + all_l[1] + all_l[2] + all_l[3];
    y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp == 0) {
#pragma unroll
      for (int s = 0; s < G; ++s) {
        const float4 u = part[s * L + x];
        y.x += u.x, y.y += u.y, y.z += u.z, y.w += u.w;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float o[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
  const bool bad = live && !not_finite(l) &&
                   (not_finite(y.x) || not_finite(y.y) || not_finite(y.z) || not_finite(y.w) || no_sum(l, row));
  if (live && grp == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int u = 4 * x + r;
      const size_t at = size_t(id) * D + size_t(Tile<D, T>::dim(u >> 4, u & 15));
      if (a.bf16)
        static_cast<__bf16*>(a.out)[at] = (__bf16)o[r];
      else
        static_cast<float*>(a.out)[at] = o[r];
    }
  }
  if (!__syncthreads_or(bad)) return;
  if (bad) again[mine] = 1;
  __syncthreads();
  for (int k = 0; k < PER; ++k)
    if (again[k]) {
      const int q = int(blockIdx.x) * PER + k;
      slow_col<D, T>(args_again(), q % a.heads / a.group, kv_heads, q / a.heads, q % a.heads, slow);
    }
}

// ---------------------------------------------------------------------------------------------------- launches

template <int D, int T, int MOD>
void launch(const ExtCall& c, const ExtPlan& p, const ExtArgs& a, hipStream_t stream, const Timed& timed) {
  if (p.few) {
    timed([&] {
      const dim3 grid{unsigned(c.kv_heads), unsigned(a.records), unsigned(p.blocks)}, block{kExtWaves * 64};
      auto go = [&](auto kernel, size_t lds) {
        allow_lds(reinterpret_cast<const void*>(kernel), lds);
        hipLaunchKernelGGL(kernel, grid, block, lds, stream, a);
      };
      if (p.cols == 16)
        go(&ext_few_kernel<D, 1, T, MOD>, few_lds<D, 1>());
      else
        go(&ext_few_kernel<D, 2, T, MOD>, few_lds<D, 2>());
      HIP_CHECK(hipGetLastError());
      return strf("ext_few_kernel<%d, %d, %d, %d>", D, p.cols / 16, T, MOD);
    });
  } else {
    if (c.k)
      timed([&] {
        const int tiles = (c.n_q + 63) / 64 * 2;
        const long long threads = (long long)tiles * c.kv_heads * (36 * D / 8);
        hipLaunchKernelGGL((ext_pack_kernel<D, T>), dim3(unsigned((threads + 255) / 256)), dim3(256), 0, stream, c.k, c.v,
                           a.bf16, c.n_q, c.kv_heads, tiles, const_cast<uint4*>(a.pk), const_cast<uint4*>(a.pv));
        HIP_CHECK(hipGetLastError());
        return strf("ext_pack_kernel<%d, %d>", D, T);
      });
    timed([&] {
      const dim3 grid{unsigned(c.kv_heads) * unsigned(p.blocks), unsigned(p.splits)};
      const size_t lds = Rows<D>::kLds;
      allow_lds(reinterpret_cast<const void*>(&ext_rows_kernel<D, T, MOD>), lds);
      hipLaunchKernelGGL((ext_rows_kernel<D, T, MOD>), grid, dim3(kExtWaves * 64), lds, stream, a, c.kv_heads);
      HIP_CHECK(hipGetLastError());
      return strf("ext_rows_kernel<%d, %d, %d>", D, T, MOD);
    });
  }
  if (a.records > 1)
    timed([&] {
      constexpr int G = 1024 / D;   // 256 threads, D / 4 a record: G records at once, or G q-cols of at most 16
      const int total = c.n_q * c.heads, groups = a.records > 16 ? G : 1;
      auto go = [&](auto kernel, int cols) {
        hipLaunchKernelGGL(kernel, dim3(unsigned((total + cols - 1) / cols)), dim3(256), 0, stream, a, c.kv_heads, total);
      };
      if (groups > 1)
        go(&ext_merge_kernel<D, T, G, 8>, 1);
      else if (a.records > 8)
        go(&ext_merge_kernel<D, T, 1, 16>, G);
      else
        go(&ext_merge_kernel<D, T, 1, 8>, G);
      HIP_CHECK(hipGetLastError());
      return strf("ext_merge_kernel<%d, %d, %d>", D, T, groups);
    });
}

template <int D, int T>
void launch_scores(const ExtCall& c, const ExtPlan& p, const ExtArgs& a, hipStream_t stream, const Timed& timed) {
  if (c.softcap > 0.f && c.slopes)
    launch<D, T, kCap | kBias>(c, p, a, stream, timed);
  else if (c.softcap > 0.f)
    launch<D, T, kCap>(c, p, a, stream, timed);
  else if (c.slopes)
    launch<D, T, kBias>(c, p, a, stream, timed);
  else
    launch<D, T, 0>(c, p, a, stream, timed);
}

// A call of heads of D dims over a cache of `dtype`; each D is compiled in a file of its own.
template <int D>
void ext_launch(const ExtCall& c, const ExtPlan& p, const ExtArgs& a, int dtype, hipStream_t stream, const Timed& timed) {
  if (dtype == kBf16)
    launch_scores<D, kBf16>(c, p, a, stream, timed);
  else if (dtype == kFp8)
    launch_scores<D, kFp8>(c, p, a, stream, timed);
  else
    launch_scores<D, kNvfp4>(c, p, a, stream, timed);
}

}  // namespace xtg::hip
