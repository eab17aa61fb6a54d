// What the kernels of attention over a cache of any dtype share: operands of the matrix ops, scores in base-2 units, a wave's
// 32-slot tile of a cache in registers, and one step of a wave over it.
//
// Both products are matrix ops with the keys as rows, S^T = K Q^T and O^T = V^T P^T: a lane holds the scores of one q-col (a
// row of the call and one of the q heads of a KV head), and the weights that it computes from them are the B operand of the
// second product as they are. A row sees the positions lo <= p < hi, so a mask is one unsigned comparison.
#pragma once

#include <cfloat>
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

// What turns a product q.k into a score in base-2 units.
struct Score {
  float f;             // times this (the scale, or with a cap what the exponential takes)
  float top, slope;    // cap * log2(e); the head's slope * log2(e)
};
// Score::f for operands whose product times global * 2^ex is q.k (a power of two too). Exponents are added as integers: those of
// a small cap, a global and a q-col pass FP32 together. (It stays finite and above zero: times an infinity one, times zero
// none.)
__device__ inline float score_factor(float factor, int factor_exp, float global, int ex) {
  return fminf(fmaxf(ldexpf(factor * global, factor_exp + ex), FLT_MIN), FLT_MAX);
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

// A load of a tile's codes. STREAM: past the caches, for a cache that is read once (decode steps of 64 sequences over 8-bit
// pages: 100.7 -> 90.6 us; but a prompt's blocks, which read the same tiles, 82 -> 86).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool STREAM>
__device__ inline uint4 load16(const uint4* p) {
  if constexpr (STREAM) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
  return *p;
}

// A wave's tile of 32 slots: the keys of a lane's scores are slots 4 g + e and 16 + 4 g + e - 4. k(b, st), v(dd): the
// operands; dim(dd, r): the dim of row r of product dd. A tile is loaded from `at`, its first slot's place in the head-major arrays
// a.ck, a.cv, a.ks and a.vs (A::kStream: load16).
template <int D, int T>
struct Tile;

template <int D>
struct Tile<D, kBf16> {
  uint4 kw[2][D / 32], vw[D / 16];
  static constexpr bool kScaled = false;
  __device__ static int q_dim(int st, int g) { return 32 * st + 8 * g; }
  __device__ static int dim(int dd, int r) { return 16 * dd + r; }
  template <class A>
  __device__ void load_k(const A& a, size_t at, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.ck) + at * (D / 8) + lane;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) kw[b][c] = load16<A::kStream>(p + (b * (D / 32) + c) * 64);
  }
  template <class A>
  __device__ void load_v(const A& a, size_t at, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.cv) + at * (D / 8) + lane;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd) vw[dd] = load16<A::kStream>(p + dd * 64);
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
  template <class A>
  __device__ void load_k(const A& a, size_t at, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.ck) + at * (D / 16) + lane;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) kw[b][c] = load16<A::kStream>(p + (b * (D / 64) + c) * 64);
    load8(ks, static_cast<const float*>(a.ks) + at + 4 * (lane >> 4));
    load8(vs, static_cast<const float*>(a.vs) + at + 4 * (lane >> 4));
  }
  __device__ static void load8(float (&x)[8], const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 16);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  template <class A>
  __device__ void load_v(const A& a, size_t at, int lane) {
    const uint4* p = reinterpret_cast<const uint4*>(a.cv) + at * (D / 16) + lane;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) vw[c] = load16<A::kStream>(p + c * 64);
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
  template <class A>
  __device__ void load_k(const A& a, size_t at, int lane) {
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
  template <class A>
  __device__ void load_v(const A& a, size_t at, int lane) {
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

// The state of a lane's q-col in each block of 16: the maximum (the same in the col's 4 lanes), the lane's own part of the
// sum, and the accumulator: rows 4 g + r of product dd.
template <int D, int QB>
struct FewState {
  float m[QB], l[QB];
  f32x4 acc[QB][D / 16];
};

// A q operand in LDS says so with kInLds: its chunks are then read one ahead of their products, no sooner (all at once they
// took as many registers as an operand that is kept there).
template <class Q, class = void>
struct InLds : std::false_type {};
template <class Q>
struct InLds<Q, std::enable_if_t<Q::kInLds>> : std::true_type {};

// One tile. q(qb, c): chunk c of the operand of a lane's q-col in block qb. next_k loads the next tile's keys once this one's are used, next_v its values: each load has about half a
// tile's work to land behind. TWO (BF16 operands): a weight is the sum of two BF16 values, 15 bits of it, else one of 8 (f16: 11).
template <int D, int QB, int MOD, bool TWO = false, class TILE, class Q, class NK, class NV>
__device__ inline void few_tile(TILE& T, Q&& q, const Span (&span)[QB],
                                const Score (&sc)[QB], FewState<D, QB>& st, int4 p0, int4 p1, NK&& next_k, NV&& next_v) {
  const int pos[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
  using X8 = decltype(q(0, 0));
  constexpr bool kAhead = InLds<std::remove_reference_t<Q>>::value;
  f32x4 s[QB][2];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) s[qb][0] = s[qb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  X8 x[QB], ahead[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) ahead[qb] = q(qb, 0);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      x[qb] = ahead[qb];
      if (c + 1 < D / 32) ahead[qb] = q(qb, c + 1);
    }
    if constexpr (kAhead) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const X8 k = T.k(b, c);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) s[qb][b] = mfma16(k, x[qb], s[qb][b]);
    }
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
  X8 w[QB], rest[QB];
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
      if constexpr (TWO) {   // cut, not rounded, and 2^-17 more: both above zero, so that an infinite value times both is one
        const float cut = __uint_as_float(__float_as_uint(p) & 0xffff0000u);
        rest[qb][e] = fmaf(p, 1.f + 0x1p-17f, -cut);
        p = cut;
      }
      w[qb][e] = p;
    }
  }
  T.begin_v();
#pragma unroll
  for (int dd = 0; dd < D / 16; ++dd) {
    const X8 v = T.v(dd);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      st.acc[qb][dd] = mfma16(v, w[qb], st.acc[qb][dd]);
      if constexpr (TWO) st.acc[qb][dd] = mfma16(v, rest[qb], st.acc[qb][dd]);
    }
  }
  next_v();
}

// ------------------------------------------------------------------------------------------ tiles in LDS

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

// A thread's number among the 256 that share tiles; GROUPS: the work-group has more than one such.
template <bool GROUPS>
__device__ inline int stage_thread() { return GROUPS ? int(threadIdx.x) & 255 : int(threadIdx.x); }

// What a thread stages of a tile: loads in flight (raw), then entries written to LDS. A cache of an odd number of 32-slot
// tiles ends in the middle of a 64-key tile (`half`): its other half is zeros.
template <int D, int T, bool GROUPS = false>
struct Stage;

// BF16: entries as they are. Also the packed own keys.
template <int D, bool GROUPS>
struct Stage<D, kBf16, GROUPS> {
  using R = Rows<D>;
  uint4 k[R::PER], v[R::PER];
  __device__ static void load(uint4 (&x)[R::PER], const uint4* c, int h, int pad, int tile, bool half) {
    const size_t at = (size_t(h) * size_t(pad) + size_t(tile) * R::TK) * (D / 8) + size_t(stage_thread<GROUPS>());
#pragma unroll
    for (int u = 0; u < R::PER; ++u) x[u] = half && 2 * u >= R::PER ? make_uint4(0, 0, 0, 0) : c[at + u * 256];
  }
  __device__ void load_k(const uint4* ck, int h, int pad, int tile, bool half) { load(k, ck, h, pad, tile, half); }
  __device__ void load_v(const uint4* cv, int h, int pad, int tile, bool half) { load(v, cv, h, pad, tile, half); }
  // The tile straight into its place in LDS: 64 entries a wave's load, a lane's the one that comes to its part of them.
  __device__ static void direct(const uint4* from, uint4* to, bool v) {
    const int lane = stage_thread<GROUPS>() & 63, half = lane >> 5, i = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(stage_thread<GROUPS>() >> 6);
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
    for (int u = 0; u < R::PER; ++u) lk[k_place(stage_thread<GROUPS>() + u * 256)] = k[u];
  }
  __device__ void store_v(uint4* lv) const {
#pragma unroll
    for (int u = 0; u < R::PER; ++u) lv[v_place(stage_thread<GROUPS>() + u * 256)] = v[u];
  }
};

// FP8: a 16-byte load is two entries' codes.
template <int D, bool GROUPS>
struct Stage<D, kFp8, GROUPS> {
  using R = Rows<D>;
  using B = Stage<D, kBf16, GROUPS>;
  uint4 k[R::PER / 2], v[R::PER / 2];
  __device__ static void load(uint4 (&x)[R::PER / 2], const uint4* c, int h, int pad, int tile, bool half) {
    const size_t at = (size_t(h) * size_t(pad) + size_t(tile) * R::TK) * (D / 16) + size_t(stage_thread<GROUPS>());
#pragma unroll
    for (int u = 0; u < R::PER / 2; ++u) {
      const bool past = half && stage_thread<GROUPS>() + u * 256 >= R::kEntries / 4;
      x[u] = past ? make_uint4(0, 0, 0, 0) : c[at + u * 256];
    }
  }
  __device__ void load_k(const uint4* ck, int h, int pad, int tile, bool half) { load(k, ck, h, pad, tile, half); }
  __device__ void load_v(const uint4* cv, int h, int pad, int tile, bool half) { load(v, cv, h, pad, tile, half); }
  __device__ static int first(int u) {   // of BF16's entries
    const int x = stage_thread<GROUPS>() + u * 256;
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
template <int D, bool GROUPS>
struct Stage<D, kNvfp4, GROUPS> {
  using R = Rows<D>;
  uint32_t k[R::PER], v[R::PER], ks;
  uint2 vs;
  template <class A>
  __device__ void load_k(const A& a, int h, int tile, bool half) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(tile) * R::TK;
    const int tid = stage_thread<GROUPS>();
#pragma unroll
    for (int u = 0; u < R::PER; ++u) k[u] = 0;
    ks = 0;
    if (half && tid >= 128) return;
    take(k, a.ck + at * (D / 2), tid);
    const uint8_t* s = static_cast<const uint8_t*>(a.ks) + at * (D / 16);
    ks = D == 64 ? s[tid] : reinterpret_cast<const uint16_t*>(s)[tid];
  }
  // V: a wave has half a 32-slot tile's words (256 dims: a quarter)
  template <class A>
  __device__ void load_v(const A& a, int h, int tile, bool half) {
    const size_t at = size_t(h) * size_t(a.slots_pad) + size_t(tile) * R::TK;
    const int tid = stage_thread<GROUPS>(), lane = tid & 63, part = tid >> 6, t = D == 256 ? 0 : part >> 1;
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
    const int tid = stage_thread<GROUPS>(), lane = tid & 63, part = tid >> 6, g = lane >> 4, i = lane & 15;
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
    const int tid = stage_thread<GROUPS>(), lane = tid & 63, part = tid >> 6, g = lane >> 4, i = lane & 15;
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

}  // namespace xtg::hip
