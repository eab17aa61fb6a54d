// Rows into the pages of a pool, rotated and normalised on the way, and rows of pages back (layouts: attention.hpp, kv4.hpp).
//
// A work-group takes what a call has of one 32-slot tile of a sequence, for one KV head: of K a thread takes 8 dims of a key
// and the 8 that they turn with, of V a wave takes a group of 8 slots and a thread a few of their dims, so that V's words,
// which hold 8 slots, are written whole where the call has all of them. Rotation: o1 = x1 cos - x2 sin, o2 = x2 cos + x1 sin
// with the angle pos * theta^(-2i/d), its sine and cosine in 64 bits (in 32 an angle of 30000 radians is off by 0.001).
// HBM bounds a prompt's rows: 4311 rows of 32 q heads and 8 KV heads of 128 dims, BF16, 106 MB, in 23 to 24 us (4.4 to 4.6 TB/s); into
// FP8 and NVFP4 pages, 97 and 93 MB, in 24. A decode step's rows are one chain of loads and stores, 4 to 7 us.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention.hpp"
#include "attention_ext.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "kv4.hpp"
#include "kv_rows.hpp"
#include "paged_device.hpp"

namespace xtg::hip {

struct AppendArgs {
  Seqs s;
  uint8_t *ck, *cv, *ks, *vs;
  const void *q, *k, *v;
  void* q_out;
  long long ldq, ldk, ldv;
  int heads, kv_heads, tasks, norm;
  const double* freq;
  const float* qscale;
  float kglobal, vglobal, kinv, vinv;   // NVFP4's, and their inverses, exact
};

// cos and sin of p quarter turns times f, in 64 bits and rounded once (in 32 bits their own roundings nearly doubled the error
// of a turned key: of BF16 keys 7e-6 against 4e-6, and 3 % of the time of a prompt's rows). p * f is off by 2^-53 of itself:
// under 2^-22 radians for positions up to 2^30, where pages end; queries may be further on, up to an int's last and a call's rows
// behind it (p * f, under 0.64 p, still fits an int). The series are cut at x^13 and x^14, of |x| <= pi / 4: under 2^-36.
__device__ inline float2 turned(double p, double f) {
  const double t = p * f, n = rint(t), x = (t - n) * 1.5707963267948966, y = x * x;
  const int quarter = int(n) & 3;
  const double s = x * fma(y, fma(y, fma(y, fma(y, fma(y, -1.0 / 39916800, 1.0 / 362880), -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
  const double c = fma(y, fma(y, fma(y, fma(y, fma(y, fma(y, 1.0 / 479001600, -1.0 / 3628800), 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5), 1.0);
  const float a = float(quarter & 1 ? s : c), b = float(quarter & 1 ? c : s);
  return make_float2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// Sum over LANES neighbours (4, 8 or 16), in each of them.
template <int LANES>
__device__ inline float over_lanes(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  if constexpr (LANES >= 8) v += dpp<kDppHalfMirror>(v);
  if constexpr (LANES >= 16) v += dpp<kDppMirror>(v);
  return v;
}

// Of a head's row, dims 8 c .. +8 and D / 2 + 8 c .. +8 (lo, hi), by D / 16 neighbouring lanes: rotated, then justnorm of
// the row.
template <int D>
__device__ inline void rotate(float (&lo)[8], float (&hi)[8], const float2 (&cs)[8], bool turn, int norm) {
  if (turn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = lo[e] * cs[e].x - hi[e] * cs[e].y;
      hi[e] = hi[e] * cs[e].x + lo[e] * cs[e].y;
      lo[e] = a;
    }
  }
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
    const float f = inv_norm_of(over_lanes<D / 16>(ss));
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] *= f, hi[e] *= f;
  }
}

__device__ inline uint32_t fp8_codes(float a, float b, float c, float d) {
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true));
}

// The scale of an FP8 row whose largest magnitude is amax, and its inverse. The scale is amax times the FP32 number nearest to
// 1/448, as torch divides by a constant, so that rows quantised by its operations get the same codes: about one BF16 row of six
// has values midway between two codes, which the last bit of the scale decides (with the quotient, a few rows were up to 0.9 %
// of their norm apart). A row below FP32's normal scales, whose inverse would be infinite, has scale 1 and is zeros.
struct Scale8 {
  float s, inv;
};
__device__ inline Scale8 scale8(float amax) {
  Scale8 r;
  r.s = amax >= 448.f * FLT_MIN ? amax * (1.f / 448.f) : 1.f;
  r.inv = 1.f / r.s;
  return r;
}

// Largest magnitude of a row's lanes; a NaN is passed over (its code is NaN).
__device__ inline float amax8(const float (&x)[8]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
  return m;
}
template <int LANES>
__device__ inline float max_over_lanes(float v) {
  v = fmaxf(v, dpp<kDppXor1>(v));
  v = fmaxf(v, dpp<kDppXor2>(v));
  if constexpr (LANES >= 8) v = fmaxf(v, dpp<kDppHalfMirror>(v));
  if constexpr (LANES >= 16) v = fmaxf(v, dpp<kDppMirror>(v));
  return v;
}

// The slots of element e of V's words of group g, and the tile and rows of a task.
__device__ inline int v_slot(int g, int e) { return e < 4 ? 4 * g + e : 12 + 4 * g + e; }

struct TileTask {
  int seq, head, tile;     // tile: its first position / 32
  int slot;                // its first slot in the page
  int page;                // -1: none
  Seq q;
  __device__ int row(int key) const {   // the call's row at the tile's position `key`, or -1
    const int r = 32 * tile + key - q.pos;
    return uint32_t(r) < uint32_t(q.n) ? q.row0 + r : -1;
  }
};
// Tiles that a sequence's rows are in.
__device__ inline int tiles_of(const Seq& q) {
  if (q.pos < 0 || q.n == 0) return 0;
  return ((q.pos + q.n - 1) >> 5) - (q.pos >> 5) + 1;
}
__device__ inline bool tile_task(const Seqs& s, int kv_heads, int id, TileTask& t) {
  const int task = id / kv_heads;
  t.head = id % kv_heads;
  int at = 0;
  if (s.starts) {
    if (!find_task(s.n_seqs, task, [&](int x) { return tiles_of(seq_at(s, x)); }, t.seq, at)) return false;
  } else {
    t.seq = task;
    if (task >= s.n_seqs) return false;
  }
  t.q = seq_at(s, t.seq);
  if (at >= tiles_of(t.q)) return false;
  t.tile = (t.q.pos >> 5) + at;
  t.page = page_of(s, t.seq, 32 * t.tile);
  t.slot = 32 * t.tile & ((1 << s.shift) - 1);
  return true;
}

template <int D, int T, class X>
__device__ inline void append_tile(const AppendArgs& a, uint32_t* not_finite) {
  constexpr int C = D / 16, KP = 256 / C < 32 ? 256 / C : 32, P = D / 64;
  const int tid = int(threadIdx.x), size = 1 << a.s.shift;
  const int c = tid % C, key0 = tid / C;
  // Loads go out as soon as what they need is known: frequencies, then the rows, then the page.
  double f[8] = {};
  if (a.freq) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = a.freq[8 * c + e];
  }
  TileTask t;
  if (!tile_task(a.s, a.kv_heads, int(blockIdx.x), t)) return;   // (the whole work-group)
  const int v_dim = (tid & 63) * P, g = tid >> 6;
  float lo[32 / KP][8], hi[32 / KP][8], v[8][P];
  float2 cs[32 / KP][8];
  uint32_t live = 0;   // of V's 8 slots
#pragma unroll
  for (int u = 0; u < 32 / KP; ++u) {
    const int key = u * KP + key0, r = key < 32 ? t.row(key) : -1;
    if (r >= 0) {
      const X* p = static_cast<const X*>(a.k) + (long long)r * a.ldk + t.head * D;
      load_row4(p + 8 * c, lo[u]);
      load_row4(p + D / 2 + 8 * c, hi[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[u][e] = hi[u][e] = 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = t.row(v_slot(g, e));
    if (r >= 0) {
      live |= 1u << e;
      load_row4(static_cast<const X*>(a.v) + (long long)r * a.ldv + t.head * D + v_dim, v[e]);
    } else {
#pragma unroll
      for (int x = 0; x < P; ++x) v[e][x] = 0.f;
    }
  }
  if (a.freq) {
#pragma unroll
    for (int u = 0; u < 32 / KP; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[u][e] = turned(32 * t.tile + u * KP + key0, f[e]);
  }

  if (t.page < 0) return;   // (the whole work-group)
  const int hh = t.page * a.kv_heads + t.head;   // the pool's head

  // ---- K
#pragma unroll
  for (int u = 0; u < 32 / KP; ++u) {
    const int key = u * KP + key0, slot = t.slot + key;
    const bool in = key < 32 && t.row(key) >= 0;
    rotate<D>(lo[u], hi[u], cs[u], a.freq != nullptr, a.norm);
    if constexpr (T == kBf16) {
      if (in) {
        store_row4(reinterpret_cast<__bf16*>(a.ck) + kv_k_index(hh, slot, 8 * c, size, D), lo[u]);
        store_row4(reinterpret_cast<__bf16*>(a.ck) + kv_k_index(hh, slot, D / 2 + 8 * c, size, D), hi[u]);
      }
    } else if constexpr (T == kFp8) {
      const Scale8 s = scale8(max_over_lanes<C>(fmaxf(amax8(lo[u]), amax8(hi[u]))));
      auto put = [&](int dim, const float (&x)[8]) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e] * s.inv;
        *reinterpret_cast<uint2*>(a.ck + kv_k8_index(hh, slot, dim, size, D)) =
            make_uint2(fp8_codes(y[0], y[1], y[2], y[3]), fp8_codes(y[4], y[5], y[6], y[7]));
      };
      if (in) {
        put(8 * c, lo[u]);
        put(D / 2 + 8 * c, hi[u]);
        if (c == 0) reinterpret_cast<float*>(a.ks)[size_t(hh) * size_t(size) + size_t(slot)] = s.s;
      }
    } else {
      auto put = [&](int dim, const float (&x)[8]) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max_bits(m, x[e]);
        m = over_block<2>(m);
        if (!in) return;
        if (m >= kInfBits) {
          atomicOr(not_finite, 1u << key);
          return;
        }
        const BlockScale s = block_scale(__uint_as_float(m) * a.kinv, a.kglobal, a.kinv);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = over_scale(x[e], s);
        uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, y[0], y[1], 1.f, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], 1.f, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], 1.f, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], 1.f, 3);
        *reinterpret_cast<uint32_t*>(a.ck + k4_code(hh, slot, dim, size, D).byte) = code;
        if (dim % 16 == 0) a.ks[k4_scale(hh, slot, dim, size, D)] = uint8_t(s.code);
      };
      put(8 * c, lo[u]);
      put(D / 2 + 8 * c, hi[u]);
    }
  }

  // ---- V: 8 slots of P dims
  const int slot0 = t.slot + 4 * g;   // element 0's
  if constexpr (T == kBf16) {
#pragma unroll
    for (int x = 0; x < P; ++x) {
      __bf16* to = reinterpret_cast<__bf16*>(a.cv) + kv_v_index(hh, slot0, v_dim + x, size, D);
      if (live == 0xffu) {
        const float y[8] = {v[0][x], v[1][x], v[2][x], v[3][x], v[4][x], v[5][x], v[6][x], v[7][x]};
        store_row4(to, y);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (live >> e & 1u) to[e] = (__bf16)v[e][x];
      }
    }
  } else if constexpr (T == kFp8) {
    float y[8][P];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!(live >> e & 1u)) continue;   // (the whole wave's)
      float m = 0.f;
#pragma unroll
      for (int x = 0; x < P; ++x) m = fmaxf(m, fabsf(v[e][x]));
      const Scale8 s = scale8(wave_max(m));
#pragma unroll
      for (int x = 0; x < P; ++x) y[e][x] = v[e][x] * s.inv;
      if ((tid & 63) == 0) reinterpret_cast<float*>(a.vs)[size_t(hh) * size_t(size) + size_t(t.slot + v_slot(g, e))] = s.s;
    }
#pragma unroll
    for (int x = 0; x < P; ++x) {
      uint8_t* to = a.cv + kv_v8_index(hh, slot0, v_dim + x, size, D);
      const uint32_t w0 = fp8_codes(y[0][x], y[1][x], y[2][x], y[3][x]), w1 = fp8_codes(y[4][x], y[5][x], y[6][x], y[7][x]);
      if (live == 0xffu) {
        *reinterpret_cast<uint2*>(to) = make_uint2(w0, w1);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (live >> e & 1u) to[e] = uint8_t((e < 4 ? w0 : w1) >> (8 * (e & 3)));
      }
    }
  } else {
    uint32_t keep = 0;   // nibbles of the words that are not the call's
#pragma unroll
    for (int e = 0; e < 8; ++e) keep |= live >> e & 1u ? 0u : 0xfu << (4 * e);
    uint32_t* words = reinterpret_cast<uint32_t*>(a.cv + v4_code(hh, slot0, v_dim, size, D).byte);
    uint32_t old[P], code[P] = {}, sc[8];
#pragma unroll
    for (int x = 0; x < P; ++x) old[x] = keep && live ? words[x] : 0u;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      BlockScale s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t m = 0;
#pragma unroll
        for (int x = 0; x < P; ++x) m = max_bits(m, v[e + u][x]);
        m = over_block<16 / P>(m);
        if (m >= kInfBits) atomicOr(not_finite, 1u << v_slot(g, e + u));
        s[u] = block_scale(m >= kInfBits ? 0.f : __uint_as_float(m) * a.vinv, a.vglobal, a.vinv);
        sc[e + u] = s[u].code;
      }
#pragma unroll
      for (int x = 0; x < P; ++x) {
        const float y0 = over_scale(v[e][x], s[0]), y1 = over_scale(v[e + 1][x], s[1]);
        if (e == 0) code[x] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[x], y0, y1, 1.f, 0);
        if (e == 2) code[x] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[x], y0, y1, 1.f, 1);
        if (e == 4) code[x] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[x], y0, y1, 1.f, 2);
        if (e == 6) code[x] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[x], y0, y1, 1.f, 3);
      }
    }
    uint8_t* vscales = a.vs + v4_scale(hh, slot0, v_dim, size, D);
    const bool scale_lane = v_dim % 16 == 0;
    if (live) {
#pragma unroll
      for (int x = 0; x < P; ++x) words[x] = (code[x] & ~keep) | (old[x] & keep);
      if (scale_lane) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (live >> e & 1u) vscales[e] = uint8_t(sc[e]);
      }
    }
    // a row with an infinity or a NaN in K or V gets NaN scales in both: its codes could not say it
    __syncthreads();
    const uint32_t bad = *not_finite;
    if (bad) {
#pragma unroll
      for (int u = 0; u < 32 / KP; ++u) {
        const int key = u * KP + key0;
        if (key < 32 && bad >> key & 1u)
          for (int dim : {8 * c, D / 2 + 8 * c})
            if (dim % 16 == 0) a.ks[k4_scale(hh, t.slot + key, dim, size, D)] = 0x7f;
      }
      for (int e = 0; e < 8; ++e)
        if (scale_lane && bad >> v_slot(g, e) & 1u) vscales[e] = 0x7f;
    }
  }
}

// A row's q heads: 8 + 8 dims of one a thread.
template <int D, class X>
__device__ inline void append_q(const AppendArgs& a, int row, float2* cs_lds) {
  constexpr int C = D / 16;
  const Seqs& s = a.s;
  const int chunks = a.heads * C;
  const X* rows = static_cast<const X*>(a.q) + (long long)row * a.ldq;
  float lo[8], hi[8];
  auto load = [&](int x) {
    const X* from = rows + x / C * D + x % C * 8;
    load_row4(from, lo);
    load_row4(from + D / 2, hi);
  };
  // loads go out first: the first row's and the frequencies
  double f = 0.0;
  if (a.freq && int(threadIdx.x) < D / 2) f = a.freq[threadIdx.x];
  if (int(threadIdx.x) < chunks) load(int(threadIdx.x));
  int seq = row;
  if (s.starts) {
    int n = 0;   // starts at or before the row
    for (int base = 0; base < s.n_seqs; base += 64) {
      const int x = base + (int(threadIdx.x) & 63);
      n += __popcll(__ballot(x < s.n_seqs && s.starts[x] <= row));
    }
    seq = n - 1;
    if (seq < 0) return;
  }
  const Seq q = seq_at(s, seq);
  const int at = row - q.row0;
  if (q.pos < 0 || uint32_t(at) >= uint32_t(q.n)) return;   // (the whole work-group)
  if (a.freq) {
    // (seq_at's position goes no further than a page's)
    if (int(threadIdx.x) < D / 2) cs_lds[threadIdx.x] = turned(double(uint32_t(s.pos[seq]) + uint32_t(at)), f);
    __syncthreads();
  }
  for (int x0 = 0; x0 < chunks; x0 += 256) {
    const int x = x0 + int(threadIdx.x), head = x / C, c = x % C;
    if (x >= chunks) break;   // (whole rows of lanes: chunks is a multiple of C)
    float2 cs[8];
    if (x0) load(x);
    if (a.freq) {
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] = cs_lds[8 * c + e];
    }
    rotate<D>(lo, hi, cs, a.freq != nullptr, a.norm);
    if (a.qscale) {
      float slo[8], shi[8];
      load_row4(a.qscale + head * D + 8 * c, slo);
      load_row4(a.qscale + head * D + D / 2 + 8 * c, shi);
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] *= slo[e], hi[e] *= shi[e];
    }
    X* to = static_cast<X*>(a.q_out) + (long long)row * a.ldq + head * D;
    store_row4(to + 8 * c, lo);
    store_row4(to + D / 2 + 8 * c, hi);
  }
}

template <int D, int T, class X>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs a) {
  __shared__ uint32_t not_finite;
  __shared__ float2 cs[D / 2];
  const int tiles = a.tasks * a.kv_heads;
  if (int(blockIdx.x) >= tiles) {
    append_q<D, X>(a, int(blockIdx.x) - tiles, cs);
    return;
  }
  if (T == kNvfp4) {
    if (threadIdx.x == 0) not_finite = 0;
    __syncthreads();
  }
  append_tile<D, T, X>(a, &not_finite);
}

// Tiles of a call, at most: those of a sequence of n rows are (n + 30) / 32 + 1 or fewer, and as many as it has rows.
static long long most_tiles(const Seqs& s) {
  if (!s.starts) return s.n_seqs;
  return std::min((long long)s.n_rows, (long long)s.n_rows / 32 + 2LL * s.n_seqs);
}

template <class F>
static void for_shape(int d, int type, bool bf16, F&& go) {
  auto of_row = [&](auto D, auto T) {
    if (bf16)
      go(D, T, __bf16{});
    else
      go(D, T, float{});
  };
  auto of_type = [&](auto D) {
    if (type == kBf16) of_row(D, std::integral_constant<int, kBf16>{});
    if (type == kFp8) of_row(D, std::integral_constant<int, kFp8>{});
    if (type == kNvfp4) of_row(D, std::integral_constant<int, kNvfp4>{});
  };
  if (d == 64) of_type(std::integral_constant<int, 64>{});
  if (d == 128) of_type(std::integral_constant<int, 128>{});
  if (d == 256) of_type(std::integral_constant<int, 256>{});
}

std::string launch_paged_append(const DevPaged& c, const Seqs& s, const PagedAppend& p, hipStream_t stream, bool named) {
  AppendArgs a = {};
  a.s = s;
  a.ck = static_cast<uint8_t*>(c.k), a.cv = static_cast<uint8_t*>(c.v);
  a.ks = static_cast<uint8_t*>(c.ks), a.vs = static_cast<uint8_t*>(c.vs);
  a.q = p.q, a.k = p.k, a.v = p.v, a.q_out = p.q_out;
  a.ldq = p.ldq, a.ldk = p.ldk, a.ldv = p.ldv;
  a.heads = p.heads, a.kv_heads = c.kv_heads, a.norm = p.norm;
  a.freq = p.freq, a.qscale = p.qscale;
  a.kglobal = c.kglobal, a.vglobal = c.vglobal, a.kinv = 1.f / c.kglobal, a.vinv = 1.f / c.vglobal;
  const long long tiles = most_tiles(s), groups = tiles * c.kv_heads + (p.q ? s.n_rows : 0);
  XTG_CHECK(groups < (1LL << 31), "paged_append: %d rows of %d sequences and %d KV heads", s.n_rows, s.n_seqs, c.kv_heads);
  a.tasks = int(tiles);
  const bool bf16 = p.x_dtype == kXBF16;
  for_shape(c.head_dim, c.type, bf16, [&](auto D, auto T, auto x) {
    paged_queue(&paged_append_kernel<D(), T(), decltype(x)>, dim3(unsigned(groups)), 256, 0, stream, a);
  });
  return named ? strf("paged_append_kernel<%d, %d, %s>", c.head_dim, c.type, bf16 ? "bf16" : "float") : std::string();
}

// ------------------------------------------------------------------------------------------------------- read

struct PagedReadArgs {
  Seqs s;
  const uint8_t *ck, *cv, *ks, *vs;
  void *k, *v;
  int kv_heads;
  float kglobal, vglobal;
};

// 8 E2M1 codes' values times a scale.
__device__ inline void fp4_values(uint32_t w, float s, float (&x)[8]) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
  x[0] = a[0] * s, x[1] = a[1] * s, x[2] = b[0] * s, x[3] = b[1] * s;
  x[4] = c[0] * s, x[5] = c[1] * s, x[6] = d[0] * s, x[7] = d[1] * s;
}

// Dealt as the append is: 8 + 8 dims of a key of K, P dims of 8 slots of V a thread. Every load goes out before the first
// store, whichever rows are the call's: the whole tile is there (32749 rows of 8 heads of 128 dims into BF16: NVFP4 44 us,
// FP8 45, BF16 56; with the loads behind each row's branch 47, 51 and 57).
template <int D, int T, class X>
__global__ void __launch_bounds__(256) paged_read_kernel(PagedReadArgs a) {
  constexpr int C = D / 16, KP = 256 / C < 32 ? 256 / C : 32, U = 32 / KP, P = D / 64;
  using Raw = std::conditional_t<T == kBf16, uint4, std::conditional_t<T == kFp8, uint2, uint32_t>>;   // 8 values
  TileTask t;
  if (!tile_task(a.s, a.kv_heads, int(blockIdx.x), t)) return;
  const int tid = int(threadIdx.x), size = 1 << a.s.shift;
  const bool held = t.page >= 0;
  const int hh = (held ? t.page : 0) * a.kv_heads + t.head;
  const int c = tid % C, key0 = tid / C, v_dim = (tid & 63) * P, g = tid >> 6, slot0 = t.slot + 4 * g;
  Raw k[U][2], v[P];
  float ks[U][2], vs[8];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int slot = t.slot + ((u * KP + key0) & 31), dim = x * (D / 2) + 8 * c;
      ks[u][x] = 1.f;
      if constexpr (T == kBf16) {
        k[u][x] = *reinterpret_cast<const Raw*>(reinterpret_cast<const __bf16*>(a.ck) + kv_k_index(hh, slot, dim, size, D));
      } else if constexpr (T == kFp8) {
        k[u][x] = *reinterpret_cast<const Raw*>(a.ck + kv_k8_index(hh, slot, dim, size, D));
        ks[u][x] = x ? ks[u][0] : reinterpret_cast<const float*>(a.ks)[size_t(hh) * size_t(size) + size_t(slot)];
      } else {
        k[u][x] = *reinterpret_cast<const Raw*>(a.ck + k4_code(hh, slot, dim, size, D).byte);
        ks[u][x] = __builtin_amdgcn_cvt_f32_fp8(int(a.ks[k4_scale(hh, slot, dim, size, D)]), 0) * a.kglobal;
      }
    }
#pragma unroll
  for (int x = 0; x < P; ++x) {
    if constexpr (T == kBf16)
      v[x] = *reinterpret_cast<const Raw*>(reinterpret_cast<const __bf16*>(a.cv) + kv_v_index(hh, slot0, v_dim + x, size, D));
    else if constexpr (T == kFp8)
      v[x] = *reinterpret_cast<const Raw*>(a.cv + kv_v8_index(hh, slot0, v_dim + x, size, D));
    else
      v[x] = *reinterpret_cast<const Raw*>(a.cv + v4_code(hh, slot0, v_dim + x, size, D).byte);
  }
  if constexpr (T == kFp8) {
    const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.vs) + size_t(hh) * size_t(size) + size_t(slot0));
    const float4 lo = s[0], hi = s[4];
    vs[0] = lo.x, vs[1] = lo.y, vs[2] = lo.z, vs[3] = lo.w, vs[4] = hi.x, vs[5] = hi.y, vs[6] = hi.z, vs[7] = hi.w;
  }
  if constexpr (T == kNvfp4) {
    const uint2 w = *reinterpret_cast<const uint2*>(a.vs + v4_scale(hh, slot0, v_dim, size, D));
#pragma unroll
    for (int e = 0; e < 8; ++e) vs[e] = __builtin_amdgcn_cvt_f32_fp8(int((e < 4 ? w.x : w.y) >> (8 * (e & 3)) & 0xffu), 0) * a.vglobal;
  }

  auto values = [&](const Raw& w, float s, float (&x)[8]) {
    if constexpr (T == kBf16)
      load_row4(reinterpret_cast<const __bf16*>(&w), x);
    else if constexpr (T == kFp8)
      fp8_values(w, s, x);
    else
      fp4_values(w, s, x);
  };
  auto dst = [&](void* rows, int r) {
    return static_cast<X*>(rows) + (size_t(r) * size_t(a.kv_heads) + size_t(t.head)) * D;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int key = u * KP + key0, r = key < 32 ? t.row(key) : -1;
    if (r < 0) continue;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float y[8] = {};
      if (held) values(k[u][x], ks[u][x], y);
      store_row4(dst(a.k, r) + x * (D / 2) + 8 * c, y);
    }
  }
  float y[P][8];
#pragma unroll
  for (int x = 0; x < P; ++x) values(v[x], 1.f, y[x]);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = t.row(v_slot(g, e));
    if (r < 0) continue;
    float z[P];
#pragma unroll
    for (int x = 0; x < P; ++x) z[x] = !held ? 0.f : T == kBf16 ? y[x][e] : y[x][e] * vs[e];
    store_row4(dst(a.v, r) + v_dim, z);
  }
}

std::string launch_paged_read(const DevPaged& c, const Seqs& s, void* k, void* v, bool bf16, hipStream_t stream, bool named) {
  PagedReadArgs a = {};
  a.s = s;
  a.ck = static_cast<const uint8_t*>(c.k), a.cv = static_cast<const uint8_t*>(c.v);
  a.ks = static_cast<const uint8_t*>(c.ks), a.vs = static_cast<const uint8_t*>(c.vs);
  a.k = k, a.v = v, a.kv_heads = c.kv_heads, a.kglobal = c.kglobal, a.vglobal = c.vglobal;
  const long long groups = most_tiles(s) * c.kv_heads;
  XTG_CHECK(groups < (1LL << 31), "paged_read: %d rows of %d sequences and %d KV heads", s.n_rows, s.n_seqs, c.kv_heads);
  for_shape(c.head_dim, c.type, bf16, [&](auto D, auto T, auto x) {
    paged_queue(&paged_read_kernel<D(), T(), decltype(x)>, dim3(unsigned(groups)), 256, 0, stream, a);
  });
  return named ? strf("paged_read_kernel<%d, %d, %s>", c.head_dim, c.type, bf16 ? "bf16" : "float") : std::string();
}

}  // namespace xtg::hip
