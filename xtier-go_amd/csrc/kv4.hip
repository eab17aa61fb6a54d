// Rows into an NVFP4 cache, and rows of any cache back (layouts: kv4.hpp and attention.hip).
//
// Both are bound by HBM for many rows, and by latency for few: 64 to 256 threads take a (KV head, 32-slot tile), so that
// a decoded token's rows are one step of a few loads in each. Of K a thread takes a few dims of a key, rows read as they
// lie; of V a few dims of 8 keys, so that it reads and writes whole words of codes. A ring's last rows and first rows can
// share a tile, which is still one work-group's in a store, since a V word holds the codes of 8 slots and the nibbles of
// other rows stay. 32749 BF16 rows of 8 heads of 128 dims written and then read: 82 us for 344 MB, 4.2 TB/s (a copy of
// 4 GB reaches 4.7); one row 9.5, which is the two calls' queueing.
#include <algorithm>

#include "attention_ext.hpp"
#include "common.hpp"
#include "kv4.hpp"
#include "kv_rows.hpp"

namespace xtg::hip {

// Threads of a (head, tile), dims of K that one takes at a time, keys of a pass over K, and its dims of V. The store's
// threads take more, which spreads what a block's scale costs.
template <int D, bool STORE>
struct Deal4 {
  static constexpr int NT = (D == 64 ? 128 : 256) / (STORE ? 2 : 1), KD = STORE ? 8 : 4, KP = NT * KD / D, P = 4 * D / NT;
};

struct Store4Args {
  const void* k;
  const void* v;
  uint8_t* ck;
  uint8_t* cv;
  uint8_t* ks;
  uint8_t* vs;
  int* slot_pos;
  long long pos;          // position of the first row stored (row `first` of the call)
  int first, rows;        // rows first .. first + rows - 1 of the call are stored
  int kv_heads, slots, slots_pad;
  int slot0, t0, tiles, total_tiles;   // the first row's slot, its tile, the tiles to visit and the cache's
  float kglobal, vglobal, kinv, vinv;   // and their inverses, exact
};

// A row that holds an infinity or a NaN in K or V gets NaN scales for both, whose E2M1 codes could not say it: queries
// that see the position get NaN, and no other (the attention takes V scales that are NaN as zero, and masks scores).
// full: the tile's 32 slots are rows r0 .. r0 + 31, and nothing has to be asked of each.
template <int D, class X, bool FULL>
__device__ inline void store4_tile(const Store4Args& a, uint32_t* not_finite, int h, int t, bool in, int r0) {
  using Deal = Deal4<D, true>;
  constexpr int NT = Deal::NT, KD = Deal::KD, KP = Deal::KP, P = Deal::P;
  const int sub = int(threadIdx.x) / NT, tid = int(threadIdx.x) % NT;
  // the row (counted from the first stored) whose position slot s takes, or -1
  auto row_of = [&](int s) {
    if (FULL) return r0 + s - 32 * t;
    const int d = s - a.slot0 + (s < a.slot0 ? a.slots : 0);
    return in && s < a.slots && d < a.rows ? d : -1;
  };
  auto src = [&](const void* rows, int r) {
    return static_cast<const X*>(rows) + (size_t(a.first + r) * size_t(a.kv_heads) + size_t(h)) * D;
  };
  const int k_dim = tid % (D / KD) * KD, k_key = tid / (D / KD);     // 8 dims of keys k_key, k_key + KP, ..
  const int v_dim = tid % (D / P) * P, g = tid / (D / P);            // P dims of slots 4 g + .., 16 + 4 g + ..
  float k[32 / KP][KD], v[8][P];
#pragma unroll
  for (int u = 0; u < 32 / KP; ++u) {
    const int r = row_of(32 * t + u * KP + k_key);
    if (FULL || r >= 0) {
      load_row4(src(a.k, r) + k_dim, k[u]);
    } else {
#pragma unroll
      for (int c = 0; c < KD; ++c) k[u][c] = 0.f;
    }
  }
  uint32_t keep = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = row_of(32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e));
    if (FULL || r >= 0) {
      load_row4(src(a.v, r) + v_dim, v[e]);
    } else {
      keep |= 0xfu << (4 * e);
#pragma unroll
      for (int c = 0; c < P; ++c) v[e][c] = 0.f;
    }
  }
  uint32_t old[P] = {};   // the words' other nibbles
  uint32_t* words = reinterpret_cast<uint32_t*>(a.cv + v4_code(h, 32 * t + 4 * g, v_dim, a.slots_pad, D).byte);
  if (keep && keep != 0xffffffffu) {
#pragma unroll
    for (int c = 0; c < P; ++c) old[c] = words[c / 4 * 256 + c % 4];   // groups of 4 are 1 KiB apart
  }
#pragma unroll
  for (int u = 0; u < 32 / KP; ++u) {
    const int key = u * KP + k_key;
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < KD; ++c) m = max_bits(m, k[u][c]);
    m = over_block<16 / KD>(m);
    if (!FULL && row_of(32 * t + key) < 0) continue;
    if (m >= kInfBits) {
      atomicOr(&not_finite[sub], 1u << key);
      continue;
    }
    const BlockScale s = block_scale(__uint_as_float(m) * a.kinv, a.kglobal, a.kinv);
    float y[KD];
#pragma unroll
    for (int c = 0; c < KD; ++c) y[c] = over_scale(k[u][c], s);
    uint32_t code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, y[0], y[1], 1.f, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], 1.f, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], 1.f, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], 1.f, 3);
    *reinterpret_cast<uint32_t*>(a.ck + k4_code(h, 32 * t + key, k_dim, a.slots_pad, D).byte) = code;
    if (k_dim % 16 == 0) a.ks[k4_scale(h, 32 * t + key, k_dim, a.slots_pad, D)] = uint8_t(s.code);
  }

  uint8_t* vscales = a.vs + v4_scale(h, 32 * t + 4 * g, v_dim, a.slots_pad, D);
  const bool scale_lane = v_dim % 16 == 0;
  uint32_t code[P] = {}, sc[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    BlockScale s[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t m = 0;
#pragma unroll
      for (int c = 0; c < P; ++c) m = max_bits(m, v[e + x][c]);
      m = over_block<16 / P>(m);
      if (m >= kInfBits) atomicOr(&not_finite[sub], 1u << (e + x < 4 ? 4 * g + e + x : 12 + 4 * g + e + x));
      s[x] = block_scale(m >= kInfBits ? 0.f : __uint_as_float(m) * a.vinv, a.vglobal, a.vinv);
      sc[e >> 2] |= s[x].code << (8 * ((e + x) & 3));
    }
#pragma unroll
    for (int c = 0; c < P; ++c) {
      const float y0 = over_scale(v[e][c], s[0]), y1 = over_scale(v[e + 1][c], s[1]);
      if (e == 0) code[c] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[c], y0, y1, 1.f, 0);
      if (e == 2) code[c] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[c], y0, y1, 1.f, 1);
      if (e == 4) code[c] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[c], y0, y1, 1.f, 2);
      if (e == 6) code[c] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code[c], y0, y1, 1.f, 3);
    }
  }
  if (keep != 0xffffffffu) {
#pragma unroll
    for (int c = 0; c < P; ++c) words[c / 4 * 256 + c % 4] = (code[c] & ~keep) | (old[c] & keep);
    if (scale_lane && keep == 0) {
      *reinterpret_cast<uint2*>(vscales) = make_uint2(sc[0], sc[1]);
    } else if (scale_lane) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(keep >> (4 * e) & 1u)) vscales[e] = uint8_t(sc[e >> 2] >> (8 * (e & 3)));
    }
  }
  if (h == 0 && tid < 32) {
    const int r = row_of(32 * t + tid);
    if (FULL || r >= 0) a.slot_pos[32 * t + tid] = int(a.pos + r);
  }

  __syncthreads();
  const uint32_t bad = not_finite[sub];
  if (bad == 0) return;
  for (int u = 0; u < 32 / KP; ++u) {
    const int key = u * KP + k_key;
    if (k_dim % 16 == 0 && bad >> key & 1u) a.ks[k4_scale(h, 32 * t + key, k_dim, a.slots_pad, D)] = 0x7f;
  }
  for (int e = 0; e < 8; ++e)
    if (scale_lane && bad >> (e < 4 ? 4 * g + e : 12 + 4 * g + e) & 1u) vscales[e] = 0x7f;
}

template <int D, class X>
__global__ void __launch_bounds__(256) kv_store4_kernel(Store4Args a) {
  constexpr int NT = Deal4<D, true>::NT;
  __shared__ uint32_t not_finite[256 / NT];   // a tile's slots
  const int w = int(blockIdx.x) * (256 / NT) + int(threadIdx.x) / NT;
  const bool in = w < a.tiles * a.kv_heads;   // (threads past the end wait for the others)
  const int h = w % a.kv_heads, t = in ? (a.t0 + w / a.kv_heads) % a.total_tiles : 0;
  if (threadIdx.x < 256 / NT) not_finite[threadIdx.x] = 0;
  const int r0 = 32 * t - a.slot0 + (32 * t < a.slot0 ? a.slots : 0);
  const bool full = in && 32 * t + 32 <= a.slots && r0 + 32 <= a.rows && (32 * t >= a.slot0 || 32 * t + 32 <= a.slot0);
  if (__syncthreads_and(full))
    store4_tile<D, X, true>(a, not_finite, h, t, in, r0);
  else
    store4_tile<D, X, false>(a, not_finite, h, t, in, r0);
}

std::string launch_kv_store4(const DevKv& c, long long pos, int first, int n, const void* k, const void* v, bool bf16,
                             hipStream_t stream) {
  Store4Args a;
  a.k = k;
  a.v = v;
  a.ck = static_cast<uint8_t*>(c.k);
  a.cv = static_cast<uint8_t*>(c.v);
  a.ks = reinterpret_cast<uint8_t*>(c.kscale);
  a.vs = reinterpret_cast<uint8_t*>(c.vscale);
  a.slot_pos = c.slot_pos;
  a.pos = pos + first;
  a.first = first;
  a.rows = n - first;
  a.kv_heads = c.kv_heads;
  a.slots = int(c.slots);
  a.slots_pad = c.slots_pad;
  a.slot0 = int(c.ring ? a.pos % c.slots : a.pos);
  a.t0 = a.slot0 / 32;
  a.total_tiles = c.slots_pad / 32;
  // to the end of the ring, and from its beginning: at most every tile once
  const int to_end = std::min(a.rows, a.slots - a.slot0);
  const int tiles = (a.slot0 + to_end - 1) / 32 - a.t0 + 1 + (a.rows - to_end + 31) / 32;
  a.tiles = std::min(tiles, a.total_tiles);
  a.kglobal = c.kglobal;
  a.vglobal = c.vglobal;
  a.kinv = 1.f / c.kglobal;
  a.vinv = 1.f / c.vglobal;
  XTG_CHECK(a.tiles * (long long)c.kv_heads < (1LL << 31), "kv_store: %d rows of %d KV heads", n, c.kv_heads);
  const int per = c.head_dim == 64 ? 4 : 2;   // (head, tile)s of a work-group
  const dim3 grid{unsigned((a.tiles * (long long)c.kv_heads + per - 1) / per)}, block{256};
#define XTG_STORE4(D)                                                                              \
  if (c.head_dim == D) {                                                                           \
    if (bf16)                                                                                      \
      hipLaunchKernelGGL((kv_store4_kernel<D, __bf16>), grid, block, 0, stream, a);                \
    else                                                                                           \
      hipLaunchKernelGGL((kv_store4_kernel<D, float>), grid, block, 0, stream, a);                 \
  }
  XTG_STORE4(64) XTG_STORE4(128) XTG_STORE4(256)
#undef XTG_STORE4
  HIP_CHECK(hipGetLastError());
  return strf("kv_store4_kernel<%d, %s>", c.head_dim, bf16 ? "bf16" : "float");
}

// ------------------------------------------------------------------------------------------------------- read

struct ReadArgs {
  const uint8_t* ck;
  const uint8_t* cv;
  const void* ks;
  const void* vs;
  const int* slot_pos;
  void* k;
  void* v;
  long long pos, base;        // first row's position; the position that slot 0 of the first lap would have
  int n, kv_heads, slots, slots_pad;
  int t0, tiles, total_tiles;   // first tile, tiles to visit (laps of a ring counted again), the cache's tiles
  float kglobal, vglobal;
};

// Every row of the call is one work-group's to write, zeros included: a tile is visited once for every lap of the ring
// that the rows take. NVFP4 is dealt as the store deals it; BF16 and FP8 by 16-byte words, a wave a tile.
template <int D, int T, class X>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadArgs a) {
  constexpr int NT = T == kNvfp4 ? Deal4<D, false>::NT : 64;
  const int w = int(blockIdx.x) * (256 / NT) + int(threadIdx.x) / NT;
  if (w >= a.tiles * a.kv_heads) return;
  const int h = w % a.kv_heads, u = a.t0 + w / a.kv_heads, lap = u / a.total_tiles, t = u % a.total_tiles;
  const long long p0 = a.base + (long long)lap * a.slots;   // slot s holds position p0 + s in this lap
  auto row_of = [&](int s) {
    const long long r = p0 + s - a.pos;
    return s < a.slots && r >= 0 && r < a.n ? int(r) : -1;
  };
  auto dst = [&](void* rows, int r) {
    return static_cast<X*>(rows) + (size_t(r) * size_t(a.kv_heads) + size_t(h)) * D;
  };
  const size_t head = size_t(h) * size_t(a.slots_pad);

  if constexpr (T == kNvfp4) {
    constexpr int KP = Deal4<D, false>::KP, P = Deal4<D, false>::P;
    const int tid = int(threadIdx.x) % NT;
    const int k_dim = tid % (D / 4) * 4, k_key = tid / (D / 4), v_dim = tid % (D / P) * P, g = tid / (D / P);
    uint32_t kc[32 / KP], word[P];
    float ks[32 / KP];
    const uint2 vs = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.vs) +
                                                     v4_scale(h, 32 * t + 4 * g, v_dim, a.slots_pad, D));
#pragma unroll
    for (int u = 0; u < 32 / KP; ++u) {
      const int slot = 32 * t + u * KP + k_key;
      kc[u] = *reinterpret_cast<const uint16_t*>(a.ck + k4_code(h, slot, k_dim, a.slots_pad, D).byte);
      const int sc = static_cast<const uint8_t*>(a.ks)[k4_scale(h, slot, k_dim, a.slots_pad, D)];
      ks[u] = a.slot_pos[slot] == int(p0 + slot) ? __builtin_amdgcn_cvt_f32_fp8(sc, 0) * a.kglobal : 0.f;
    }
    const uint32_t* words = reinterpret_cast<const uint32_t*>(a.cv + v4_code(h, 32 * t + 4 * g, v_dim, a.slots_pad, D).byte);
#pragma unroll
    for (int c = 0; c < P; ++c) word[c] = words[c];
#pragma unroll
    for (int u = 0; u < 32 / KP; ++u) {
      const int r = row_of(32 * t + u * KP + k_key);
      if (r < 0) continue;
      const auto x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(kc[u], 1.f, 0), y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(kc[u], 1.f, 1);
      const float out[4] = {x[0] * ks[u], x[1] * ks[u], y[0] * ks[u], y[1] * ks[u]};
      store_row4(dst(a.k, r) + k_dim, out);
    }
    const int4 at0 = *reinterpret_cast<const int4*>(a.slot_pos + 32 * t + 4 * g);
    const int4 at1 = *reinterpret_cast<const int4*>(a.slot_pos + 32 * t + 16 + 4 * g);
    const int at[8] = {at0.x, at0.y, at0.z, at0.w, at1.x, at1.y, at1.z, at1.w};
    float val[P][8];
#pragma unroll
    for (int c = 0; c < P; ++c) {
      const auto e0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[c], 1.f, 0), e2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[c], 1.f, 1);
      const auto e4 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[c], 1.f, 2), e6 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word[c], 1.f, 3);
      val[c][0] = e0[0], val[c][1] = e0[1], val[c][2] = e2[0], val[c][3] = e2[1];
      val[c][4] = e4[0], val[c][5] = e4[1], val[c][6] = e6[0], val[c][7] = e6[1];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int slot = 32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e), r = row_of(slot);
      if (r < 0) continue;
      const int sc = int((e < 4 ? vs.x : vs.y) >> (8 * (e & 3)) & 0xffu);
      const float s = at[e] == int(p0 + slot) ? __builtin_amdgcn_cvt_f32_fp8(sc, 0) * a.vglobal : 0.f;
      float out[P];
#pragma unroll
      for (int c = 0; c < P; ++c) out[c] = val[c][e] * s;
      store_row4(dst(a.v, r) + v_dim, out);
    }
  } else {
    // K: 8 consecutive dims of slot i of a block are a lane's; V: one dim of 8 slots
    constexpr int ND = D / 16;
    const int lane = int(threadIdx.x) & 63, g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int slot = 32 * t + 16 * b + i, r = row_of(slot);
      if (r < 0) continue;
      const bool held = a.slot_pos[slot] == int(p0 + slot);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float x[8] = {};
        if (held && T == kBf16) {
          load_row4(reinterpret_cast<const __bf16*>(a.ck) + kv_k_index(h, slot, 32 * c + 8 * g, a.slots_pad, D), x);
        } else if (held) {
          const uint2 wd = *reinterpret_cast<const uint2*>(a.ck + kv_k8_index(h, slot, 32 * c + 8 * g, a.slots_pad, D));
          const float s = static_cast<const float*>(a.ks)[head + size_t(slot)];
          fp8_values(wd, s, x);
        }
        store_row4(dst(a.k, r) + 32 * c + 8 * g, x);
      }
    }
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) {
      float x[8];
      const int slot0 = 32 * t + 4 * g;
      if constexpr (T == kBf16) {
        load_row4(reinterpret_cast<const __bf16*>(a.cv) + kv_v_index(h, slot0, 16 * dd + i, a.slots_pad, D), x);
      } else {
        fp8_values(*reinterpret_cast<const uint2*>(a.cv + kv_v8_index(h, slot0, 16 * dd + i, a.slots_pad, D)), 1.f, x);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int slot = 32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e), r = row_of(slot);
        if (r < 0) continue;
        const bool held = a.slot_pos[slot] == int(p0 + slot);
        float y = held ? x[e] : 0.f;
        if (T == kFp8 && held) y *= static_cast<const float*>(a.vs)[head + size_t(slot)];   // (infinite: zeros are NaN)
        dst(a.v, r)[16 * dd + i] = X(y);
      }
    }
  }
}

std::string launch_kv_read(const DevKv& c, long long pos, int n, void* k, void* v, bool bf16, hipStream_t stream) {
  ReadArgs a;
  a.ck = static_cast<const uint8_t*>(c.k);
  a.cv = static_cast<const uint8_t*>(c.v);
  a.ks = c.kscale;
  a.vs = c.vscale;
  a.slot_pos = c.slot_pos;
  a.k = k;
  a.v = v;
  a.pos = pos;
  a.n = n;
  a.kv_heads = c.kv_heads;
  a.slots = int(c.slots);
  a.slots_pad = c.slots_pad;
  const long long slot0 = c.ring ? pos % c.slots : pos, last = slot0 + n - 1;
  a.base = pos - slot0;
  a.t0 = int(slot0 / 32);
  a.total_tiles = c.slots_pad / 32;
  const long long tiles = last / c.slots * a.total_tiles + last % c.slots / 32 - a.t0 + 1;
  XTG_CHECK(tiles * c.kv_heads < (1LL << 31), "kv_read: %d rows of %d KV heads", n, c.kv_heads);
  a.tiles = int(tiles);
  a.kglobal = c.kglobal;
  a.vglobal = c.vglobal;
  const int per = !c.fp4 ? 4 : c.head_dim == 64 ? 2 : 1;   // (head, tile)s of a work-group
  const dim3 grid{unsigned((tiles * c.kv_heads + per - 1) / per)}, block{256};
#define XTG_READ(D, T)                                                                    \
  if (c.head_dim == D && c.dtype() == T) {                                                \
    if (bf16)                                                                             \
      hipLaunchKernelGGL((kv_read_kernel<D, T, __bf16>), grid, block, 0, stream, a);      \
    else                                                                                  \
      hipLaunchKernelGGL((kv_read_kernel<D, T, float>), grid, block, 0, stream, a);       \
  }
  XTG_READ(64, 0) XTG_READ(64, 1) XTG_READ(64, 2) XTG_READ(128, 0) XTG_READ(128, 1) XTG_READ(128, 2)
  XTG_READ(256, 0) XTG_READ(256, 1) XTG_READ(256, 2)
#undef XTG_READ
  HIP_CHECK(hipGetLastError());
  return strf("kv_read_kernel<%d, %d, %s>", c.head_dim, c.dtype(), bf16 ? "bf16" : "float");
}

}  // namespace xtg::hip
