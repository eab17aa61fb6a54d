// Rows into an NVFP4 cache, and rows of any cache back (layouts: kv4.hpp and attention.hip).
//
// Both take one wave per (KV head, 32-slot tile): a wave's lanes hold the tile as the cache's operand layout deals it,
// so a lane reads and writes whole words. Of a call's rows a tile's slots hold the ones at their positions; a ring's
// last rows and first rows can share a tile, which is still one wave's in a store, since a V word holds the codes of
// 8 slots and the wave rewrites the nibbles of the call's rows only.
#include <algorithm>

#include "attention.hpp"
#include "common.hpp"
#include "kv4.hpp"

namespace xtg::hip {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves4 = 4;   // waves per work-group

// N consecutive elements of a row as FP32 (N a multiple of 4, aligned to 4 elements).
template <int N>
__device__ inline void load_row4(const float* p, float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const float4 a = *reinterpret_cast<const float4*>(p + e);
    x[e] = a.x, x[e + 1] = a.y, x[e + 2] = a.z, x[e + 3] = a.w;
  }
}
template <int N>
__device__ inline void load_row4(const __bf16* p, float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const uint2 a = *reinterpret_cast<const uint2*>(p + e);
    x[e] = __uint_as_float(a.x << 16), x[e + 1] = __uint_as_float(a.x & 0xffff0000u);
    x[e + 2] = __uint_as_float(a.y << 16), x[e + 3] = __uint_as_float(a.y & 0xffff0000u);
  }
}

template <int N>
__device__ inline void store_row4(float* p, const float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
}
// Rounded to nearest even (an FP8 row's values; NVFP4 and BF16 rows' are exact).
template <int N>
__device__ inline void store_row4(__bf16* p, const float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    __bf16 b[4] = {(__bf16)x[e], (__bf16)x[e + 1], (__bf16)x[e + 2], (__bf16)x[e + 3]};
    *reinterpret_cast<uint2*>(p + e) = __builtin_bit_cast(uint2, *reinterpret_cast<const uint64_t*>(b));
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
template <int D, class X>
__global__ void __launch_bounds__(kWaves4 * 64) kv_store4_kernel(Store4Args a) {
  constexpr int ND = D / 16, CH = D < 128 ? D : 128, LD = CH / 4, NCH = D / CH;
  const int w = int(blockIdx.x) * kWaves4 + int(threadIdx.x >> 6);
  if (w >= a.tiles * a.kv_heads) return;   // whole waves
  const int h = w % a.kv_heads, t = (a.t0 + w / a.kv_heads) % a.total_tiles;
  const int lane = int(threadIdx.x) & 63, g = lane >> 4, i = lane & 15;
  // the row (counted from the first stored) whose position slot s takes, or -1
  auto row_of = [&](int s) {
    const int d = s - a.slot0 + (s < a.slot0 ? a.slots : 0);
    return s < a.slots && d < a.rows ? d : -1;
  };
  auto src = [&](const void* rows, int r) {
    return static_cast<const X*>(rows) + (size_t(a.first + r) * size_t(a.kv_heads) + size_t(h)) * D;
  };

  // V: the lane's ND dims of 8 slots
  uint32_t* words = reinterpret_cast<uint32_t*>(a.cv + v4_code(h, 32 * t, 0, a.slots_pad, D).byte) + lane * 4;
  uint8_t* vscales = a.vs + v4_scale(h, 32 * t + 4 * g, i * ND, a.slots_pad, D);
  const bool scale_lane = (i * ND) % 16 == 0;   // of the lanes that share a block, the one that writes its scales
  uint32_t code[ND], keep = 0, vbad = 0, vrows = 0;
#pragma unroll
  for (int dd = 0; dd < ND; ++dd) code[dd] = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = row_of(32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e));
    if (r < 0) keep |= 0xfu << (4 * e);
    float x[ND] = {};
    if (r >= 0) load_row4(src(a.v, r) + i * ND, x);
    uint32_t m = 0;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) m = max_bits(m, x[dd]);
    if constexpr (ND < 16) m = dpp_max<kDppXor1>(m);   // the block's other lanes
    if constexpr (ND < 8) m = dpp_max<kDppXor2>(m);
    const bool bad = m >= kInfBits;
    const uint32_t sc = bad ? 0u : block_scale_code(__uint_as_float(m) * a.vinv);
    const float s = e4m3_scale_value(uint8_t(sc)) * a.vglobal;
    vbad |= bad ? 1u << e : 0u;
    vrows |= r >= 0 ? 1u << e : 0u;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) code[dd] |= e2m1_code(x[dd], s) << (4 * e);
    if (r >= 0 && scale_lane) vscales[e] = uint8_t(sc);
  }
#pragma unroll
  for (int q = 0; q < ND / 4; ++q) {
    uint4* at = reinterpret_cast<uint4*>(words + q * 256);
    uint4 n = make_uint4(code[4 * q], code[4 * q + 1], code[4 * q + 2], code[4 * q + 3]);
    if (keep == 0xffffffffu) continue;
    if (keep) {
      const uint4 o = *at;
      n.x |= o.x & keep, n.y |= o.y & keep, n.z |= o.z & keep, n.w |= o.w & keep;
    }
    *at = n;
  }

  // K: LD dims of a chunk of slot i of each 16-slot block
  uint32_t kbad = 0;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int slot = 32 * t + 16 * b + i, r = row_of(slot);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (r < 0) continue;
      const int dim = c * CH + g * LD;
      float x[LD];
      load_row4(src(a.k, r) + dim, x);
      uint8_t* out = a.ck + k4_code(h, slot, dim, a.slots_pad, D).byte;
      uint8_t* scales = a.ks + k4_scale(h, slot, dim, a.slots_pad, D);
#pragma unroll
      for (int j = 0; j < LD / 16; ++j) {
        uint32_t m = 0, word[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e) m = max_bits(m, x[16 * j + e]);
        const bool bad = m >= kInfBits;
        const uint32_t sc = bad ? 0u : block_scale_code(__uint_as_float(m) * a.kinv);
        const float s = e4m3_scale_value(uint8_t(sc)) * a.kglobal;
        kbad |= bad ? 1u << b : 0u;
#pragma unroll
        for (int e = 0; e < 16; ++e) word[e >> 3] |= e2m1_code(x[16 * j + e], s) << (4 * (e & 7));
        *reinterpret_cast<uint2*>(out + 8 * j) = make_uint2(word[0], word[1]);
        scales[j] = uint8_t(sc);
      }
    }
  }
  if (h == 0 && lane < 32) {
    const int slot = 32 * t + lane, r = row_of(slot);
    if (r >= 0) a.slot_pos[slot] = int(a.pos + r);
  }

  if (__ballot(vbad | kbad) == 0) return;
  // slots that are not finite, over all lanes: bit b of a K lane's slot 16 b + i, bit e of a V lane's 8 slots
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) vbad |= uint32_t(__shfl_xor(int(vbad), x));
  kbad |= uint32_t(__shfl_xor(int(kbad), 16));
  kbad |= uint32_t(__shfl_xor(int(kbad), 32));
  const uint32_t of_v = uint32_t(__shfl(int(vbad), (i >> 2) * 16));
#pragma unroll
  for (int e = 0; e < 8; ++e)
    vbad |= ((uint32_t(__shfl(int(kbad), 4 * g + (e & 3))) >> (e >> 2)) & 1u) << e;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int slot = 32 * t + 16 * b + i;
    if (row_of(slot) < 0 || !((kbad >> b | of_v >> (4 * b + (i & 3))) & 1u)) continue;
    for (int c = 0; c < NCH; ++c)
      for (int j = 0; j < LD / 16; ++j)
        a.ks[k4_scale(h, slot, c * CH + g * LD + 16 * j, a.slots_pad, D)] = 0x7f;
  }
  for (int e = 0; e < 8; ++e)
    if (scale_lane && (vbad & vrows) >> e & 1u) vscales[e] = 0x7f;
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
  const dim3 grid{unsigned((a.tiles * (long long)c.kv_heads + kWaves4 - 1) / kWaves4)}, block{kWaves4 * 64};
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

constexpr int kBf16 = 0, kFp8 = 1, kNvfp4 = 2;   // XTG_KV_*

// Every row of the call is one wave's to write, zeros included: a tile is visited once for every lap of the ring that
// the rows take.
template <int D, int T, class X>
__global__ void __launch_bounds__(kWaves4 * 64) kv_read_kernel(ReadArgs a) {
  constexpr int ND = D / 16;
  const int w = int(blockIdx.x) * kWaves4 + int(threadIdx.x >> 6);
  if (w >= a.tiles * a.kv_heads) return;
  const int h = w % a.kv_heads, u = a.t0 + w / a.kv_heads, lap = u / a.total_tiles, t = u % a.total_tiles;
  const int lane = int(threadIdx.x) & 63, g = lane >> 4, i = lane & 15;
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
    constexpr int CH = D < 128 ? D : 128, LD = CH / 4, NCH = D / CH;
    uint32_t word[ND];
    const uint4* words = reinterpret_cast<const uint4*>(a.cv + v4_code(h, 32 * t, 0, a.slots_pad, D).byte);
#pragma unroll
    for (int q = 0; q < ND / 4; ++q) {
      const uint4 x = words[q * 64 + lane];
      word[4 * q] = x.x, word[4 * q + 1] = x.y, word[4 * q + 2] = x.z, word[4 * q + 3] = x.w;
    }
    const uint8_t* vscales =
        static_cast<const uint8_t*>(a.vs) + v4_scale(h, 32 * t + 4 * g, i * ND, a.slots_pad, D);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int slot = 32 * t + (e < 4 ? 4 * g + e : 12 + 4 * g + e), r = row_of(slot);
      if (r < 0) continue;
      float x[ND] = {};
      if (a.slot_pos[slot] == int(p0 + slot)) {
        const float s = e4m3_scale_value(vscales[e]) * a.vglobal;
#pragma unroll
        for (int dd = 0; dd < ND; ++dd) x[dd] = e2m1_value(int(word[dd] >> (4 * e) & 15u)) * s;
      }
      store_row4(dst(a.v, r) + i * ND, x);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int slot = 32 * t + 16 * b + i, r = row_of(slot);
      if (r < 0) continue;
      const bool held = a.slot_pos[slot] == int(p0 + slot);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int dim = c * CH + g * LD;
        const uint8_t* in = a.ck + k4_code(h, slot, dim, a.slots_pad, D).byte;
        const uint8_t* scales = static_cast<const uint8_t*>(a.ks) + k4_scale(h, slot, dim, a.slots_pad, D);
#pragma unroll
        for (int j = 0; j < LD / 16; ++j) {
          float x[16] = {};
          if (held) {
            const uint2 wd = *reinterpret_cast<const uint2*>(in + 8 * j);
            const float s = e4m3_scale_value(scales[j]) * a.kglobal;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = e2m1_value(int((e < 8 ? wd.x : wd.y) >> (4 * (e & 7)) & 15u)) * s;
          }
          store_row4(dst(a.k, r) + dim + 16 * j, x);
        }
      }
    }
  } else {
    // K: 8 consecutive dims of slot i of a block are a lane's; V: one dim of 8 slots
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
        float y = a.slot_pos[slot] == int(p0 + slot) ? x[e] : 0.f;
        if (T == kFp8 && y != 0.f) y *= static_cast<const float*>(a.vs)[head + size_t(slot)];
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
  const dim3 grid{unsigned((tiles * c.kv_heads + kWaves4 - 1) / kWaves4)}, block{kWaves4 * 64};
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
