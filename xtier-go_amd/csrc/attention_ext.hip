// How an attention call with capped, biased and masked scores is cut up and queued (kernels: attention_ext_kernels.hpp,
// compiled for each head size in attention_ext_d64.hip, _d128.hip and _d256.hip).
#include <algorithm>
#include <climits>
#include <cmath>

#include "attention_ext.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace xtg::hip {

// Calls of up to this many q-cols take ext_few_kernel, which starts sooner (one launch less, no barriers) and dequantises
// a tile again for every 32 of them: over 4000 NVFP4 keys of 128 dims, 32 / 8 heads, 384 q-cols took 27.6 us (many: 44.1),
// 768 51.6 (63.6), 1024 64.4 (53.9). One number of q-cols for every length and head size: other shapes were not measured, and
// the longer the cache, the fewer q-cols it takes for the other kernel to be faster.
constexpr int kFewCols = 768;

// The plan for the cache's slots lo .. slots - 1.
static ExtPlan plan_of(const ExtCall& a, int cus, long long lo, long long slots) {
  ExtPlan p;
  const int group = a.heads / a.kv_heads;
  const long long cols = (long long)a.n_q * group;
  const int own_tiles = a.k ? (a.n_q + 31) / 32 : 0;
  p.few = cols <= kFewCols && cols * group <= 65536;
  if (p.few) {
    p.tile_lo = int(lo / 32);
    p.tiles = slots > lo ? int((slots + 31) / 32) - p.tile_lo : 0;
    // at least a tile for each wave; a work-group a CU (one and a half where blocks of q-cols share what they read); where
    // that leaves CUs idle, blocks of 16 q-cols instead of 32
    const int most = (p.tiles + kExtWaves - 1) / kExtWaves;
    p.cols = cols <= 16 || (cols <= 32 && 2 * most * a.kv_heads <= cus) ? 16 : 32;
    p.blocks = int((cols + p.cols - 1) / p.cols);
    p.splits = std::min(std::max(1, (p.blocks > 2 ? cus * 3 / 2 : cus) / (a.kv_heads * p.blocks)), most);
    if (!a.k) p.splits = std::max(p.splits, 1);
    p.own = (own_tiles + kExtWaves - 1) / kExtWaves;
    const size_t records = size_t(p.splits) + size_t(p.own);
    if (records > 1)
      p.record_bytes = records * size_t(a.kv_heads) * size_t(p.blocks * p.cols) * size_t(a.d + 2) * sizeof(float);
    return p;
  }
  p.blocks = int((cols + 127) / 128);
  p.tiles = int(slots);
  const int tk = a.d == 256 ? 32 : 64;
  const long long keys = slots - lo + (a.k ? a.n_q : 0), tiles = (keys + tk - 1) / tk;
  const long long groups = (long long)p.blocks * a.kv_heads;
  // as many as leave every work-group resident at once (two a CU), four tiles each at least
  p.splits = int(std::max(1LL, std::min(2LL * cus / groups, tiles / 4)));
  if (p.splits > 1)
    p.record_bytes = size_t(p.splits) * size_t(groups) * 128 * size_t(a.d + 2) * sizeof(float);
  if (a.k) p.pack_bytes = 2 * size_t(a.kv_heads) * size_t((a.n_q + 63) / 64 * 64) * size_t(a.d) * 2;
  return p;
}

ExtPlan ext_plan(const ExtCall& a, int cus) {
  // the slots that can hold a position which a row sees: a linear cache's are positions
  const long long all = a.cache ? a.cache->slots : 0;
  long long slots = all, lo = 0;
  if (a.cache) {
    const long long past = a.k ? a.pos0 : a.end ? slots : a.pos0 + a.n_q;
    if (!a.cache->ring || a.k) slots = std::min(slots, past);   // (a ring fills from its first slot on)
    if (!a.cache->ring && a.window > 0) lo = std::max(0LL, std::min(slots, a.pos0 - a.window + 1));
  }
  ExtPlan p = plan_of(a, cus, lo, slots);
  // Records grow with the slots until the splits fill the CUs. Scratch is what the whole cache takes, so that later
  // positions of a decode loop, or of a graph captured after an early call, never ask for more.
  p.scratch = plan_of(a, cus, 0, all).used_bytes();
  return p;
}

void launch_attn_ext(const ExtCall& c, const ExtPlan& p, void* scratch, hipStream_t stream, const Timed& timed) {
  ExtArgs a = {};
  a.q = c.q, a.k = c.k, a.v = c.v, a.out = c.out;
  if (const DevKv* kv = c.cache) {
    a.ck = static_cast<const uint8_t*>(kv->k);
    a.cv = static_cast<const uint8_t*>(kv->v);
    a.ks = kv->kscale, a.vs = kv->vscale, a.slot_pos = kv->slot_pos;
    a.slots_pad = kv->slots_pad, a.ring = kv->ring;
    a.kglobal = kv->kglobal, a.vglobal = kv->vglobal;
  }
  a.tile_lo = p.tile_lo, a.tiles = p.tiles, a.splits = p.splits, a.cols = p.cols;
  a.own = c.k ? c.n_q : 0;
  a.records = p.splits + p.own;
  a.n_q = c.n_q, a.pos0 = int(c.pos0), a.heads = c.heads, a.group = c.heads / c.kv_heads, a.window = c.window;
  a.group_inv = (65536u + uint32_t(a.group) - 1u) / uint32_t(a.group);
  a.bf16 = c.x_dtype == kXBF16;
  a.cached_end = c.k ? a.pos0 : INT_MAX;
  const double log2e = kLog2e;
  a.factor = float(std::frexp(std::fabs(double(c.scale)) * (c.softcap > 0.f ? 2 * log2e / c.softcap : log2e), &a.factor_exp));
  a.scale = c.scale, a.softcap = c.softcap, a.slopes = c.slopes, a.first = c.first, a.end = c.end;
  char* at = static_cast<char*>(scratch);
  a.pk = reinterpret_cast<const uint4*>(at);
  a.pv = reinterpret_cast<const uint4*>(at + p.pack_bytes / 2);
  a.acc = reinterpret_cast<float*>(at + p.pack_bytes);
  a.ml = a.acc + p.record_bytes / sizeof(float) / size_t(c.d + 2) * size_t(c.d);
  const int dtype = c.cache ? c.cache->dtype() : kBf16;
  if (c.d == 64)
    ext_launch<64>(c, p, a, dtype, stream, timed);
  else if (c.d == 128)
    ext_launch<128>(c, p, a, dtype, stream, timed);
  else if (c.d == 256)
    ext_launch<256>(c, p, a, dtype, stream, timed);
  else
    fail("attention_ext: head_dim %d", c.d);
}

}  // namespace xtg::hip
