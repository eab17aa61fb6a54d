// Attention with capped, biased and masked scores over a cache of any dtype (plan: attention_ext.hip; kernels:
// attention_ext_kernels.hpp).
#pragma once

#include <hip/hip_runtime.h>

#include <functional>
#include <string>

#include "attention.hpp"

namespace xtg::hip {

// One call (the fields of xtg_attn_ext).
struct ExtCall {
  const DevKv* cache;
  int n_q;
  long long pos0;
  int heads, kv_heads, d, window;
  float scale;
  const void *q, *k, *v;
  void* out;
  int x_dtype;
  float softcap;
  const float* slopes;
  const int* first;
  const int* end;
};

// How a call is cut up. A q-col is a (row, q head of a KV head); a work-group takes `cols` of them for one KV head and
// one of `splits` parts of the keys, and leaves a record (accumulator, maximum, sum) for each where there are more
// than one. few: the work-groups' waves take cache tiles of their own, and `own` work-groups more the call's own keys.
// Otherwise blocks of 128 q-cols share tiles, the call's own keys packed as tiles too.
struct ExtPlan {
  bool few = false;
  int cols = 128, blocks = 1, splits = 1, own = 0;
  int tile_lo = 0, tiles = 0;    // few: the cache's 32-slot tiles to scan; else tile_lo = 0 and the slots to scan
  size_t pack_bytes = 0;         // own keys and values as BF16 tiles
  size_t record_bytes = 0;
  size_t used_bytes() const { return pack_bytes + record_bytes; }
  size_t scratch = 0;            // used_bytes() at most, whatever the call's positions and window
};
ExtPlan ext_plan(const ExtCall& a, int cus);

constexpr int kBf16 = 0, kFp8 = 1, kNvfp4 = 2;   // XTG_KV_*
constexpr int kExtWaves = 4;                     // waves of a work-group
constexpr float kLog2e = 1.44269504088896341f;

// What the kernels take.
struct ExtArgs {
  const void *q, *k, *v;
  void* out;
  const uint8_t *ck, *cv;
  const void *ks, *vs;
  const int* slot_pos;
  const uint4 *pk, *pv;          // packed own keys and values
  float *acc, *ml;               // records [block][KV head][split][cols][d], [..][2]; row r of product dd at 16 dd + r
  int slots_pad, tile_lo, tiles;
  int ring, splits, records, cols, own;   // splits of the cached keys (few) or of all keys; own keys: their number
  int n_q, pos0, heads, group, window, bf16;
  uint32_t group_inv;            // ceil(2^16 / group): (col * group_inv) >> 16 is col / group for col * group <= 2^16
  int cached_end;                // cached positions from here on are not seen
  float factor;                  // what a product q.k is multiplied by in base-2 units (score_factor): factor * 2^factor_exp
  int factor_exp;
  float scale, kglobal, vglobal, softcap;
  const float* slopes;
  const int* first;
  const int* end;
};

// Queues the call's launches on scratch of the plan's size, each a callable that returns its name, given to `timed`.
using Timed = std::function<void(const std::function<std::string()>&)>;
void launch_attn_ext(const ExtCall& a, const ExtPlan& p, void* scratch, hipStream_t stream, const Timed& timed);

// The launches for heads of D dims (64, 128, 256) over a cache of `dtype`.
template <int D>
void ext_launch(const ExtCall& c, const ExtPlan& p, const ExtArgs& a, int dtype, hipStream_t stream, const Timed& timed);

}  // namespace xtg::hip
