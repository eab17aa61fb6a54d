// How an attention call over paged caches is cut up and queued (kernels: paged_attention_kernels.hpp, compiled for each head
// size in paged_attention_d64.hip, _d128.hip and _d256.hip).
#include <algorithm>
#include <cmath>

#include "attention_ext.hpp"
#include "common.hpp"
#include "kernels.hpp"
#include "paged.hpp"

namespace xtg::hip {

PagedPlan paged_plan(const PagedAttnCall& a, int cus) {
  PagedPlan p;
  const int kv_heads = a.cache->kv_heads, group = a.heads / kv_heads, seqs = a.seqs.n_seqs;
  const long long cols = (long long)a.seqs.n_rows * group;
  // 32 q-cols a work-group where sequences have more than 16 on the average, but not a prompt's number (16 sequences of 8 rows
  // of 4 q heads a KV head over NVFP4 pages: 37 us; as blocks of many q-cols 62)
  p.cols = cols > 16LL * seqs && cols <= 32LL * seqs ? 32 : 16;
  // (heads of 256 dims: 32 do not fit a wave's registers where work-groups have eight)
  const long long most = a.seqs.starts ? cols : group;   // q-cols of a sequence
  if (a.cache->head_dim == 256 && most > p.cols) p.cols = 16;
  p.many = most > p.cols;
  // the work-groups that are resident at once (half to four times as many: within 2 % or slower)
  p.budget = std::max(1, (p.many ? cus : 2 * cus) / kv_heads);
  // a sequence's last block and a block's last part are begun ones; and total / budget is rounded, in FP32
  const long long parts = p.budget + p.budget / 64 + 1, tasks = (p.many ? cols / kManyCols : 0) + seqs + parts;
  XTG_CHECK(tasks * kv_heads < (1LL << 31), "paged_attention: %d rows of %d sequences and %d heads", a.seqs.n_rows, seqs, a.heads);
  p.tasks = int(tasks);
  // a block of several parts has at least one whole part's tiles for every two of them
  p.records = int(std::min(tasks, 2 * parts)) * (p.many ? kManyCols : p.cols);
  // (tables of a few hundred positions: no block has a second part, and no merge is launched)
  if (((long long)a.seqs.max_pages << a.seqs.shift) <= 32 * kFewLeast) p.records = 0;
  const size_t n = size_t(p.records) * size_t(kv_heads);
  p.acc_bytes = n * size_t(a.cache->head_dim) * sizeof(float);
  p.ml_bytes = n * 2 * sizeof(float);
  p.info_bytes = size_t(a.seqs.n_rows) * size_t(group) * sizeof(int4);
  return p;
}

void launch_paged_attn(const PagedAttnCall& c, const PagedPlan& p, void* scratch, hipStream_t stream, const PagedTimed& timed) {
  const DevPaged& kv = *c.cache;
  PagedArgs a = {};
  a.s = c.seqs;
  a.q = c.q, a.out = c.out, a.ldq = c.ldq;
  a.ck = static_cast<const uint8_t*>(kv.k), a.cv = static_cast<const uint8_t*>(kv.v);
  a.ks = kv.ks, a.vs = kv.vs;
  char* at = static_cast<char*>(scratch);
  a.acc = reinterpret_cast<float*>(at);
  a.ml = reinterpret_cast<float*>(at + p.acc_bytes);
  a.info = reinterpret_cast<int4*>(at + p.acc_bytes + p.ml_bytes);
  a.heads = c.heads, a.kv_heads = kv.kv_heads, a.group = c.heads / kv.kv_heads;
  a.group_inv = (65536u + uint32_t(a.group) - 1u) / uint32_t(a.group);
  a.cols = p.cols, a.budget = p.budget, a.records = p.records;
  a.window = c.window, a.bf16 = c.x_dtype == kXBF16;
  const double log2e = kLog2e;
  a.factor = float(std::frexp(std::fabs(double(c.scale)) * (c.softcap > 0.f ? 2 * log2e / c.softcap : log2e), &a.factor_exp));
  a.scale = c.scale, a.kglobal = kv.kglobal, a.vglobal = kv.vglobal, a.softcap = c.softcap;
  if (kv.head_dim == 64)
    paged_launch<64>(c, p, a, stream, timed);
  else if (kv.head_dim == 128)
    paged_launch<128>(c, p, a, stream, timed);
  else if (kv.head_dim == 256)
    paged_launch<256>(c, p, a, stream, timed);
  else
    fail("paged_attention: head_dim %d", kv.head_dim);
}

}  // namespace xtg::hip
