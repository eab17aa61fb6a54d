// Attention with capped, biased and masked scores over a cache of any dtype: for each (row, q head) the softmax of the
// scores of the keys it sees, times their values, in one pass with a running maximum and sum.
#include <cfloat>
#include <climits>
#include <cmath>

#include "attention_ext.hpp"
#include "common.hpp"
#include "kv4.hpp"

namespace xtg::hip {

constexpr float kLog2e = 1.44269504088896341f;

struct ExtArgs {
  const void *q, *k, *v;
  void* out;
  const uint8_t *ck, *cv;
  const void *ks, *vs;
  const int* slot_pos;
  int dtype, slots, slots_pad;   // slots 0: no cache
  float kglobal, vglobal;
  int n_q, pos0, heads, kv_heads, d, window, bf16;
  int cached_end;                // cached positions from here on are not seen
  float scale, softcap;
  const float* slopes;
  const int* first;
  const int* end;
};

__device__ inline float row_value(const void* p, size_t at, int bf16) {
  return bf16 ? __uint_as_float(uint32_t(static_cast<const uint16_t*>(p)[at]) << 16)
              : float((__bf16)static_cast<const float*>(p)[at]);
}

__device__ inline float cached_value(const ExtArgs& a, bool v, int h, int slot, int dim) {
  const uint8_t* c = v ? a.cv : a.ck;
  const void* s = v ? a.vs : a.ks;
  const int d = a.d, pad = a.slots_pad;
  if (a.dtype == 0)
    return __uint_as_float(uint32_t(reinterpret_cast<const uint16_t*>(
               c)[v ? kv_v_index(h, slot, dim, pad, d) : kv_k_index(h, slot, dim, pad, d)]) << 16);
  if (a.dtype == 1) {
    const int code = c[v ? kv_v8_index(h, slot, dim, pad, d) : kv_k8_index(h, slot, dim, pad, d)];
    return __builtin_amdgcn_cvt_f32_fp8(code, 0) * static_cast<const float*>(s)[size_t(h) * size_t(pad) + size_t(slot)];
  }
  const Code4 at = v ? v4_code(h, slot, dim, pad, d) : k4_code(h, slot, dim, pad, d);
  const uint8_t sc = static_cast<const uint8_t*>(s)[v ? v4_scale(h, slot, dim, pad, d) : k4_scale(h, slot, dim, pad, d)];
  return e2m1_value(c[at.byte] >> (4 * at.high) & 15) * e4m3_scale_value(sc) * (v ? a.vglobal : a.kglobal);
}

// One work-group per (row, q head): 256 keys at a time, a score each thread, then a dim each thread.
__global__ void __launch_bounds__(256) attn_ext_kernel(ExtArgs a) {
  __shared__ float q[256], p[256], red[8];
  const int row = int(blockIdx.x), head = int(blockIdx.y), h = head / (a.heads / a.kv_heads), tid = int(threadIdx.x);
  const int t = a.pos0 + row;
  const int lo = max(max(0, a.first ? a.first[row] : 0), a.window > 0 ? t - a.window + 1 : 0);
  const int hi = a.end ? a.end[row] : t + 1;
  const size_t qrow = (size_t(row) * size_t(a.heads) + size_t(head)) * size_t(a.d);
  if (tid < a.d) q[tid] = row_value(a.q, qrow + size_t(tid), a.bf16);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc = 0.f;
  const int own = a.k ? a.n_q : 0;
  for (int k0 = 0; k0 < a.slots + own; k0 += 256) {
    const int key = k0 + tid, j = key - a.slots;   // own key j
    int pos = -1;
    if (key < a.slots) {
      pos = a.slot_pos[key];
      if (pos >= a.cached_end) pos = -1;
    } else if (j < own) {
      pos = a.pos0 + j;
    }
    float s = -INFINITY;
    if (pos >= lo && pos < hi) {
      s = 0.f;
      for (int x = 0; x < a.d; ++x)
        s += q[x] * (j < 0 ? cached_value(a, false, h, key, x)
                           : row_value(a.k, (size_t(j) * size_t(a.kv_heads) + size_t(h)) * size_t(a.d) + size_t(x), a.bf16));
      s *= a.scale;
      if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
      if (a.slopes) s -= a.slopes[head] * fabsf(float(t - pos));
      s *= kLog2e;
    }
    const float m_new = fmaxf(m, block_max<256>(s, red)), ref = m_new == -INFINITY ? 0.f : m_new;
    const float w = exp2f(s - ref), corr = exp2f(m - ref);
    p[tid] = pos >= lo && pos < hi ? w : -1.f;   // -1: not seen
    l = l * corr + block_sum<256>(w, red);
    m = m_new;
    acc *= corr;
    __syncthreads();
    if (tid < a.d)
      for (int x = 0; x < 256; ++x) {
        if (p[x] < 0.f) continue;
        const int kx = k0 + x, jx = kx - a.slots;
        acc += p[x] * (jx < 0 ? cached_value(a, true, h, kx, tid)
                              : row_value(a.v, (size_t(jx) * size_t(a.kv_heads) + size_t(h)) * size_t(a.d) + size_t(tid), a.bf16));
      }
    __syncthreads();
  }
  if (tid < a.d) {
    const float y = l > 0.f || l != l ? acc / l : 0.f;
    if (a.bf16)
      static_cast<__bf16*>(a.out)[qrow + size_t(tid)] = (__bf16)y;
    else
      static_cast<float*>(a.out)[qrow + size_t(tid)] = y;
  }
}

std::string launch_attn_ext(const ExtCall& c, hipStream_t stream) {
  ExtArgs a = {};
  a.q = c.q, a.k = c.k, a.v = c.v, a.out = c.out;
  if (const DevKv* kv = c.cache) {
    a.ck = static_cast<const uint8_t*>(kv->k);
    a.cv = static_cast<const uint8_t*>(kv->v);
    a.ks = kv->kscale, a.vs = kv->vscale, a.slot_pos = kv->slot_pos;
    a.dtype = kv->dtype(), a.slots = int(kv->slots), a.slots_pad = kv->slots_pad;
    a.kglobal = kv->kglobal, a.vglobal = kv->vglobal;
  }
  a.n_q = c.n_q, a.pos0 = int(c.pos0), a.heads = c.heads, a.kv_heads = c.kv_heads, a.d = c.d, a.window = c.window;
  a.bf16 = c.x_dtype == kXBF16;
  a.cached_end = c.k ? a.pos0 : INT_MAX;
  a.scale = c.scale, a.softcap = c.softcap, a.slopes = c.slopes, a.first = c.first, a.end = c.end;
  hipLaunchKernelGGL(attn_ext_kernel, dim3(unsigned(c.n_q), unsigned(c.heads)), dim3(256), 0, stream, a);
  HIP_CHECK(hipGetLastError());
  return "attn_ext_kernel";
}

}  // namespace xtg::hip
