// Kernels of attention over the pages of many sequences (the mathematics: attention_ext_kernels.hpp).
//
//   paged_attn_kernel: each wave takes 32-slot tiles of its own straight from the pages' operand layout into registers. A
//     work-group has 16 or 32 q-cols of one sequence and a part of their keys, for one KV head.
//   paged_merge_kernel: joins a q-col's parts in their order.
//
// What is beside a sequence's last row in its page, or before a window, is another time's: scores of it are masked, and its
// values are taken as zeros, since a weight of zero does not take away a NaN. A value that is not finite and that some
// rows of a work-group see reaches the others as NaN; such q-cols, whose sum of weights is finite, are computed again key
// by key (slow_col). A key without a page makes NaN of the rows that see it.
#pragma once

#include "attention_tiles.hpp"
#include "paged_device.hpp"

namespace xtg::hip {

// A tile whose slots are not all its sequence's.
template <int D, int T>
struct PagedTile : Tile<D, T> {
  bool partial = false;
  uint32_t valid = 0xffu;   // of the lane's 8 keys
  __device__ void begin_v() {
    if constexpr (T != kNvfp4) {   // (NVFP4: scales that are not numbers are zero already, and codes are finite)
      if (partial) {
        auto pair = [&](int e) { return (valid >> e & 1u ? 0xffffu : 0u) | (valid >> (e + 1) & 1u ? 0xffff0000u : 0u); };
        auto four = [&](int e) {
          uint32_t m = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) m |= valid >> (e + x) & 1u ? 0xffu << (8 * x) : 0u;
          return m;
        };
        const uint4 keep = T == kBf16 ? make_uint4(pair(0), pair(2), pair(4), pair(6))
                                      : make_uint4(four(0), four(4), four(0), four(4));
#pragma unroll
        for (auto& w : this->vw) w.x &= keep.x, w.y &= keep.y, w.z &= keep.z, w.w &= keep.w;
      }
    }
    Tile<D, T>::begin_v();
  }
};

// A work-group's piece.
struct Piece {
  int seq, block, split, splits, rec;   // rec: its record
  int blocks;
  Seq q;
  int cap;
};
__device__ inline bool piece_of(const PagedArgs& a, int task, Piece& p) {
  // about `budget` work-groups a KV head share the tiles of all blocks evenly
  const int lane = int(__lane_id());
  float total = 0.f;
  for (int s = lane; s < a.s.n_seqs; s += 64) {
    const Extent x = extent(a, s);
    total += float(x.blocks) * float(x.tiles);
  }
  total = wave_sum(total);
  int tasks = 0, recs = 0;
  for (int base = 0; base < a.s.n_seqs; base += 64) {
    const int s = base + lane;
    int n = 0, splits = 1;
    Extent x = {};
    if (s < a.s.n_seqs) {
      x = extent(a, s);
      splits = parts_of(a, x.tiles, total);
      n = x.blocks * splits;
    }
    const int r = splits > 1 ? n : 0, sum = wave_scan(n), rsum = wave_scan(r);
    const uint64_t hit = __ballot(uint32_t(task - tasks - (sum - n)) < uint32_t(n));
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int at = task - tasks - (of(sum) - of(n));
      p.seq = base + l;
      p.blocks = of(x.blocks);
      p.splits = of(splits);
      p.split = at / p.blocks;
      p.block = at - p.split * p.blocks;
      p.rec = recs + of(rsum) - of(r) + at;
      p.q = Seq{of(x.q.pos), of(x.q.row0), of(x.q.n)};
      p.cap = a.s.max_pages << a.s.shift;
      return true;
    }
    tasks += __builtin_amdgcn_readlane(sum, 63);
    recs += __builtin_amdgcn_readlane(rsum, 63);
  }
  return false;
}

// The positions lo <= p < lo + len that a sequence's row at position t sees.
__device__ inline Span paged_span(const PagedArgs& a, int t) {
  Span s;
  s.t = t;
  s.lo = a.window > 0 ? max(0, t - a.window + 1) : 0;
  s.len = t >= 0 ? uint32_t(t + 1 - s.lo) : 0u;
  return s;
}

__device__ inline Score paged_score(const PagedArgs& a, float global, int ex) {
  Score s;
  s.f = score_factor(a.factor, a.factor_exp, global, ex);
  s.top = fmaxf(a.softcap * kLog2e, FLT_MIN);
  s.slope = 0.f;
  return s;
}

// ------------------------------------------------------------------------------------------- a q-col key by key

template <int D, int T>
__device__ inline float paged_value(const PagedArgs& a, bool v, int h, int slot, int dim) {
  const uint8_t* c = v ? a.cv : a.ck;
  const void* s = v ? a.vs : a.ks;
  const int size = 1 << a.s.shift;
  if constexpr (T == kBf16) {
    const uint16_t x = reinterpret_cast<const uint16_t*>(c)[v ? kv_v_index(h, slot, dim, size, D) : kv_k_index(h, slot, dim, size, D)];
    return __uint_as_float(uint32_t(x) << 16);
  } else if constexpr (T == kFp8) {
    const int code = c[v ? kv_v8_index(h, slot, dim, size, D) : kv_k8_index(h, slot, dim, size, D)];
    return __builtin_amdgcn_cvt_f32_fp8(code, 0) * static_cast<const float*>(s)[size_t(h) * size_t(size) + size_t(slot)];
  } else {
    const Code4 at = v ? v4_code(h, slot, dim, size, D) : k4_code(h, slot, dim, size, D);
    const uint8_t sc = static_cast<const uint8_t*>(s)[v ? v4_scale(h, slot, dim, size, D) : k4_scale(h, slot, dim, size, D)];
    return e2m1_value(c[at.byte] >> (4 * at.high) & 15) * e4m3_scale_value(sc) * (v ? a.vglobal : a.kglobal);
  }
}

// One q-col by a work-group of 256 threads: 256 keys at a time, a score each thread, then a dim each thread. Keys without a
// page are NaN. lds: 768 + D floats.
template <int D, int T>
__device__ inline void paged_slow_col(const PagedArgs& a, int seq, int row, int t, int head, float* lds) {
  float *q = lds, *w = lds + D, *red = lds + D + 256;
  int* place = reinterpret_cast<int*>(lds + D + 272);   // [256]: the pool's head; [256]: the slot
  const int tid = int(threadIdx.x), h = head / a.group;
  const Span span = paged_span(a, t);
  const Score sc = paged_score(a, 1.f, 0);
  const size_t at = size_t(row) * size_t(a.ldq) + size_t(head * D + tid);
  __syncthreads();
  if (tid < D) q[tid] = a.bf16 ? (float)static_cast<const __bf16*>(a.q)[at] : (float)(__bf16) static_cast<const float*>(a.q)[at];
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int k0 = span.lo; k0 <= t; k0 += 256) {
    const int p = k0 + tid;
    const bool seen = uint32_t(p - span.lo) < span.len;
    const int page = seen ? page_of(a.s, seq, p) : -1, hh = max(page, 0) * a.kv_heads + h, slot = p & ((1 << a.s.shift) - 1);
    float s = -INFINITY;
    if (seen) {
      s = 0.f;
      for (int x = 0; x < D; ++x) s += q[x] * paged_value<D, T>(a, false, hh, slot, x);
      if (a.scale < 0.f) s = -s;
      s = page < 0 ? NAN : a.softcap > 0.f ? changed<kCap>(sc, s, 0) : changed<0>(sc, s, 0);
    }
    const float top = block_max<256>(seen ? fmaxf(s, -FLT_MAX) : -INFINITY, red), m_new = fmaxf(m, top);
    const float e = __builtin_amdgcn_exp2f(s - m_new), corr = __builtin_amdgcn_exp2f(m - m_new);
    place[tid] = hh, place[256 + tid] = slot;
    w[tid] = seen ? e : -1.f;   // -1: not seen
    l = l * corr + block_sum<256>(seen ? e : 0.f, red);
    m = m_new;
    acc *= corr;
    __syncthreads();
    if (tid < D)
      for (int x = 0; x < 256; ++x) {
        if (w[x] == -1.f) continue;
        acc += w[x] * paged_value<D, T>(a, true, place[x], place[256 + x], tid);
      }
    __syncthreads();
  }
  if (tid < D) {
    const float y = l == 0.f ? (span.len ? NAN : 0.f) : acc / l;
    const size_t to = (size_t(row) * size_t(a.heads) + size_t(head)) * D + size_t(tid);
    if (a.bf16)
      static_cast<__bf16*>(a.out)[to] = (__bf16)y;
    else
      static_cast<float*>(a.out)[to] = y;
  }
}

// ------------------------------------------------------------------------------------------------- the scan

template <int D, int QB>
constexpr size_t paged_lds() { return size_t(kPagedWaves) * QB * (2 * 16 + D * 16) * sizeof(float); }

template <int D, int QB, int T, int MOD>
__global__ void __launch_bounds__(kPagedWaves * 64, QB * D > 256 ? 1 : 2) paged_attn_kernel(PagedArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  float* lds = reinterpret_cast<float*>(smem);
  __shared__ uint32_t again;   // q-cols to be computed again
  using X8 = typename OperandOf<T>::type;
  constexpr int ND = D / 16;
  const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), g = lane >> 4, i = lane & 15;
  const int h = int(blockIdx.x) % a.kv_heads, task = int(blockIdx.x) / a.kv_heads;
  Piece p;
  if (!piece_of(a, task, p)) return;   // (the whole work-group: every wave finds the same)
  if (p.splits > 1 && p.rec >= a.records) return;   // (only where starts decrease)
  if (threadIdx.x == 0) again = 0;

  // the block's q-cols: c0 .. c0 + cols - 1 of the sequence, rows r0 .. r1
  const long long c0 = (long long)p.block * a.cols;
  const int r0 = int(c0 / a.group), rem = int(c0 - (long long)r0 * a.group);
  const int r1 = int(min((long long)p.q.n, (c0 + a.cols + a.group - 1) / a.group)) - 1;
  const bool out_of = p.q.pos < 0;
  const int first = out_of ? -1 : p.q.pos + r0, last = out_of ? -1 : p.q.pos + r1;
  const int lo = paged_span(a, first).lo, hi = min(last + 1, p.cap);   // positions that some row of the block sees
  const int tlo = lo >> 5, tiles = max(0, ((hi + 31) >> 5) - tlo);
  const int t_begin = tlo + int((long long)tiles * p.split / p.splits), t_end = tlo + int((long long)tiles * (p.split + 1) / p.splits);

  // a q-col's row in the sequence (n or more: none), and its head
  auto col_row = [&](int c) { return r0 + int(uint32_t(rem + c) * a.group_inv >> 16); };
  auto col_head = [&](int c) { return h * a.group + rem + c - (col_row(c) - r0) * a.group; };

  FewState<D, QB> st;
  bf16x8 x[QB][D / 32];
  X8 q[QB][D / 32];
  Span span[QB];
  Score sc[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    st.m[qb] = -INFINITY, st.l[qb] = 0.f;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int row = col_row(qb * 16 + i);
    const bool live = row < p.q.n;
    const size_t at = live ? size_t(p.q.row0 + row) * size_t(a.ldq) + size_t(col_head(qb * 16 + i)) * D : 0;
    row_chunks(a.q, a.bf16, live, [&](int c) { return at + size_t(Tile<D, T>::q_dim(c, g)); }, x[qb]);
    span[qb] = live && !out_of ? paged_span(a, p.q.pos + row) : Span{0, 0u, 0};
    sc[qb] = paged_score(a, 1.f, 0);
  }

  int t = t_begin + wave;
  if (t < t_end) {
    // the pages of the wave's next 64 tiles, one a lane
    int pages = 0, k = 0;
    auto load_pages = [&](int from) {
      const int tile = from + kPagedWaves * lane;
      pages = tile < t_end ? page_of(a.s, p.seq, 32 * tile) : -1;
    };
    auto place = [&](int page, int tile) {
      return (((size_t(uint32_t(max(page, 0))) * size_t(a.kv_heads) + size_t(h)) << a.s.shift) +
              size_t((32 * tile) & ((1 << a.s.shift) - 1)));
    };
    load_pages(t);
    int page = __builtin_amdgcn_readlane(pages, 0);
    PagedTile<D, T> tile;
    size_t at = place(page, t);
    tile.load_k(a, at, lane);
    tile.load_v(a, at, lane);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if (a.scale < 0.f) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) x[qb][c] = -x[qb][c];
      }
      const int ex = to_operand<T != kBf16>(x[qb], q[qb], [](float v) { return xor32_max(xor16_max(v)); });
      sc[qb].f = score_factor(a.factor, a.factor_exp, T == kNvfp4 ? a.kglobal : 1.f, ex);
    }
    for (; t < t_end; t += kPagedWaves) {
      const int n = t + kPagedWaves;
      const bool lost = page < 0;
      const int base = 32 * t + 4 * g;
      tile.partial = 32 * t < lo || 32 * t + 32 > hi;
      if (tile.partial) {
        tile.valid = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int pos = base + (e < 4 ? e : 12 + e);
          tile.valid |= pos >= lo && pos < hi ? 1u << e : 0u;
        }
      }
      if (lost) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (uint32_t(base + (e < 4 ? e : 12 + e) - span[qb].lo) < span[qb].len) st.l[qb] = NAN;
      }
      if (++k == 64) {
        k = 0;
        load_pages(n);
      }
      page = __builtin_amdgcn_readlane(pages, k);
      if (n < t_end) at = place(page, n);   // past the end: the same tile again, which is not used
      few_tile<D, QB, MOD>(tile, q, span, sc, st, make_int4(base, base + 1, base + 2, base + 3),
                           make_int4(base + 16, base + 17, base + 18, base + 19), [&] { tile.load_k(a, at, lane); },
                           [&] { tile.load_v(a, at, lane); });
    }
  }
  // a row past the last position that its table has a page for
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    if (span[qb].len && span[qb].t >= p.cap) st.l[qb] = NAN;
  if (T == kNvfp4 && a.vglobal != 1.f) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] *= a.vglobal;
  }

  // the waves' states joined: the maxima and sums, then the accumulators, each wave a part of the sums
  float* ml = lds;                                     // [wave][QB * 16][2]
  float* part = lds + kPagedWaves * QB * 2 * 16;       // [wave][QB][products][64 lanes][4]
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
    for (int w = 0; w < kPagedWaves; ++w) m = fmaxf(m, ml[(w * QB * 16 + qb * 16 + i) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w)
      l += ml[(w * QB * 16 + qb * 16 + i) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * QB * 16 + qb * 16 + i) * 2] - ref);
    const float corr = __builtin_amdgcn_exp2f(st.m[qb] - ref);
    m_all[qb] = m;
    l_all[qb] = l;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] *= corr;
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int dd = 0; dd < ND; ++dd)
      *reinterpret_cast<f32x4*>(part + (((wave * QB + qb) * ND + dd) * 64 + lane) * 4) = st.acc[qb][dd];
  __syncthreads();
  const size_t rec = (size_t(p.rec) * size_t(a.kv_heads) + size_t(h)) * size_t(a.cols);
  const bool several = r1 > r0;   // rows
#pragma unroll
  for (int u = 0; u < QB * ND; u += kPagedWaves) {
    const int qd = u + wave, qb = qd / ND, dd = qd % ND;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) y += *reinterpret_cast<const f32x4*>(part + ((w * QB * ND + qd) * 64 + lane) * 4);
    const int mine = qb * 16 + i, row = col_row(mine);
    if (row >= p.q.n) continue;
    float l = l_all[0];
    if constexpr (QB == 2) l = qb ? l_all[1] : l;
    if (p.splits == 1) {
      const bool sees = !out_of;
      bool bad = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) bad |= several && !not_finite(l) && not_finite(y[r]);
      if (bad) atomicOr(&again, 1u << mine);
      const float inv = l == 0.f ? (sees ? NAN : 0.f) : 1.f / l;   // (scores of minus infinity alone: NaN)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int dim = Tile<D, T>::dim(dd, 4 * g + r);
        const size_t to = (size_t(p.q.row0 + row) * size_t(a.heads) + size_t(col_head(mine))) * D + size_t(dim);
        if (a.bf16)
          static_cast<__bf16*>(a.out)[to] = (__bf16)(y[r] * inv);
        else
          static_cast<float*>(a.out)[to] = y[r] * inv;
      }
    } else {
      *reinterpret_cast<f32x4*>(a.acc + (rec + size_t(mine)) * D + size_t(16 * dd + 4 * g)) = y;
    }
  }
  if (wave == 0 && g < QB) {
    const int col = g * 16 + i, row = col_row(col);
    float m = m_all[0], l = l_all[0];
    if constexpr (QB == 2) m = g ? m_all[1] : m, l = g ? l_all[1] : l;
    if (row < p.q.n) {
      if (p.splits > 1) {
        a.ml[(rec + size_t(col)) * 2] = m;
        a.ml[(rec + size_t(col)) * 2 + 1] = l;
      }
      if (p.split == 0 && h == 0)
        a.info[size_t(p.q.row0 + row) * size_t(a.group) + size_t(col_head(col))] = make_int4(p.rec, p.blocks, p.splits << 8 | col, p.seq);
    }
  }
  if (p.splits > 1) return;
  __syncthreads();
  for (uint32_t bits = again; bits; bits &= bits - 1) {
    const int col = __builtin_ctz(bits), row = col_row(col);
    paged_slow_col<D, T>(a, p.seq, p.q.row0 + row, p.q.pos + row, col_head(col), lds);
  }
}

// ---------------------------------------------------------------------------------------------------- merge

// One q-col a work-group: D / 4 lanes to a record's accumulator, 1024 / D records at once.
template <int D, int T>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedArgs a) {
  constexpr int L = D / 4, G = 256 / L;
  __shared__ float4 part[256];
  __shared__ float slow[784 + D], all_m[4], all_l[4];
  const int row = int(blockIdx.x) / a.heads, head = int(blockIdx.x) % a.heads, h = head / a.group;
  const int tid = int(threadIdx.x), x = tid % L, grp = tid / L;
  if (a.s.starts && (row < a.s.starts[0] || row >= a.s.starts[a.s.n_seqs])) return;   // no sequence's
  const int4 info = a.info[size_t(row) * size_t(a.group) + size_t(head % a.group)];
  const int splits = info.z >> 8, step = info.y;
  if (splits <= 1 || info.x < 0 || (long long)info.x + (long long)(splits - 1) * step >= a.records) return;
  const size_t stride = size_t(step) * size_t(a.kv_heads) * size_t(a.cols);
  const size_t rec0 = (size_t(info.x) * size_t(a.kv_heads) + size_t(h)) * size_t(a.cols) + size_t(info.z & 0xff);
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + rec0;
  const float* acc = a.acc + rec0 * D + size_t(4 * x);
  float m = -INFINITY;
  for (int s = tid; s < splits; s += 256) m = fmaxf(m, ml[size_t(s) * stride].x);
  m = wave_max(m);
  if ((tid & 63) == 0) all_m[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(all_m[0], all_m[1]), fmaxf(all_m[2], all_m[3]));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = grp; s < splits; s += G) {
    const float2 w = ml[size_t(s) * stride];
    const float4 v = *reinterpret_cast<const float4*>(acc + size_t(s) * stride * D);
    const float f = __builtin_amdgcn_exp2f(w.x - ref);
    l += w.y * (w.x == -INFINITY && !not_finite(w.y) ? 0.f : f);   // (a NaN without a maximum: a key without a page)
    if (f != 0.f) y.x += v.x * f, y.y += v.y * f, y.z += v.z * f, y.w += v.w * f;
  }
  part[tid] = y;
  l = wave_sum(x == 0 ? l : 0.f);
  if ((tid & 63) == 0) all_l[tid >> 6] = l;
  __syncthreads();
  l = all_l[0] + all_l[1] + all_l[2] + all_l[3];
  bool bad = false;
  const Seq q = seq_at(a.s, info.w);
  if (grp == 0) {
    y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < G; ++s) {
      const float4 u = part[s * L + x];
      y.x += u.x, y.y += u.y, y.z += u.z, y.w += u.w;
    }
    bad = q.n > 1 && !not_finite(l) && (not_finite(y.x) || not_finite(y.y) || not_finite(y.z) || not_finite(y.w));
    const float inv = l == 0.f ? NAN : 1.f / l;
    const float o[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int u = 4 * x + r;
      const size_t at = (size_t(row) * size_t(a.heads) + size_t(head)) * D + size_t(Tile<D, T>::dim(u >> 4, u & 15));
      if (a.bf16)
        static_cast<__bf16*>(a.out)[at] = (__bf16)o[r];
      else
        static_cast<float*>(a.out)[at] = o[r];
    }
  }
  if (!__syncthreads_or(bad)) return;
  paged_slow_col<D, T>(a, info.w, row, q.pos + row - q.row0, head, slow);
}

// ---------------------------------------------------------------------------------------------------- launches

template <int D, int T, int MOD>
void paged_go(const PagedAttnCall& c, const PagedPlan& p, const PagedArgs& a, hipStream_t stream, const PagedTimed& timed) {
  timed([&] {
    const dim3 grid{unsigned(p.tasks) * unsigned(a.kv_heads)}, block{kPagedWaves * 64};
    auto go = [&](auto kernel, size_t lds) {
      allow_lds(reinterpret_cast<const void*>(kernel), lds);
      hipLaunchKernelGGL(kernel, grid, block, lds, stream, a);
    };
    if (p.cols == 16)
      go(&paged_attn_kernel<D, 1, T, MOD>, paged_lds<D, 1>());
    else
      go(&paged_attn_kernel<D, 2, T, MOD>, paged_lds<D, 2>());
    HIP_CHECK(hipGetLastError());
    return strf("paged_attn_kernel<%d, %d, %d, %d>", D, p.cols / 16, T, MOD);
  });
  timed([&] {
    hipLaunchKernelGGL((paged_merge_kernel<D, T>), dim3(unsigned(c.seqs.n_rows) * unsigned(c.heads)), dim3(256), 0, stream, a);
    HIP_CHECK(hipGetLastError());
    return strf("paged_merge_kernel<%d, %d>", D, T);
  });
}

template <int D>
void paged_launch(const PagedAttnCall& c, const PagedPlan& p, const PagedArgs& a, hipStream_t stream, const PagedTimed& timed) {
  auto of = [&](auto t) {
    constexpr int T = decltype(t)::value;
    if (c.softcap > 0.f)
      paged_go<D, T, kCap>(c, p, a, stream, timed);
    else
      paged_go<D, T, 0>(c, p, a, stream, timed);
  };
  if (c.cache->type == kBf16) of(std::integral_constant<int, kBf16>{});
  if (c.cache->type == kFp8) of(std::integral_constant<int, kFp8>{});
  if (c.cache->type == kNvfp4) of(std::integral_constant<int, kNvfp4>{});
}

}  // namespace xtg::hip
