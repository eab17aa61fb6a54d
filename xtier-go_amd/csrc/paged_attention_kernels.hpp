// Kernels of attention over the pages of many sequences (the mathematics: attention_ext_kernels.hpp).
//
//   paged_attn_kernel: a work-group finds its piece (a block of one sequence's q-cols, a part of their keys, one KV head) and
//     does it in one of two ways, side by side in one launch, so that prompts, which the matrix ops bound, run beside decoded
//     tokens, which the pages' bytes bound:
//     few_piece: up to 16 or 32 q-cols, the sequence's only block. Each wave takes 32-slot tiles of its own straight from the
//       pages' operand layout into registers.
//     many_piece: 128 q-cols, 32 a wave. Four waves share tiles through LDS, each dequantised once; another four do the same
//       with every other tile, so that a SIMD has two waves whatever the number of blocks.
//     Work-groups have four waves, and two fit a CU; where a call may have many_pieces, eight.
//   paged_merge_kernel: joins a q-col's parts in their order.
// Decode steps read their pages at 5.6 to 5.7 TB/s (64 sequences of up to 8192 FP8 positions of 8 KV heads of 128 dims: 85 us and
// a merge of 4); over NVFP4 pages, 4.1 TB/s (64 us), the vector operations that make operands of codes take 42 % of all cycles. Prompts: 512 rows of 32 heads of
// 128 dims over 16384 BF16 positions take 171 us (0.8 PFLOP/s), bound by LDS reads and the waits at a step's barrier; short
// prompts by their longest block's chain of steps (2 to 2.5 us of two tiles of 256 dims) and 13 us before and behind it.
//
// What is beside a sequence's last row in its page, or before a window, is another time's: scores of it are masked, and its
// values are taken as zeros, since a weight of zero does not take away a NaN. A value that is not finite and that some
// rows of a work-group see reaches the others as NaN; such q-cols, whose sum of weights is finite, are computed again key
// by key (slow_col), also where the value is the row's own (64 rows of 32 heads over 8000 positions with one NaN in V that all see: 8.3 ms,
// without it 33 us). A key without a page makes NaN of the rows that see it.
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
  int seq, block, split, splits;
  long long rec;   // its records' place: q-cols of a KV head before it
  int blocks;
  bool many;
  Seq q;
  int cap;         // positions that the table has pages for
};
template <bool MANY>
__device__ inline bool piece_of(const PagedArgs& a, int task, Piece& p) {
  // about `budget` work-groups a KV head share the tiles of all blocks evenly
  const int lane = int(__lane_id());
  Extent own = {};   // of the lane's sequence among the first 64, which is looked up once
  if (lane < a.s.n_seqs) own = extent(a, lane);
  auto extent_of = [&](int s) { return s < 64 ? own : extent(a, s); };
  float total = 0.f;
  int all = 0;
  for (int s = lane; s < a.s.n_seqs; s += 64) {
    const Extent x = extent_of(s);
    total += float(x.blocks) * float(x.tiles);
    all += x.blocks;
  }
  all = wave_total(all);
  int chunk = first_chunk(a, wave_sum(total), all);
  for (int step = 0; step < kChunkSteps && all < a.budget; ++step) {
    int n = 0;
    for (int s = lane; s < a.s.n_seqs; s += 64) {
      const Extent x = extent_of(s);
      n += x.blocks * parts_of(x, chunk);
    }
    if (!next_chunk(a, chunk, wave_total(n), all)) break;
  }
  int tasks = 0, recs = 0;
#pragma unroll
  for (int role = MANY ? 1 : 0; role >= 0; --role)   // those of many q-cols, whose work-groups take longest, first
    for (int base = 0; base < a.s.n_seqs; base += 64) {
      const int s = base + lane;
      int n = 0, splits = 1;
      Extent x = {};
      if (s < a.s.n_seqs) {
        x = extent_of(s);
        splits = parts_of(x, chunk);
        n = int(x.many) == role ? x.blocks * splits : 0;
      }
      const int cols = role ? kManyCols : a.cols, r = splits > 1 ? n : 0, sum = wave_scan(n), rsum = wave_scan(r);
      const uint64_t hit = __ballot(uint32_t(task - tasks - (sum - n)) < uint32_t(n));
      if (hit) {
        const int l = __builtin_ctzll(hit);
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        const int at = task - tasks - (of(sum) - of(n));
        p.seq = base + l;
        p.many = role != 0;
        p.blocks = of(x.blocks);
        p.splits = of(splits);
        p.split = at / p.blocks;
        p.block = p.blocks - 1 - (at - p.split * p.blocks);   // later rows, which see most, first
        p.rec = recs + (long long)(of(rsum) - of(r) + p.split * p.blocks + p.block) * cols;
        p.q = Seq{of(x.q.pos), of(x.q.row0), of(x.q.n)};
        p.cap = a.s.max_pages << a.s.shift;
        return true;
      }
      tasks += __builtin_amdgcn_readlane(sum, 63);
      recs += __builtin_amdgcn_readlane(rsum, 63) * cols;
    }
  return false;
}

// Where a page's slot of position p lies for KV head h, counted in slots. (No page: page 0's, which is there.)
__device__ inline size_t place_of(const PagedArgs& a, int page, int h, int p) {
  return ((size_t(uint32_t(max(page, 0))) * size_t(a.kv_heads) + size_t(h)) << a.s.shift) + size_t(p & ((1 << a.s.shift) - 1));
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

// Values 4 u .. +4 of a record's order into an output row: neighbours but for NVFP4's order.
template <int D, int T, class X>
__device__ inline void put4(X* row, int u, const float (&y)[4]) {
  const int dim = Tile<D, T>::dim(u >> 2, 4 * (u & 3));
  if constexpr (T == kNvfp4) {
#pragma unroll
    for (int r = 0; r < 4; ++r) row[Tile<D, T>::dim(u >> 2, 4 * (u & 3) + r)] = X(y[r]);
  } else if constexpr (sizeof(X) == 2) {
    const X z[4] = {X(y[0]), X(y[1]), X(y[2]), X(y[3])};
    *reinterpret_cast<uint2*>(row + dim) = __builtin_bit_cast(uint2, z);
  } else {
    *reinterpret_cast<float4*>(row + dim) = make_float4(y[0], y[1], y[2], y[3]);
  }
}
template <int D, int T>
__device__ inline void put4(const PagedArgs& a, size_t at, int u, const float (&y)[4]) {
  if (a.bf16)
    put4<D, T>(static_cast<__bf16*>(a.out) + at, u, y);
  else
    put4<D, T>(static_cast<float*>(a.out) + at, u, y);
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

// One q-col by 256 threads of a work-group (the others wait with them): 256 keys at a time, a score each thread, then a dim
// each thread. Keys without a page are NaN. lds: 784 + D floats.
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
    const bool seen = tid < 256 && uint32_t(p - span.lo) < span.len;
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
    if (tid < 256) {
      place[tid] = hh, place[256 + tid] = slot;
      w[tid] = seen ? e : -1.f;   // -1: not seen
    }
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

// ------------------------------------------------------------------------------------------------- few q-cols

template <int D, int QB>
constexpr size_t few_floats() { return size_t(4) * QB * (2 * 16 + D * 16); }

// Heads of 256 dims: a wave's q operand is in LDS (the same for every wave), so that a tile fits the registers beside the
// accumulators. (With it in registers, 128 of them spilled: 256 sequences' windows of 1024 took 219 us.)
template <int D>
constexpr bool kQInLds = D == 256;
template <int D, int QB>
constexpr size_t few_lds() {
  const size_t join = few_floats<D, QB>() * sizeof(float), q = kQInLds<D> ? size_t(QB) * 32 * D : 0;
  return join > q ? join : q;
}

// Weights over BF16 and FP8 pages, whose values are BF16 operands, are sums of two BF16 values: with one, outputs were off by 1.4
// times what FP32 weights and the rounding of BF16 rows are (2.3e-3 of their norm, 1.7e-3), and up to 16 q-cols, which wait for the
// pages' bytes, take no longer with two (64 tokens over 8192 FP8 positions 90.0 us and 90.1, 256 windows over BF16 pages 169.4 and
// 169.7). More q-cols do: 64 x 8 rows over FP8 pages 145 us and 154, and prompts, which the matrix ops bound, 49 and 56 (a chunk beside
// single tokens 136 and 138); so 32 q-cols, and many_piece's, have one of 8 bits. NVFP4 pages' operands are f16, weights of 11 bits.
template <int QB, int T>
constexpr bool kTwoTerms = T != kNvfp4 && QB == 1;

template <int D, int QB, class X8, bool LDS>
struct FewQ {
  static constexpr bool kInLds = LDS;
  const X8* p;   // [QB][D / 32], in LDS a lane's 64 apart
  __device__ X8 operator()(int qb, int c) const { return p[(qb * (D / 32) + c) * (LDS ? 64 : 1)]; }
};

template <int D, int QB, int T, int MOD, int WAVES>
__device__ inline void few_piece(const PagedArgs& a, const Piece& p, int h, uint8_t* smem, uint32_t& again) {
  using X8 = typename OperandOf<T>::type;
  constexpr int ND = D / 16;
  float* lds = reinterpret_cast<float*>(smem);
  const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), g = lane >> 4, i = lane & 15;
  const bool out_of = p.q.pos < 0;
  const int last = out_of ? -1 : p.q.pos + p.q.n - 1;
  const int lo = paged_span(a, out_of ? -1 : p.q.pos).lo, hi = min(last + 1, p.cap);   // positions that some row sees
  const int tlo = lo >> 5, tiles = max(0, ((hi + 31) >> 5) - tlo);
  const int t_begin = tlo + int((long long)tiles * p.split / p.splits), t_end = tlo + int((long long)tiles * (p.split + 1) / p.splits);

  // a q-col's row in the sequence (n or more: none), and its head
  auto col_row = [&](int c) { return int(uint32_t(c) * a.group_inv >> 16); };
  auto col_head = [&](int c) { return h * a.group + c - col_row(c) * a.group; };

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
  // the pages of the wave's next 64 tiles, one a lane
  int pages = -1, k = 0;
  auto load_pages = [&](int from) {
    const int tile = from + WAVES * lane;
    pages = tile < t_end ? page_of(a.s, p.seq, 32 * tile) : -1;
  };
  load_pages(t);
  int page = __builtin_amdgcn_readlane(pages, 0);
  PagedTile<D, T> tile;
  size_t at = place_of(a, page, h, 32 * t);
  if (t < t_end) {
    tile.load_k(a, at, lane);
    tile.load_v(a, at, lane);
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    if (a.scale < 0.f) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) x[qb][c] = -x[qb][c];
    }
    const int ex = to_operand<T != kBf16>(x[qb], q[qb], [](float v) { return xor32_max(xor16_max(v)); });
    sc[qb].f = score_factor(a.factor, a.factor_exp, T == kNvfp4 ? a.kglobal : 1.f, ex);
  }
  X8* ql = reinterpret_cast<X8*>(smem);   // [QB][D / 32][64 lanes]
  if constexpr (kQInLds<D>) {
    if (wave == 0) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int c = 0; c < D / 32; ++c) ql[(qb * (D / 32) + c) * 64 + lane] = q[qb][c];
    }
    __syncthreads();
  }
  const FewQ<D, QB, X8, kQInLds<D>> q_at{kQInLds<D> ? ql + lane : &q[0][0]};
  for (; t < t_end; t += WAVES) {
    const int n = t + WAVES;
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
    if (n < t_end) at = place_of(a, page, h, 32 * n);   // past the end: the same tile again, which is not used
    few_tile<D, QB, MOD, kTwoTerms<QB, T>>(tile, q_at, span, sc, st, make_int4(base, base + 1, base + 2, base + 3),
                         make_int4(base + 16, base + 17, base + 18, base + 19), [&] { tile.load_k(a, at, lane); },
                         [&] { tile.load_v(a, at, lane); });
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
  if constexpr (kQInLds<D>) __syncthreads();   // q's place is the states'

  // the waves' states joined: the maxima and sums, then the accumulators, each wave a part of the sums
  float* ml = lds;                           // [wave][QB * 16][2]
  float* part = lds + 4 * QB * 2 * 16;       // [wave][QB][products][64 lanes][4]
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) st.l[qb] = xor32_sum(xor16_sum(st.l[qb]));
  const bool lead = wave < 4;
  if constexpr (WAVES == 8) {   // the last four into the first four
    const int of = wave & 3;
    if (!lead) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        if (g == 0) ml[(of * QB * 16 + qb * 16 + i) * 2] = st.m[qb], ml[(of * QB * 16 + qb * 16 + i) * 2 + 1] = st.l[qb];
#pragma unroll
        for (int dd = 0; dd < ND; ++dd)
          *reinterpret_cast<f32x4*>(part + (((of * QB + qb) * ND + dd) * 64 + lane) * 4) = st.acc[qb][dd];
      }
    }
    __syncthreads();
    if (lead) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const float m2 = ml[(of * QB * 16 + qb * 16 + i) * 2], l2 = ml[(of * QB * 16 + qb * 16 + i) * 2 + 1];
        const float m = fmaxf(st.m[qb], m2), ref = m == -INFINITY ? 0.f : m;
        const float f = __builtin_amdgcn_exp2f(st.m[qb] - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
        st.m[qb] = m;
        st.l[qb] = st.l[qb] * f + l2 * f2;
#pragma unroll
        for (int dd = 0; dd < ND; ++dd)
          st.acc[qb][dd] = st.acc[qb][dd] * f + *reinterpret_cast<const f32x4*>(part + (((of * QB + qb) * ND + dd) * 64 + lane) * 4) * f2;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float l = st.l[qb];
    if (g == 0 && lead) {
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
    for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[(w * QB * 16 + qb * 16 + i) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      l += ml[(w * QB * 16 + qb * 16 + i) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * QB * 16 + qb * 16 + i) * 2] - ref);
    const float corr = __builtin_amdgcn_exp2f(st.m[qb] - ref);
    m_all[qb] = m;
    l_all[qb] = l;
#pragma unroll
    for (int dd = 0; dd < ND; ++dd) st.acc[qb][dd] *= corr;
  }
  if (lead) {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int dd = 0; dd < ND; ++dd)
        *reinterpret_cast<f32x4*>(part + (((wave * QB + qb) * ND + dd) * 64 + lane) * 4) = st.acc[qb][dd];
  }
  __syncthreads();
  const size_t rec = size_t(p.rec) * size_t(a.kv_heads) + size_t(h * a.cols);
#pragma unroll
  for (int u = lead ? 0 : QB * ND; u < QB * ND; u += 4) {
    const int qd = u + wave, qb = qd / ND, dd = qd % ND;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) y += *reinterpret_cast<const f32x4*>(part + ((w * QB * ND + qd) * 64 + lane) * 4);
    const int mine = qb * 16 + i, row = col_row(mine);
    if (row >= p.q.n) continue;
    float l = l_all[0];
    if constexpr (QB == 2) l = qb ? l_all[1] : l;
    if (p.splits == 1) {
      bool bad = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) bad |= p.q.n > 1 && !not_finite(l) && not_finite(y[r]);
      if (bad) atomicOr(&again, 1u << mine);
      const float inv = l == 0.f ? (out_of ? 0.f : NAN) : 1.f / l;   // (scores of minus infinity alone: NaN)
      put4<D, T>(a, (size_t(p.q.row0 + row) * size_t(a.heads) + size_t(col_head(mine))) * D, 4 * dd + g,
                 {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv});
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
        a.info[size_t(p.q.row0 + row) * size_t(a.group) + size_t(col_head(col))] = make_int4(int(p.rec), p.blocks << 1, p.splits << 8 | col, p.seq);
    }
  }
  if (p.splits > 1) return;
  __syncthreads();
  for (uint32_t bits = again; bits; bits &= bits - 1) {
    const int col = __builtin_ctz(bits), row = col_row(col);
    paged_slow_col<D, T>(a, p.seq, p.q.row0 + row, p.q.pos + row, col_head(col), lds);
  }
}

// ------------------------------------------------------------------------------------------------ many q-cols

// What a thread stages of a tile of TK keys (attention_tiles.hpp) whose 32-slot halves are at at0 and at1, counted in slots
// (heads of 256 dims: a tile is 32 slots, at0). first: of the tile's first position; lo, hi: values of other positions
// are taken as zeros.
template <int D, int T>
struct PagedStage : Stage<D, T, true> {
  using R = Rows<D>;
  using S = Stage<D, T, true>;
  __device__ static uint32_t valid_of(int base, int lo, int hi) {   // of keys base + e, base + 16 + e (e = 0 .. 3)
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int pos = base + (e < 4 ? e : 12 + e);
      m |= pos >= lo && pos < hi ? 1u << e : 0u;
    }
    return m;
  }
  __device__ static uint32_t pair(uint32_t valid, int e) {
    return (valid >> e & 1u ? 0xffffu : 0u) | (valid >> (e + 1) & 1u ? 0xffff0000u : 0u);
  }
  __device__ static uint32_t four(uint32_t valid, int e) {
    uint32_t m = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) m |= valid >> (e + x) & 1u ? 0xffu << (8 * x) : 0u;
    return m;
  }
  // 16-byte pieces tid, tid + 256, .. of the tile's N, half of them at each place
  template <int N>
  __device__ static void load(uint4 (&x)[N / 256], const uint4* c, size_t at0, size_t at1) {
    const int tid = stage_thread<true>();
#pragma unroll
    for (int u = 0; u < N / 256; ++u) {
      if constexpr (D == 256) {
        x[u] = c[at0 * (N / R::TK) + size_t(tid + u * 256)];
      } else if constexpr (N / 2 >= 256) {
        constexpr int HALF = N / 2;
        x[u] = u * 256 < HALF ? c[at0 * (N / R::TK) + size_t(tid + u * 256)] : c[at1 * (N / R::TK) + size_t(tid + u * 256 - HALF)];
      } else {
        x[u] = c[tid < N / 2 ? at0 * (N / R::TK) + size_t(tid) : at1 * (N / R::TK) + size_t(tid - N / 2)];
      }
    }
  }
  __device__ void load_k(const PagedArgs& a, size_t at0, size_t at1) {
    const int tid = stage_thread<true>();
    if constexpr (T == kFp8) {
      load<R::kEntries / 2>(this->k, reinterpret_cast<const uint4*>(a.ck), at0, at1);
    } else {
      const size_t at = D == 256 || tid < 128 ? at0 : at1;
      const int mine = D == 256 ? tid : tid & 127;   // of the half's threads
      this->take(this->k, a.ck + at * (D / 2), mine);
      const uint8_t* s = static_cast<const uint8_t*>(a.ks) + at * (D / 16);
      this->ks = D == 64 ? s[mine] : reinterpret_cast<const uint16_t*>(s)[mine];
    }
  }
  __device__ void load_v(const PagedArgs& a, size_t at0, size_t at1) {
    const int tid = stage_thread<true>(), lane = tid & 63, part = tid >> 6;
    if constexpr (T == kFp8) {
      load<R::kEntries / 2>(this->v, reinterpret_cast<const uint4*>(a.cv), at0, at1);
    } else {
      const size_t at = D == 256 || tid < 128 ? at0 : at1;
      this->take_v(a.cv + at * (D / 2), D == 256 ? part : part & 1, lane);
      const uint2* sv = reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.vs) + at * (D / 16));
      this->vs = sv[(lane >> 4) * (D / 16) + (lane & 15) * (D / 16) / 16];
    }
  }
  __device__ void mask_v(int first, int lo, int hi) {
    if constexpr (T == kFp8) {
#pragma unroll
      for (int u = 0; u < R::PER / 2; ++u) {
        const int x = S::first(u);
        const uint32_t ok = valid_of(first + 32 * (x / (4 * D)) + 4 * (x >> 4 & 3), lo, hi), a = four(ok, 0), b = four(ok, 4);
        uint4& w = this->v[u];
        w.x &= a, w.y &= b, w.z &= a, w.w &= b;
      }
    }   // (NVFP4: as in PagedTile)
  }
  // BF16 tiles straight into LDS: 64 entries a wave's load, a lane's the one that comes to its part of them; and the mask of
  // what a lane loaded, once it is there
  __device__ static void direct(const uint4* c, size_t at0, size_t at1, uint4* to, bool v) {
    const int tid = stage_thread<true>(), half = tid >> 5 & 1, i = tid & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
    for (int u = 0; u < R::PER; ++u) {
      const int row = u * 4 + wave;   // of 64 entries
      // of the 32-slot half: entries of 16-slot blocks and 32-dim chunks, or of 16-dim blocks
      int part, x;
      if (v) {
        const int ks = row % R::KS;
        part = ks >> 1, x = (row / R::KS * 2 + (i >> 4)) * 64 + ((ks & 1) * 2 + half) * 16 + (i & 15);
      } else {
        const int st = row % R::NS;
        part = row / R::NS, x = (i >> 4) * 2 * D + (st >> 1) * 64 + ((st & 1) * 2 + half) * 16 + (i & 15);
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(c + (part ? at1 : at0) * (D / 8) + x),
                                       (__attribute__((address_space(3))) void*)(to + row * 64), 16, 0, 0);
    }
  }
  __device__ static void mask_direct(uint4* lv, int first, int lo, int hi) {
    const int lane = int(threadIdx.x) & 63, wave = stage_thread<true>() >> 6;
#pragma unroll
    for (int u = 0; u < R::PER; ++u) {
      const int row = u * 4 + wave, ks = row % R::KS;
      const uint32_t ok = valid_of(first + 32 * (ks >> 1) + 8 * (ks & 1) + 4 * (lane >> 5), lo, hi);
      uint4& w = lv[row * 64 + lane];
      w.x &= pair(ok, 0), w.y &= pair(ok, 2), w.z &= pair(ok, 4), w.w &= pair(ok, 6);
    }
  }
};

// Heads of 256 dims: chunks of a wave's q operand that are in LDS, shared by the groups, so that nothing in the loop spills (a
// reload from scratch memory waits for the next tile's loads before it: 4 prompts of 150 to 1100 rows over FP8 pages took
// 73 us with two chunks there). Before the loop 2 to 5 registers are spilled, and loaded behind it.
template <int D, int T>
constexpr int kQChunks = D == 256 ? (T == kBf16 ? 2 : 6) : 0;
// LDS of a group: two buffers of a tile, and the scales
template <int D>
constexpr size_t kGroupLds = size_t(Rows<D>::kEntries) * 64 + size_t(Rows<D>::TK) * 16;
template <int D, int T>
constexpr size_t many_lds() {
  const size_t tiles = 2 * kGroupLds<D> + 4096 * kQChunks<D, T>, states = size_t(D) * 512 + 1024, turned = 4 * 32 * (D > 128 ? 528 : D * 4 + 16);
  return tiles > states ? (tiles > turned ? tiles : turned) : states > turned ? states : turned;
}

// The accumulators of the first four waves' 128 q-cols, 32 a wave, times inv as rows of `to`, a lane's at `out` (-1: not
// written). A lane has a q-col's values 512 bytes or more from its neighbour's: they are turned in LDS, a wave its own 32
// rows, four values at a time (one at a time, and by all eight waves, took 9 us of a block of 256 dims, the others' 1.4).
template <int D, int T, class X>
__device__ inline void turned_rows(X* to, const f32x16 (&acc)[Rows<D>::NB], float inv, long long out, uint8_t* smem) {
  using R = Rows<D>;
  constexpr int DP = sizeof(X) == 4 && D > 128 ? 128 : D, PITCH = DP + 16 / int(sizeof(X));   // dims of a pass
  const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6, half = lane >> 5;
  const bool lead = wave < 4;
  X* mine = reinterpret_cast<X*>(smem) + (wave & 3) * 32 * PITCH;
#pragma unroll
  for (int p = 0; p < D; p += DP) {
    if (p) __syncthreads();
    if (lead) {
#pragma unroll
      for (int d = 0; d < R::NB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int v = 32 * d + 8 * j;   // and 4 half
          const int low = Tile<D, T>::dim(v >> 4, v & 15), step = Tile<D, T>::dim(0, 4) - Tile<D, T>::dim(0, 0);
          const int last = Tile<D, T>::dim(v >> 4, (v & 15) + 3);
          if (T != kNvfp4 && (low < p || low >= p + DP)) continue;   // (with half = 1 on the same side)
          if (T == kNvfp4 && (last < p || low >= p + DP)) continue;
          X* row = mine + (lane & 31) * PITCH - p + half * step;
          const float y[4] = {acc[d][4 * j] * inv, acc[d][4 * j + 1] * inv, acc[d][4 * j + 2] * inv, acc[d][4 * j + 3] * inv};
          if constexpr (T == kNvfp4) {
#pragma unroll
            for (int r = 0; r < 4; ++r) row[Tile<D, T>::dim(v >> 4, (v & 15) + r)] = X(y[r]);
          } else {
            put4<D, T>(row, v / 4, y);
          }
        }
    }
    __syncthreads();
    if (!lead) continue;
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
}

template <int D, int T, int MOD>
__device__ inline void many_piece(const PagedArgs& a, const Piece& p, int h, uint8_t* smem, int (&bad_cols)[8]) {
  using R = Rows<D>;
  using X8 = typename OperandOf<T>::type;
  const int tid = stage_thread<true>(), lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 8);
  const bool out_of = p.q.pos < 0;
  // rows of the block and of the wave, and positions that some row of the block sees
  const long long c0 = (long long)p.block * kManyCols, w0 = c0 + wave * 32;
  const int r0 = int(c0 / a.group), r1 = int(min((long long)p.q.n, (c0 + kManyCols + a.group - 1) / a.group)) - 1;
  const int wr0 = int(w0 / a.group), wr1 = int(min((long long)p.q.n, (w0 + 32 + a.group - 1) / a.group)) - 1;
  const int lo = out_of ? 0 : paged_span(a, p.q.pos + r0).lo, hi = out_of ? 0 : min(p.q.pos + r1 + 1, p.cap);
  // positions from lo_top to below hi_low are seen by all of the wave's q-cols, from w_hi on by none
  const bool any = wr0 <= wr1 && !out_of;
  const int lo_top = any ? paged_span(a, p.q.pos + wr1).lo : 0, hi_low = any ? p.q.pos + wr0 + 1 : 0;
  const int w_hi = any ? p.q.pos + wr1 + 1 : 0, w_lo = any ? paged_span(a, p.q.pos + wr0).lo : 0;
  const int tlo = lo / R::TK, tiles = max(0, (hi + R::TK - 1) / R::TK - tlo);
  const int f = tlo + int((long long)tiles * p.split / p.splits), e = tlo + int((long long)tiles * (p.split + 1) / p.splits);

  const int rem = int(w0 - (long long)wr0 * a.group) + (lane & 31), drow = int(uint32_t(rem) * a.group_inv >> 16);
  const int row = wr0 + drow, head = h * a.group + rem - drow * a.group;
  const bool live = row < p.q.n;
  const Span span = live && !out_of ? paged_span(a, p.q.pos + row) : Span{0, 0u, 0};

  float m = -INFINITY, l = 0.f;
  f32x16 acc[R::NB];
#pragma unroll
  for (int d = 0; d < R::NB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;

  uint8_t* const mem = smem + size_t(group) * kGroupLds<D>;
  uint4* const kbuf = reinterpret_cast<uint4*>(mem);             // two buffers each
  uint4* const vbuf = kbuf + 2 * R::kEntries;
  float* const scales = reinterpret_cast<float*>(mem + size_t(R::kEntries) * 64);   // FP8: [2][K, V][TK]

  if (f < e) {
    X8 q[R::NS];
    constexpr int QL = kQChunks<D, T>;
    X8* const ql = reinterpret_cast<X8*>(smem + 2 * kGroupLds<D>) + wave * 64 + lane;
    bf16x8 x[R::NS];
    const size_t q_at = live ? size_t(p.q.row0 + row) * size_t(a.ldq) + size_t(head) * D + size_t(8 * half) : size_t(8 * half);
    row_chunks(a.q, a.bf16, live, [&](int c) { return q_at + size_t(16 * c); }, x);
    PagedStage<D, T> stage;
    constexpr bool kDirect = T == kBf16;
    // the pages of the next 64 tiles' 32-slot halves, one a lane
    int pages = -1, from = f;
    constexpr int HALVES = R::TK / 32;
    auto load_pages = [&](int t) {
      from = t;
      const int pos = t * R::TK + 32 * lane;
      pages = pos < hi ? page_of(a.s, p.seq, pos) : -1;
    };
    auto page_at = [&](int t, int x) { return __builtin_amdgcn_readlane(pages, (t - from) * HALVES + x); };
    const int t0 = f + group;   // the group's tiles: t0, t0 + 2, ..
    load_pages(f);
    int page0 = page_at(t0, 0), page1 = HALVES == 2 ? page_at(t0, 1) : page0;
    float ks = 0.f, vs = 0.f;
    auto buffer = [&](int t) { return ((t - t0) >> 1 & 1) * R::kEntries; };
    auto load = [&](int t) {
      if (kDirect && t >= e) return;
      t = min(t, e - 1);   // past the last: loaded again, and not used
      const size_t at0 = place_of(a, page0, h, t * R::TK), at1 = HALVES == 2 ? place_of(a, page1, h, t * R::TK + 32) : at0;
      if constexpr (kDirect) {
        stage.direct(reinterpret_cast<const uint4*>(a.ck), at0, at1, kbuf + buffer(t), false);
        stage.direct(reinterpret_cast<const uint4*>(a.cv), at0, at1, vbuf + buffer(t), true);
      } else {
        stage.load_k(a, at0, at1);
        stage.load_v(a, at0, at1);
      }
      if constexpr (T == kFp8) {
        const size_t at = (tid & 32) && HALVES == 2 ? at1 : at0;
        if (tid < R::TK) {
          ks = static_cast<const float*>(a.ks)[at + size_t(tid & 31)];
          vs = static_cast<const float*>(a.vs)[at + size_t(tid & 31)];
        }
      }
    };
    auto store = [&](int t) {
      const int buf = (t - t0) >> 1 & 1, first = t * R::TK;
      const bool partial = first < lo || first + R::TK > hi;
      if constexpr (kDirect) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the tile's loads into LDS, before the barrier behind
        if (t < e && partial) stage.mask_direct(vbuf + buf * R::kEntries, first, lo, hi);
      } else {
        if (partial) stage.mask_v(first, lo, hi);
        stage.store_k(kbuf + buf * R::kEntries);
        stage.store_v(vbuf + buf * R::kEntries);
      }
      if constexpr (T == kFp8) {   // a key whose V scale is not finite is NaN itself, and the scale zero
        if (tid < R::TK) {
          scales[buf * 2 * R::TK + tid] = not_finite(vs) ? NAN : ks;
          scales[buf * 2 * R::TK + R::TK + tid] = not_finite(vs) ? 0.f : vs;
        }
      }
    };
    load(t0);
    if (a.scale < 0.f) {
#pragma unroll
      for (int c = 0; c < R::NS; ++c) x[c] = -x[c];
    }
    const int ex = to_operand<T != kBf16>(x, q, [](float y) { return xor32_max(y); });
    const Score sc = paged_score(a, T == kNvfp4 ? a.kglobal : 1.f, ex);
#pragma unroll
    for (int c = 0; c < QL; ++c)
      if (!group) ql[c * 256] = q[R::NS - QL + c];
    store(t0);
    __syncthreads();
    for (int t = t0; t < e + group; t += 2) {   // (both groups as often, for the barriers)
      const bool lost0 = page0 < 0, lost1 = page1 < 0;
      if (t + 2 < e) {
        if ((t + 2 - from) * HALVES + HALVES > 64) load_pages(t + 2);
        page0 = page_at(t + 2, 0), page1 = HALVES == 2 ? page_at(t + 2, 1) : page0;
      }
      load(t + 2);
      const int first = t * R::TK;
      if (t < e && first < w_hi && first + R::TK > w_lo) {   // (else none of the wave's q-cols sees the tile)
        const X8* lk = reinterpret_cast<const X8*>(kbuf + buffer(t));
        const X8* lv = reinterpret_cast<const X8*>(vbuf + buffer(t));
        const float4* lf4 = reinterpret_cast<const float4*>(scales + ((t - t0) >> 1 & 1) * 2 * R::TK) + half;
        f32x16 s[R::KB];
#pragma unroll
        for (int b = 0; b < R::KB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
#pragma unroll
        for (int c = 0; c < R::NS; ++c)
#pragma unroll
          for (int b = 0; b < R::KB; ++b) s[b] = mfma32(lk[(b * R::NS + c) * 64 + lane], c < R::NS - QL ? q[c] : ql[(c - R::NS + QL) * 256], s[b]);
        // scores begun; row 8 j + r' of block b (r = 4 j + r') is key 32 b + 8 j + 4 half + r'
        float y[R::KB][16];
#pragma unroll
        for (int b = 0; b < R::KB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float k4[4] = {1.f, 1.f, 1.f, 1.f};
            if constexpr (T == kFp8) {
              const float4 z = lf4[b * 8 + j * 2];
              k4[0] = z.x, k4[1] = z.y, k4[2] = z.z, k4[3] = z.w;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) y[b][4 * j + r] = begin<MOD>(sc, T == kFp8 ? s[b][4 * j + r] * k4[r] : s[b][4 * j + r], 0);
          }
        if (first < lo_top || first + R::TK > hi_low) {
          asm volatile("");   // (kept behind the branch: asked for every tile, masks are a fifth of its vector operations)
          const int at = first + 4 * half - span.lo;
#pragma unroll
          for (int b = 0; b < R::KB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (uint32_t(at + 32 * b + 8 * (r >> 2) + (r & 3)) >= span.len) y[b][r] = masked<MOD>();
        }
        if (lost0 || lost1) {
#pragma unroll
          for (int b = 0; b < R::KB; ++b) {
            const int from32 = max(first + 32 * b, span.lo), to = min(first + 32 * b + 32, span.lo + int(span.len));
            if ((b ? lost1 : lost0) && from32 < to) l = NAN;
          }
        }
        float mx = masked<MOD>();
#pragma unroll
        for (int b = 0; b < R::KB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = best<MOD>(mx, y[b][r]);
        mx = xor32_max(finish<MOD>(sc, mx, 0.f));
        float sc_f = sc.f;   // (1: the scores have been multiplied)
        if constexpr (MOD == 0) {
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
        const float ref = (m == -INFINITY ? 0.f : m) - kUp;
        float sum = 0.f;
        X8 w[R::KS];
#pragma unroll
        for (int b = 0; b < R::KB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float v4[4] = {1.f, 1.f, 1.f, 1.f};
            if constexpr (T == kFp8) {
              const float4 z = lf4[R::TK / 4 + b * 8 + j * 2];
              v4[0] = z.x, v4[1] = z.y, v4[2] = z.z, v4[3] = z.w;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float o = __builtin_amdgcn_exp2f(MOD ? finish<MOD>(sc, y[b][4 * j + r], ref) : fmaf(y[b][4 * j + r], sc_f, -ref));
              sum += o;
              if constexpr (T == kFp8) o *= v4[r];
              w[2 * b + (j & 1)][(j >> 1) * 4 + r] = o;
            }
          }
        l += sum;
#pragma unroll
        for (int k = 0; k < R::KS; ++k)
#pragma unroll
          for (int d = 0; d < R::NB; ++d) acc[d] = mfma32(lv[(d * R::KS + k) * 64 + lane], w[k], acc[d]);
      }
      store(t + 2);
      __syncthreads();
    }
  }
  if (span.len && span.t >= p.cap) l = NAN;
  if (T == kNvfp4 && a.vglobal != 1.f) {
#pragma unroll
    for (int d = 0; d < R::NB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= a.vglobal;
  }
  l = xor32_sum(l);
  const int col = wave * 32 + (lane & 31);
  {   // the second group's state into the first's
    float4* part = reinterpret_cast<float4*>(smem) + wave * 64 + lane;   // [product][row / 4][wave][lane]
    float2* ml = reinterpret_cast<float2*>(smem + size_t(D) * 128 * 4) + col;
    if (group) {
#pragma unroll
      for (int d = 0; d < R::NB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          part[(4 * d + j) * 256] = make_float4(acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]);
      if (half == 0) *ml = make_float2(m, l);
    }
    __syncthreads();
    if (!group) {
      const float2 o = *ml;
      const float to = fmaxf(m, o.x), ref = to == -INFINITY ? 0.f : to;
      const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(o.x - ref);
      m = to;
      l = l * f0 + o.y * f1;
#pragma unroll
      for (int d = 0; d < R::NB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 u = part[(4 * d + j) * 256];
          acc[d][4 * j] = acc[d][4 * j] * f0 + u.x * f1, acc[d][4 * j + 1] = acc[d][4 * j + 1] * f0 + u.y * f1;
          acc[d][4 * j + 2] = acc[d][4 * j + 2] * f0 + u.z * f1, acc[d][4 * j + 3] = acc[d][4 * j + 3] * f0 + u.w * f1;
        }
    }
  }
  const bool mine = live && !group;   // to write
  if (mine && half == 0 && p.split == 0 && h == 0)
    a.info[size_t(p.q.row0 + row) * size_t(a.group) + size_t(head)] = make_int4(int(p.rec), p.blocks << 1 | 1, p.splits << 8 | col, p.seq);
  if (p.splits > 1) {
    if (!mine) return;
    const size_t rec = size_t(p.rec) * size_t(a.kv_heads) + size_t(h * kManyCols + col);
#pragma unroll
    for (int d = 0; d < R::NB; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(a.acc + rec * D + size_t(32 * d + 8 * j + 4 * half)) =
            f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]};
    if (half == 0) a.ml[rec * 2] = m, a.ml[rec * 2 + 1] = l;
    return;
  }
  const float inv = l == 0.f ? (out_of ? 0.f : NAN) : 1.f / l;
  bool bad = false;
#pragma unroll
  for (int d = 0; d < R::NB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad |= mine && not_finite(acc[d][r]);
  const long long out = mine ? (long long)((size_t(p.q.row0 + row) * size_t(a.heads) + size_t(head)) * D) : -1;
  const uint64_t again = __ballot(bad && !not_finite(l));
  if (lane == 0 && !group) bad_cols[wave] = int(uint32_t(again) | uint32_t(again >> 32));
  __syncthreads();   // the states' place
  if (a.bf16)
    turned_rows<D, T>(static_cast<__bf16*>(a.out), acc, inv, out, smem);
  else
    turned_rows<D, T>(static_cast<float*>(a.out), acc, inv, out, smem);
  for (int w = 0; w < 4; ++w)
    for (uint32_t bits = uint32_t(bad_cols[w]); bits; bits &= bits - 1) {
      const long long c = c0 + w * 32 + __builtin_ctz(bits);
      const int r = int(c / a.group);
      paged_slow_col<D, T>(a, p.seq, p.q.row0 + r, p.q.pos + r, h * a.group + int(c - (long long)r * a.group), reinterpret_cast<float*>(smem));
    }
}

template <int D, int QB, int T, bool MANY>
constexpr size_t paged_lds() {
  const size_t few = few_lds<D, QB>(), many = MANY ? many_lds<D, T>() : 0;
  return few > many ? few : many;
}

// MANY: some sequence can have more q-cols than one block of QB * 16.
template <int D, int QB, int T, int MOD, bool MANY>
__global__ void __launch_bounds__(MANY ? 512 : 256, !MANY && QB * D > 256 ? 1 : 2) paged_attn_kernel(PagedArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ uint32_t again;
  __shared__ int bad_cols[8];
  const int h = int(blockIdx.x) % a.kv_heads, task = int(blockIdx.x) / a.kv_heads;
  Piece p;
  if (!piece_of<MANY>(a, task, p)) return;   // (the whole work-group: every wave finds the same)
  if (p.splits > 1 && p.rec + (p.many ? kManyCols : a.cols) > a.records) return;   // (only where starts decrease)
  if constexpr (MANY) {
    if (p.many) {
      many_piece<D, T, MOD>(a, p, h, smem, bad_cols);
      return;
    }
  }
  if (threadIdx.x == 0) again = 0;
  few_piece<D, QB, T, MOD, MANY ? 8 : 4>(a, p, h, smem, again);
}

// ---------------------------------------------------------------------------------------------------- merge

// Up to this many q-cols have a work-group each (they have many records then), more a wave, and from kMergeMost on a wave has
// several, most of which have none: where every block of 30640 q-cols was one part, asking a wave each took 9.6 us.
constexpr int kMergeFew = 1024, kMergeMost = 8192;

// Where a q-col's records are; none where its block was one part, or its row is no sequence's.
__device__ inline int4 merge_info(const PagedArgs& a, int id, int total) {
  int4 info = make_int4(0, 0, 0, 0);
  if (id >= total) return info;
  const int row = id / a.heads, head = id - row * a.heads;
  if (a.s.starts && (row < a.s.starts[0] || row >= a.s.starts[a.s.n_seqs])) return info;
  info = a.info[size_t(row) * size_t(a.group) + size_t(head % a.group)];
  const int splits = info.z >> 8, cols = info.y & 1 ? kManyCols : a.cols;
  const long long last = info.x + (splits - 1LL) * (info.y >> 1) * cols + cols;
  // (where starts decrease, a row's place may be of another call)
  if (splits <= 1 || info.x < 0 || info.y < 0 || last > a.records || (info.z & 0xff) >= cols ||
      uint32_t(info.w) >= uint32_t(a.s.n_seqs))
    info.z = 0;
  return info;
}

// One q-col by W waves: D / 4 lanes to a record's accumulator, W * 256 / D records at once, B of them a lane in flight.
// Returns whether it has to be computed again key by key.
template <int D, int T, int W>
__device__ inline bool merge_col(const PagedArgs& a, int id, int4 info, float4* part, float* all_m, float* all_l) {
  constexpr int L = D / 4, G = W * 64 / L, B = 8;
  const int tid = int(threadIdx.x) & (64 * W - 1), wave = tid >> 6, x = tid % L, grp = tid / L;
  const int row = id / a.heads, head = id - row * a.heads, h = head / a.group;
  // (a part's records are those of all blocks behind the one before)
  const int splits = info.z >> 8, cols = info.y & 1 ? kManyCols : a.cols;
  const size_t stride = size_t(info.y >> 1) * size_t(cols) * size_t(a.kv_heads);
  const size_t rec0 = size_t(info.x) * size_t(a.kv_heads) + size_t(h * cols + (info.z & 0xff));
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + rec0;
  const float* acc = a.acc + rec0 * D + size_t(4 * x);
  float4 v[B];
  float2 w[B];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int s = s0 + k * G;
      w[k] = s < splits ? ml[size_t(s) * stride] : make_float2(-INFINITY, 0.f);
      v[k] = s < splits ? *reinterpret_cast<const float4*>(acc + size_t(s) * stride * D) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  load(grp);
  const int rows = seq_at(a.s, info.w).n;
  float m = -INFINITY;
  for (int s = tid; s < splits; s += 64 * W) m = fmaxf(m, ml[size_t(s) * stride].x);
  m = wave_max(m);
  if constexpr (W == 4) {
    if ((tid & 63) == 0) all_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(all_m[0], all_m[1]), fmaxf(all_m[2], all_m[3]));
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = grp; s0 < splits; s0 += B * G) {
    if (s0 != grp) load(s0);
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const float f = __builtin_amdgcn_exp2f(w[k].x - ref);
      // (a NaN stays one, of a key without a page or a value, also times zero: a row is the same however its keys are cut; one
      // of a part that the row sees nothing of is taken back by the computation key by key)
      l += w[k].y * f;
      y.x += v[k].x * f, y.y += v[k].y * f, y.z += v[k].z * f, y.w += v[k].w * f;
    }
  }
  l = wave_sum(x == 0 ? l : 0.f);
  if constexpr (W == 4) {
    part[tid] = y;
    if ((tid & 63) == 0) all_l[wave] = l;
    __syncthreads();
    l = all_l[0] + all_l[1] + all_l[2] + all_l[3];
    if (grp == 0) {
      y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < G; ++s) {
        const float4 u = part[s * L + x];
        y.x += u.x, y.y += u.y, y.z += u.z, y.w += u.w;
      }
    }
  } else {
    auto join = [&](float& c) {
      if constexpr (L <= 16) c = xor16_sum(c);
      if constexpr (L <= 32) c = xor32_sum(c);
    };
    join(y.x), join(y.y), join(y.z), join(y.w);
  }
  if (grp != 0) return false;
  const float inv = l == 0.f ? NAN : 1.f / l;
  put4<D, T>(a, size_t(id) * D, x, {y.x * inv, y.y * inv, y.z * inv, y.w * inv});
  return rows > 1 && !not_finite(l) && (not_finite(y.x) || not_finite(y.y) || not_finite(y.z) || not_finite(y.w));
}

// W waves a q-col (4), or N q-cols a wave (W = 1).
template <int D, int T, int W, int N>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedArgs a, int total) {
  constexpr int PER = W == 4 ? 1 : 4 * N;   // q-cols of a work-group
  __shared__ float4 part[W == 4 ? 256 : 1];
  __shared__ float slow[784 + D], all_m[4], all_l[4];
  __shared__ uint32_t again;
  if (threadIdx.x == 0) again = 0;
  const int lane = int(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), id0 = int(blockIdx.x) * PER;
  uint32_t bad = 0;   // of the work-group's q-cols
  bool any = false;
  if constexpr (W == 4) {
    const int4 info = merge_info(a, id0, total);
    if (info.z == 0) return;   // (the whole work-group)
    any = true;
    bad = merge_col<D, T, W>(a, id0, info, part, all_m, all_l);
  } else {
    const int4 mine = lane < N ? merge_info(a, id0 + wave * N + lane, total) : make_int4(0, 0, 0, 0);
    for (uint64_t bits = __ballot(mine.z != 0); bits; bits &= bits - 1) {
      const int k = __builtin_ctzll(bits);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, k); };
      if (merge_col<D, T, W>(a, id0 + wave * N + k, make_int4(of(mine.x), of(mine.y), of(mine.z), of(mine.w)), part, all_m, all_l))
        bad |= 1u << (wave * N + k);
      any = true;
    }
  }
  if (!__syncthreads_or(any && bad)) return;
  if (bad) atomicOr(&again, bad);
  __syncthreads();
  for (uint32_t bits = again; bits; bits &= bits - 1) {
    const int id = id0 + __builtin_ctz(bits), row = id / a.heads, head = id - row * a.heads;
    const int seq = a.info[size_t(row) * size_t(a.group) + size_t(head % a.group)].w;
    const Seq q = seq_at(a.s, seq);
    paged_slow_col<D, T>(a, seq, row, q.pos + row - q.row0, head, slow);
  }
}

// ---------------------------------------------------------------------------------------------------- launches

template <int D, int T, int MOD>
void paged_go(const PagedAttnCall& c, const PagedPlan& p, const PagedArgs& a, hipStream_t stream, const PagedTimed& timed) {
  timed([&] {
    const dim3 grid{unsigned(p.tasks) * unsigned(a.kv_heads)};
    auto go = [&](auto kernel, size_t lds) {
      allow_lds(reinterpret_cast<const void*>(kernel), lds);
      paged_queue(kernel, grid, p.many ? 512 : 256, lds, stream, a);
    };
    if (p.cols == 32 && !p.many)
      go(&paged_attn_kernel<D, 2, T, MOD, false>, paged_lds<D, 2, T, false>());
    else if (!p.many)
      go(&paged_attn_kernel<D, 1, T, MOD, false>, paged_lds<D, 1, T, false>());
    else if (p.cols == 16)
      go(&paged_attn_kernel<D, 1, T, MOD, true>, paged_lds<D, 1, T, true>());
    else if constexpr (D < 256)
      go(&paged_attn_kernel<D, 2, T, MOD, true>, paged_lds<D, 2, T, true>());
    else
      fail("paged_attention: a plan of 32 q-cols for heads of 256 dims");
    return c.named ? strf("paged_attn_kernel<%d, %d, %d, %d, %d>", D, p.cols / 16, T, MOD, int(p.many)) : std::string();
  });
  if (p.records > 0) timed([&] {
    const int total = c.seqs.n_rows * c.heads, n = total <= kMergeFew ? 0 : total <= kMergeMost ? 1 : 4;
    auto go = [&](auto kernel, int cols) {
      paged_queue(kernel, dim3(unsigned((total + cols - 1) / cols)), 256, 0, stream, a, total);
    };
    if (n == 0)
      go(&paged_merge_kernel<D, T, 4, 1>, 1);
    else if (n == 1)
      go(&paged_merge_kernel<D, T, 1, 1>, 4);
    else
      go(&paged_merge_kernel<D, T, 1, 4>, 16);
    return c.named ? strf("paged_merge_kernel<%d, %d, %d, %d>", D, T, n == 0 ? 4 : 1, n > 1 ? n : 1) : std::string();
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
