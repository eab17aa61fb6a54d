// Paged KV caches: many sequences' keys and values in pages of one pool (rows: paged_rows.hip; attention:
// paged_attention.hip, and its kernels in paged_attention_kernels.hpp).
//
// Page p holds `size` positions of every KV head, in the layouts of a linear cache (attention.hpp, kv4.hpp): the pool is laid
// out as one of pages * kv_heads heads of `size` slots each, of which page p has heads p * kv_heads .. +kv_heads. `size` is a
// power of two and a multiple of 32, so that a tile of 32 slots is always one page's and its place one addition away from it.
//
// What a call's rows belong to is read on the device, by every kernel for itself: positions, first rows and pages change from
// step to step while a captured graph, and a plan made on the host, stay. So grids and scratch are sized by the number of rows
// and sequences alone, and a work-group finds its piece of work by a prefix sum over the sequences (find_task).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <functional>
#include <string>

#include "common.hpp"

namespace xtg::hip {

struct DevPaged {
  int kv_heads = 0, head_dim = 0;
  int pages = 0, size = 0, shift = 0;   // positions of a page: size = 2^shift
  int type = 0;                         // XTG_KV_*
  void *k = nullptr, *v = nullptr, *ks = nullptr, *vs = nullptr;   // codes or values, and scales (FP32, E4M3)
  float kglobal = 1.f, vglobal = 1.f;   // NVFP4: what every scale is multiplied by, powers of two
  bool written = false;
  size_t elems() const { return size_t(pages) * size_t(size) * size_t(kv_heads) * size_t(head_dim); }
  size_t data_bytes() const { return type == 2 ? elems() / 2 : elems() * (type == 1 ? 1 : 2); }
  size_t scale_bytes() const { return type == 2 ? elems() / 16 : type == 1 ? elems() / size_t(head_dim) * sizeof(float) : 0; }
};

// The sequences of a call, as the kernels take them (the fields of xtg_paged_rows).
struct Seqs {
  const int* pos;
  const int* starts;   // NULL: row s is sequence s's
  const int* table;    // [n_seqs][max_pages]
  int n_seqs, n_rows, max_pages;
  int pages, shift;    // the pool's
};

// No position from here on has a page, and a call has fewer rows: sums of the two fit an int.
constexpr int kMostPositions = 1 << 30;

// Sequences of a call, at most. Every work-group looks for its piece among all of them, so that a call takes a time that grows
// with their square beside its own work (one row each over 60 positions of 8 KV heads of 128 dims: 1024 sequences 0.18 ms, with
// starts 0.83; 4096 2.0 and 11; 16384 29 and 170): 2^20 would take the GPU minutes.
constexpr int kMostSeqs = 1 << 14;

// A sequence's rows in the call, row0 .. row0 + n - 1, at positions pos .. pos + n - 1 (pos < 0: left out). Starts out of the
// call's rows, or that decrease, are clamped: what they name is still in range.
struct Seq {
  int pos, row0, n;
};
__host__ __device__ inline Seq seq_at(const Seqs& a, int s) {
  const int pos = a.pos[s];
  Seq q = {pos < kMostPositions ? pos : kMostPositions, s, 1};
  if (a.starts) {
    const int r0 = a.starts[s], r1 = a.starts[s + 1], end = r1 < a.n_rows ? r1 : a.n_rows;
    q.row0 = r0 < 0 ? 0 : r0 < a.n_rows ? r0 : a.n_rows;
    q.n = end > q.row0 ? end - q.row0 : 0;
  }
  return q;
}

// The page of position p >= 0 of sequence s, or -1 where its table or the pool has none.
__host__ __device__ inline int page_of(const Seqs& a, int s, int p) {
  const int j = p >> a.shift;
  if (uint32_t(j) >= uint32_t(a.max_pages)) return -1;
  const int page = a.table[size_t(s) * size_t(a.max_pages) + size_t(j)];
  return uint32_t(page) < uint32_t(a.pages) ? page : -1;
}

struct PagedAppend {
  int heads;
  const void *q, *k, *v;
  void* q_out;
  long long ldq, ldk, ldv;   // elements from a row to the next
  int x_dtype, norm;
  const double* freq;        // quarter turns a position of each pair (Backend::turn_freq), NULL: no rotation
  const float* qscale;
};
// A launch's name is made where it is asked for (`named`): making it takes 0.1 to 0.2 us, a call 5.
std::string launch_paged_append(const DevPaged& c, const Seqs& s, const PagedAppend& a, hipStream_t stream, bool named);
// Rows into k, v [n_rows][kv_heads][head_dim]; zeros where there is no page, nothing behind the last sequence's rows.
std::string launch_paged_read(const DevPaged& c, const Seqs& s, void* k, void* v, bool bf16, hipStream_t stream, bool named);

struct PagedAttnCall {
  const DevPaged* cache;
  Seqs seqs;
  int heads;
  const void* q;
  void* out;
  long long ldq;
  int x_dtype, window;
  float scale, softcap;
  bool named;
};

// How an attention call is cut up. A q-col is a (row, q head of a KV head). A sequence of up to `cols` of them (a decode or
// verify step) is one block of `cols`, whose work-groups' waves take tiles of their own; one of more goes in blocks of
// kManyCols, whose work-groups' waves share tiles. Of a block's keys a work-group takes one of several parts for one KV head,
// about `budget` work-groups a KV head in all, and leaves a record (accumulator, maximum, sum) for each q-col where there is
// more than one part.
struct PagedPlan {
  int cols = 16, budget = 1;
  bool many = false;             // a sequence of the call can have more than `cols` q-cols
  int tasks = 1;                 // work-groups a KV head, at most
  int records = 0;               // q-cols of a KV head with records, at most: those of its work-groups with more than one part
  size_t acc_bytes = 0, ml_bytes = 0, info_bytes = 0;
  size_t bytes() const { return acc_bytes + ml_bytes + info_bytes; }
};
PagedPlan paged_plan(const PagedAttnCall& a, int cus);

constexpr int kManyCols = 128;
// Fewest tiles of a part: one a wave; and of a block of many q-cols (300 rows of 256 dims over 3000 positions: 57 us with 32,
// 43 with 16 or 12, 46 with 8).
constexpr int kFewLeast = 4, kManyLeast = 16;

struct PagedArgs {
  static constexpr bool kStream = true;   // a sequence of one block: its tiles are read once
  Seqs s;
  const void* q;
  void* out;
  const uint8_t *ck, *cv;
  const void *ks, *vs;
  float *acc, *ml;               // records: of a piece, [KV head][its q-cols][d], [..][2]
  int4* info;                    // of each q-col [row][q head of its KV head]: its piece's place, the blocks of its sequence
                                 // << 1 | many, parts << 8 | col, sequence
  long long ldq;
  int heads, kv_heads, group, cols, budget, records, window, bf16;
  uint32_t group_inv;            // ceil(2^16 / group)
  float factor;                  // what a product q.k is multiplied by in base-2 units: factor * 2^factor_exp
  int factor_exp;
  float scale, kglobal, vglobal, softcap;
};

// What a sequence's rows of a call ask for: blocks of q-cols, and tiles lo .. lo + tiles - 1 that they see (all blocks'). A
// sequence that is left out has its rows' blocks, and no tile.
struct Extent {
  Seq q;
  bool many;
  int blocks, tiles, lo;
  __host__ __device__ int cols(const PagedArgs& a) const { return many ? kManyCols : a.cols; }
};
__host__ __device__ inline Extent extent(const PagedArgs& a, int s) {
  Extent x = {seq_at(a.s, s), false, 0, 0, 0};
  const long long cols = (long long)x.q.n * a.group;
  x.many = cols > a.cols;
  x.blocks = int((cols + x.cols(a) - 1) / x.cols(a));
  if (x.q.pos >= 0 && x.q.n > 0) {
    const int cap = a.s.max_pages << a.s.shift, end = x.q.pos + x.q.n < cap ? x.q.pos + x.q.n : cap;
    const int lo = a.window > 0 && x.q.pos >= a.window ? x.q.pos - a.window + 1 : 0;
    x.lo = lo >> 5;
    x.tiles = ((end + 31) >> 5) - x.lo;
    if (x.tiles < 0) x.tiles = 0;
  }
  return x;
}
// The parts of a block's tiles, `chunk` tiles each; of many q-cols about as many.
__host__ __device__ inline int parts_of(const Extent& x, int chunk) {
  if (x.many && chunk < kManyLeast) chunk = kManyLeast;
  const int n = (x.tiles + (x.many ? chunk / 2 : chunk - 1)) / chunk;
  return n > 1 ? n : 1;
}
// The tiles of a part: an even share of all blocks' tiles `total` for each of `budget` work-groups, then, as begun parts
// make more than that (`tasks`), a larger one, unless the blocks alone are as many. Returns whether it changed.
// One long sequence takes half as many work-groups, one a CU: more than 32 records of a q-col cost the merge more than the
// second one a CU brings (one token over 32768 BF16 positions of 8 KV heads of 128 dims: 32.2 -> 30.0 us).
__host__ __device__ inline int first_chunk(const PagedArgs& a, float total, int blocks) {
  const float share = total / float(blocks * 32LL < a.budget ? (a.budget + 1) / 2 : a.budget);
  const int chunk = share < 1e9f ? int(share) + 1 : 1000000000;
  return chunk < kFewLeast ? kFewLeast : chunk;
}
__host__ __device__ inline bool next_chunk(const PagedArgs& a, int& chunk, int tasks, int blocks) {
  if (tasks <= a.budget || blocks >= a.budget || chunk >= 1 << 24) return false;
  chunk += int(float(chunk) * float(tasks - a.budget) / float(a.budget)) + 1;
  return true;
}
constexpr int kChunkSteps = 3;

// A launch whose error is its own return value: asking for the last error after one takes the host another 0.9 us, a quarter
// of what the launch does.
// The grid's threads are a 32-bit number.
template <class... A>
void paged_queue(void (*kernel)(A...), dim3 grid, unsigned threads, size_t lds, hipStream_t stream, A... args) {
  XTG_CHECK((unsigned long long)grid.x * threads < (1ULL << 32), "a launch of %u work-groups of %u threads: a call of so many rows and sequences",
            grid.x, threads);
  void* list[] = {&args...};
  HIP_CHECK(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), list, lds, stream));
}

using PagedTimed = std::function<void(const std::function<std::string()>&)>;
void launch_paged_attn(const PagedAttnCall& a, const PagedPlan& p, void* scratch, hipStream_t stream, const PagedTimed& timed);

// The launches for heads of D dims (64, 128, 256).
template <int D>
void paged_launch(const PagedAttnCall& c, const PagedPlan& p, const PagedArgs& a, hipStream_t stream, const PagedTimed& timed);

}  // namespace xtg::hip
