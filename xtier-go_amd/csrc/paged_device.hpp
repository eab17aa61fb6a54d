// Device helpers of the paged caches' kernels: which piece of a call's work is a work-group's.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "paged.hpp"
#include "rowops.hpp"

namespace xtg::hip {

// Sum of v over lanes 0 .. l of a wave, in lane l.
__device__ inline int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // rows of 16: from 1, 2, 4 and 8 lanes below
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // the last lane of rows 0 and 2 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // lane 31 to rows 2 and 3
  return v;
}

// Sum of v over a wave, in every lane.
__device__ inline int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Piece `task` of the sequences' pieces laid end to end, count(s) of sequence s: its sequence and its number there, by a wave
// (every lane gets both); false past the last.
template <class C>
__device__ inline bool find_task(int n_seqs, int task, C&& count, int& seq, int& at) {
  int before = 0;
  for (int base = 0; base < n_seqs; base += 64) {
    const int lane = int(__lane_id()), s = base + lane;
    const int c = s < n_seqs ? count(s) : 0, sum = wave_scan(c);
    const uint64_t hit = __ballot(uint32_t(task - before - (sum - c)) < uint32_t(c));
    if (hit) {
      const int l = __builtin_ctzll(hit);
      seq = base + l;
      at = task - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(c, l));
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

}  // namespace xtg::hip
