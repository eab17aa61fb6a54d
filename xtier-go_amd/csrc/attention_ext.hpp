// Attention with capped, biased and masked scores over a cache of any dtype (attention_ext.hip).
#pragma once

#include <hip/hip_runtime.h>

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

std::string launch_attn_ext(const ExtCall& a, hipStream_t stream);

}  // namespace xtg::hip
