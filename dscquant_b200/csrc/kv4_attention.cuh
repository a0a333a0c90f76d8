// Causal attention over the 4-bit paged cache (kv4.cuh): for row t of sequence b at position p,
//   s_j = scale * q . k_j,  j = 0 .. p;   out = sum_j softmax(s)_j v_j,   k_j, v_j = code * step + low.
// Rows of no sequence and rows that see no key are zero.
#pragma once
#include "kv4.cuh"

namespace dscq {

struct Kv4AttnParams {
  Kv4Batch b;
  const void* q;
  void* out;  // [T, hq, D] contiguous
  int64_t q_t, q_h;
  int T, hq, group;
  float scale_log2;  // scale * log2(e)
};

}  // namespace dscq
