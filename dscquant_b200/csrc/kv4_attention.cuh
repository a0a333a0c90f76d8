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
  uint32_t group_mul, group_shift;  // r / group by multiplication (row_token)
  float scale_log2;                 // scale * log2(e)

  void set_group(int g) {
    group = g;
    group_shift = 0;
    while ((1u << group_shift) < static_cast<uint32_t>(g)) ++group_shift;
    group_mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << group_shift) - g)) / g + 1);
  }
  // r / group for 0 <= r < 2^31: (r + floor(r m / 2^32)) >> shift with m = 2^32 (2^shift - group) / group + 1.
  __device__ __forceinline__ int row_token(int r) const {
    const uint32_t u = static_cast<uint32_t>(r);
    return static_cast<int>((__umulhi(u, group_mul) + u) >> group_shift);
  }
};

}  // namespace dscq
