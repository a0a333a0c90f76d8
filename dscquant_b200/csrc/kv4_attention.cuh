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

// One warp per (row, head): a lane holds D/32 elements, one key at a time with a running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attention_rows(const Kv4AttnParams p) {
  constexpr int E = D / 32;  // elements per lane: 2 or 4, consecutive
  const int lane = threadIdx.x & 31;
  const int64_t item = blockIdx.x * 4ll + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(p.T) * p.hq) return;
  const int t = static_cast<int>(item / p.hq), h = static_cast<int>(item % p.hq);
  const Kv4Batch& b = p.b;
  float o[E], qf[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    o[e] = 0.f;
    qf[e] = to_float<T>(static_cast<const T*>(p.q)[t * p.q_t + h * p.q_h + lane * E + e]) * p.scale_log2;
  }
  float m = -INFINITY, l = 0.f;
  int s = -1;
  int64_t keys = 0;
  if (b.B > 0) {
    s = kv4_find_seq(b.q_start, b.B, t);
    const int q0 = b.q_start[s], q1 = b.q_start[s + 1];
    if (t >= q0 && t < q1) keys = static_cast<int64_t>(b.lengths[s]) - (q1 - static_cast<int64_t>(t)) + 1;
    const int64_t cap = static_cast<int64_t>(b.P) << b.ps_log2;
    if (keys > cap) {
      if (lane == 0) raise_status(kStatusBadIndex);
      keys = cap;
    }
  }
  const int hk = h / p.group;
  for (int64_t j = 0; j < keys; ++j) {
    const int64_t page = b.table[s * b.ld_table + (j >> b.ps_log2)];
    if (page < 0 || page >= b.pages) {
      if (lane == 0) raise_status(kStatusBadIndex);
      continue;
    }
    const int64_t row = ((page * b.hk + hk) << b.ps_log2) + (j & ((1 << b.ps_log2) - 1));
    const float2 ka = unpack2<T>(b.ka[row]), va = unpack2<T>(b.va[row]);
    uint32_t kw, vw;
    if constexpr (E == 4) {
      kw = reinterpret_cast<const uint16_t*>(b.kc + row * (D / 2))[lane];
      vw = reinterpret_cast<const uint16_t*>(b.vc + row * (D / 2))[lane];
    } else {
      kw = b.kc[row * (D / 2) + lane];
      vw = b.vc[row * (D / 2) + lane];
    }
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) d = fmaf(qf[e], fmaf(static_cast<float>((kw >> (4 * e)) & 15u), ka.x, ka.y), d);
#pragma unroll
    for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    const float nm = fmaxf(m, d);
    const float f = exp2f(m - nm), w = exp2f(d - nm);
    m = nm;
    l = fmaf(l, f, w);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], f, w * fmaf(static_cast<float>((vw >> (4 * e)) & 15u), va.x, va.y));
  }
  T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(t) * p.hq + h) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_float<T>(l == 0.f ? 0.f : o[e] / l);
}

}  // namespace dscq
