// Log probabilities of given tokens, entropy and the top alternatives of each row of logits (no counterpart in
// the reference, which scores with its model's own loss):
//   lse = log sum exp x,  logprob = x[target] - lse,  entropy = lse - sum softmax(x) x,
//   top: the k largest x - lse with their ids, larger first, equal ones by the lower id.
// A row holding NaN or +inf gives NaN log probabilities, as log_softmax does; a row of -inf alone gives -inf and entropy 0.
#pragma once
#include "kv4.cuh"

namespace dscq {

struct LogprobParams {
  const void* x;
  const int64_t* target;
  float *logprob, *entropy, *top;
  int64_t* top_ids;
  int64_t ld;
  int rows, V, k;
};

// Order-preserving 32-bit key of a logit: -0 equals +0, NaN above everything (and all NaN equal).
__device__ __forceinline__ uint32_t logit_key(float v) {
  v += 0.f;
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  if (k == 0xffffffffu) return __int_as_float(0x7fc00000);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ uint64_t umax64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// One CTA per row; passes over the row for the maximum, the sums and each alternative.
template <typename T>
__global__ void __launch_bounds__(256) logprob_rows(const LogprobParams p) {
  __shared__ uint64_t red[8];
  __shared__ float rs[8], rd[8];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + r * p.ld;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto best = [&](uint64_t below) {  // largest (key, ~id) under `below`
    uint64_t m = 0;
    for (int i = tid; i < p.V; i += 256) {
      const uint64_t c = (static_cast<uint64_t>(logit_key(to_float<T>(x[i]))) << 32) | static_cast<uint32_t>(~i);
      if (c < below) m = umax64(m, c);
    }
    for (int o = 16; o; o >>= 1) m = umax64(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();
    if (lane == 0) red[warp] = m;
    __syncthreads();
    for (int w = 0; w < 8; ++w) m = umax64(m, red[w]);
    return m;
  };
  uint64_t top = best(~0ull);
  const float mx = key_logit(static_cast<uint32_t>(top >> 32));
  float s = 0.f, d = 0.f;
  for (int i = tid; i < p.V; i += 256) {
    const float v = to_float<T>(x[i]) - mx, e = expf(v);
    s += e;
    d += e == 0.f ? 0.f : e * v;
  }
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    d += __shfl_xor_sync(0xffffffffu, d, o);
  }
  if (lane == 0) rs[warp] = s, rd[warp] = d;
  __syncthreads();
  s = d = 0.f;
  for (int w = 0; w < 8; ++w) s += rs[w], d += rd[w];
  const bool none = mx == -INFINITY;
  const float logs = none ? 0.f : logf(s);
  auto lp = [&](float v) { return none ? v : (v - mx) - logs; };
  if (tid == 0) {
    const int64_t t = p.target[r];
    float out = 0.f;
    if (t >= p.V) {
      raise_status(kStatusBadIndex);
      out = __int_as_float(0x7fc00000);
    } else if (t >= 0) {
      out = lp(to_float<T>(x[t]));
    }
    p.logprob[r] = out;
    p.entropy[r] = none ? 0.f : logs - d / s;
  }
  for (int i = 0; i < p.k; ++i) {
    if (tid == 0) {
      p.top[r * p.k + i] = lp(key_logit(static_cast<uint32_t>(top >> 32)));
      p.top_ids[r * p.k + i] = static_cast<uint32_t>(~static_cast<uint32_t>(top));
    }
    if (i + 1 < p.k) top = best(top);
  }
}

}  // namespace dscq
