// Log probabilities of given tokens, entropy and the top alternatives of each row of logits (no counterpart in
// the reference, which scores with its model's own loss):
//   lse = log sum exp x,  logprob = x[target] - lse,  entropy = lse - sum softmax(x) x,
//   top: the k largest x - lse with their ids, larger first, equal ones by the lower id.
// A row holding NaN or +inf gives NaN log probabilities, as log_softmax does; a row of -inf alone gives -inf and entropy 0.
#pragma once
#include "kv4_decode.cuh"

namespace dscq {

struct LogprobParams {
  const void* x;
  const int64_t* target;
  float *logprob, *entropy, *top;
  int64_t* top_ids;
  int64_t ld;
  int rows, V, k;
  int parts;  // CTAs a row (a cluster)
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
// (value, index) as one number: larger values first, equal ones by the lower index; unique within a row.
__device__ __forceinline__ uint64_t logit_rank(float v, uint32_t i) {
  return static_cast<uint64_t>(logit_key(v)) << 32 | static_cast<uint32_t>(~i);
}

// A row's running maximum m with s = sum 2^t and d = sum 2^t t over its logits, t = (x - m) log2 e. The largest
// term is 1, so nothing overflows; -inf adds nothing, NaN and +inf turn s into NaN.
struct LogitSums {
  float m, s, d;
  __device__ __forceinline__ void move(float to) {  // to >= m
    const float t = fmaxf((m - to) * 1.4426950408889634f, -1000.f), f = s == 0.f ? 0.f : ex2(t);
    d = s == 0.f ? 0.f : f * fmaf(t, s, d);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x) {
    const float t = (x - (m == -INFINITY ? 0.f : m)) * 1.4426950408889634f, e = ex2(t);
    s += e;
    d = fmaf(e, fmaxf(t, -1000.f), d);
  }
};

constexpr int kLpThreads = 256;
constexpr int kLpGroups = 64;   // threads in fours: their maxima bound the k-th largest logit from below
constexpr int kLpCands = 1024;  // candidates kept

// A CTA (or a cluster of them, each with a slice) per row, one pass over the row from HBM: 16-byte loads, a running
// (m, s, d) a thread. The k-th largest of 64 group maxima is a bound that at least k logits reach;
// about k ln 64 at most do in earnest, and only the few threads whose own maximum does look at their logits again
// (from L2). Those candidates are ranked by counting. A row where more than 1024 reach it (equal logits, a
// masked vocabulary) takes the strictly larger ones and the first k equal ones in index order; should even
// those not fit, or the row hold NaN or +inf, k passes for the next largest. Slices of a row meet through
// distributed shared memory: their sums, and their k best each.
//
// Measured on a B200: 4096 rows of 32000 bf16 logits in 57 us without alternatives (4.65 TB/s, 0.72 of the copy rate; the
// exponentials alone need 30 us), 77 us with 20; one row 5 us (8 us with 5). Eight CTAs an SM (32 registers) hide the
// trips to memory: 102 us at six with each thread going over its own logits again, 81 with its warp doing it.
template <typename T>
__global__ void __launch_bounds__(kLpThreads, 8) logprob_rows(const LogprobParams p) {
  constexpr int VE = 16 / sizeof(T);  // elements of a 16-byte load
  __shared__ uint64_t cand[kLpCands];
  __shared__ uint64_t best[64];  // this slice's top k
  __shared__ uint64_t red64[8];
  __shared__ __align__(16) float gmax[kLpGroups];
  __shared__ float redm[8], reds[8], redd[8];
  __shared__ __align__(16) float slice[4];  // m, s, d for the cluster
  __shared__ int found, scan[9];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int parts = p.parts, part = static_cast<int>(blockIdx.x) % parts;
  const int64_t r = blockIdx.x / parts;
  const T* x = static_cast<const T*>(p.x) + r * p.ld;
  // The row: `head` elements up to a 16-byte boundary, `nv` loads, a tail. This slice has the loads [v0, v1); the
  // first slice the head as well, the last the tail.
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / static_cast<int>(sizeof(T));
  const int head = min(off ? VE - off : 0, p.V), nv = (p.V - head) / VE;
  const int v0 = static_cast<int>(static_cast<int64_t>(nv) * part / parts);
  const int v1 = static_cast<int>(static_cast<int64_t>(nv) * (part + 1) / parts);
  const int tail0 = head + nv * VE;
  const int lone = part == 0 && tid < head ? tid : part == parts - 1 && tid >= VE && tail0 + tid - VE < p.V && tid < 2 * VE
                                                       ? tail0 + tid - VE : -1;  // a single element of this thread
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  auto unpack = [](const uint4& w, float (&f)[VE]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VE == 4) {
        f[i] = __uint_as_float(a[i]);
      } else {
        const float2 v = unpack2<T>(a[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
      }
    }
  };

  LogitSums a{-INFINITY, 0.f, 0.f};
  auto feed = [&](const uint4& w) {
    float f[VE];
    unpack(w, f);
    float m = f[0];
#pragma unroll
    for (int e = 1; e < VE; ++e) m = fmaxf(m, f[e]);
    if (m > a.m) a.move(m);
#pragma unroll
    for (int e = 0; e < VE; ++e) a.add(f[e]);
  };
  int v = v0 + tid;
  for (; v + 3 * kLpThreads < v1; v += 4 * kLpThreads) {
    uint4 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = __ldg(xv + v + u * kLpThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u) feed(w[u]);
  }
  for (; v < v1; v += kLpThreads) feed(__ldg(xv + v));
  float alone = -INFINITY;
  if (lone >= 0) {
    alone = to_float<T>(x[lone]);
    if (alone > a.m) a.move(alone);
    a.add(alone);
  }
  const float mine = a.m;  // the thread's largest logit

  float m = mine;
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
  if (lane % 4 == 0) gmax[tid / 4] = m;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) redm[warp] = m;
  if (tid == 0) found = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, redm[w]);
  a.move(m);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.d += __shfl_xor_sync(0xffffffffu, a.d, o);
  }
  if (lane == 0) reds[warp] = a.s, redd[warp] = a.d;
  __shared__ float bound;
  if (p.k && tid < kLpGroups) {  // the k-th largest group maximum
    const float g = gmax[tid];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < kLpGroups; j += 4) {
      const float4 o = *reinterpret_cast<const float4*>(gmax + j);
      rank += (o.x > g || (o.x == g && j < tid)) + (o.y > g || (o.y == g && j + 1 < tid)) +
              (o.z > g || (o.z == g && j + 2 < tid)) + (o.w > g || (o.w == g && j + 3 < tid));
    }
    if (rank == p.k - 1) bound = g;
  }
  __syncthreads();
  a.s = a.d = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) a.s += reds[w], a.d += redd[w];

  if (p.k) {
    const float tau = bound;
    // f(value, index) over the elements of the threads with `mine_in`; a warp goes over each such thread's loads
    // together, one a lane, so looking again costs one trip to memory and not a chain of them
    auto each_of = [&](bool mine_in, auto f) {
      for (unsigned in = __ballot_sync(0xffffffffu, mine_in); in; in &= in - 1) {
        const int first = v0 + warp * 32 + __ffs(in) - 1;
#pragma unroll 1
        for (int u = first + lane * kLpThreads; u < v1; u += 32 * kLpThreads) {
          float y[VE];
          unpack(__ldg(xv + u), y);
#pragma unroll
          for (int e = 0; e < VE; ++e) f(y[e], head + u * VE + e);
        }
      }
      if (mine_in && lone >= 0) f(alone, lone);
    };
    const bool plain = a.s == a.s;  // no NaN, no +inf
    int n = 0;
    bool rounds = !plain;
    if (plain) {
      // (once there are too many, how many no longer matters)
      each_of(mine >= tau, [&](float y, int i) {
        if (y >= tau && *static_cast<volatile int*>(&found) <= kLpCands) {
          const int at = atomicAdd(&found, 1);
          if (at < kLpCands) cand[at] = logit_rank(y, i);
        }
      });
      __syncthreads();
      n = found;
      if (n > kLpCands) {
        // ---- many equal logits: the strictly larger ones, then the first k equal ones
        __syncthreads();
        if (tid == 0) found = 0;
        __syncthreads();
        each_of(mine > tau, [&](float y, int i) {
          if (y > tau && *static_cast<volatile int*>(&found) <= kLpCands) {
            const int at = atomicAdd(&found, 1);
            if (at < kLpCands - 64) cand[at] = logit_rank(y, i);
          }
        });
        __syncthreads();
        n = found;
        rounds = n > kLpCands - 64;
        const int lo = part == 0 ? 0 : head + v0 * VE, hi = part == parts - 1 ? p.V : head + v1 * VE;
        for (int i0 = lo, got = 0; !rounds && i0 < hi && got < p.k; i0 += kLpThreads) {
          const bool eq = i0 + tid < hi && to_float<T>(x[i0 + tid]) == tau;
          const unsigned b = __ballot_sync(0xffffffffu, eq);
          if (lane == 0) scan[warp] = __popc(b);
          __syncthreads();
          int at = got + __popc(b & ((1u << lane) - 1));
          for (int w = 0; w < 8; ++w) {
            if (w < warp) at += scan[w];
            got += scan[w];
          }
          if (eq && at < p.k) cand[n + at] = logit_rank(tau, i0 + tid);
          __syncthreads();
          if (got >= p.k || i0 + kLpThreads >= hi) n += min(got, p.k);
        }
      }
    }
    if (rounds) {
      uint64_t below = 0;
      for (int i = 0; i < p.k; ++i) {
        uint64_t c = 0;
        each_of(true, [&](float y, int j) {
          const uint64_t z = logit_rank(y, j);
          if (i == 0 || z < below) c = umax64(c, z);  // NaN at index 0 has the largest rank there is
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) c = umax64(c, __shfl_xor_sync(0xffffffffu, c, o));
        __syncthreads();
        if (lane == 0) red64[warp] = c;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) c = umax64(c, red64[w]);
        if (tid == 0) best[i] = c;
        below = c;
      }
    } else {
      for (int i = tid; i < n; i += kLpThreads) {
        const uint64_t c = cand[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += cand[j] > c;
        if (rank < p.k) best[rank] = c;
      }
      for (int i = n + tid; i < p.k; i += kLpThreads) best[i] = 0;  // a slice of fewer than k
    }
    __syncthreads();
  }

  int n = p.k;
  const uint64_t* top = best;
  if (parts > 1) {
    if (tid == 0) slice[0] = m, slice[1] = a.s, slice[2] = a.d;
    cluster_sync();
    if (part == 0) {
      for (int i = tid; i < parts * p.k; i += kLpThreads) {
        const uint32_t at = dsmem_map(smem_u32(best + i % p.k), static_cast<uint32_t>(i / p.k));
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(cand[i]) : "r"(at) : "memory");
      }
      float big = -INFINITY;
      LogitSums o[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (w >= parts) break;
        const int4 y = dsmem_ld_v4(dsmem_map(smem_u32(slice), static_cast<uint32_t>(w)));
        o[w] = LogitSums{__int_as_float(y.x), __int_as_float(y.y), __int_as_float(y.z)};
        big = fmaxf(big, o[w].m);
      }
      a.s = a.d = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (w >= parts) break;
        o[w].move(big);
        a.s += o[w].s, a.d += o[w].d;
      }
      m = big;
    }
    cluster_sync();
    if (part) return;
    n = parts * p.k;
    top = cand;
  }
  const bool none = m == -INFINITY && a.s == 0.f;
  const float logs = none ? 0.f : logf(a.s);
  auto lp = [&](float y) { return none ? y : (y - m) - logs; };
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
    p.entropy[r] = none ? 0.f : fmaf(a.d / a.s, -0.6931471805599453f, logs);
  }
  for (int i = tid; i < n; i += kLpThreads) {
    const uint64_t c = top[i];
    int rank = parts > 1 ? 0 : i;
    if (parts > 1)
      for (int j = 0; j < n; ++j) rank += top[j] > c;
    if (rank < p.k && c) {
      p.top[r * p.k + rank] = lp(key_logit(static_cast<uint32_t>(c >> 32)));
      p.top_ids[r * p.k + rank] = static_cast<uint32_t>(~static_cast<uint32_t>(c));
    }
  }
}

}  // namespace dscq
