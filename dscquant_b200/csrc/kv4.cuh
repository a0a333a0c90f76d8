// 4-bit paged key/value cache: layout, position lookup, appending and reading back (no counterpart in the
// reference, whose model keeps its cache in the model's own precision).
//
// One cached row is the D keys (or values) of one token and one key head: D/2 bytes of codes (element 2j in
// the low nibble of byte j, 2j+1 in the high one, 0..15) and two 16-bit numbers (step, low) of the cache's
// type; element = code * step + low. Pages are [kv_heads][page_size] rows, so the rows of one head in one page
// are one contiguous run of page_size * D/2 bytes.
//
//   low  = round16(min y)      step = round16((max y - low) / 15)
//   code = clamp(rint((y - low) / step), 0, 15), 0 where step == 0
//   a row whose low or step is not finite stores step = low = NaN and codes 0, so every reader sees NaN
//
// min and low are taken on the unrounded (rotated) row: rounding it to 16 bits first would cost up to half a
// 16-bit step on every element for nothing, since only codes are kept.
#pragma once
#include "ptx.cuh"

namespace dscq {

// The ragged batch every cache operator takes: rows q_start[b] .. q_start[b+1]-1 of the token axis belong to
// sequence b and are its newest tokens; lengths[b] counts its cached tokens including them.
struct Kv4Batch {
  uint8_t* kc;         // [pages, hk, ps, D/2]
  uint8_t* vc;
  uint32_t* ka;        // [pages, hk, ps] (step, low) pairs
  uint32_t* va;
  const int32_t* table;    // [B, ld_table], entries outside [0, pages) are unmapped
  const int32_t* q_start;  // [B + 1]
  const int32_t* lengths;  // [B]
  int64_t pages, ld_table;
  int B, P, hk, ps_log2;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  T v[2];
  memcpy(v, &w, 4);
  return make_float2(to_float<T>(v[0]), to_float<T>(v[1]));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  T v[2] = {from_float<T>(a), from_float<T>(b)};
  uint32_t w;
  memcpy(&w, v, 4);
  return w;
}

// Largest b in [0, B) with q_start[b] <= t, 32 candidates a round (the whole warp calls it with one t).
__device__ __forceinline__ int kv4_find_seq(const int32_t* q_start, int B, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lane * step;
    const unsigned le = __ballot_sync(0xffffffffu, at < n && q_start[lo + (at < n ? at : 0)] <= t);
    const int hit = le ? 31 - __clz(le) : 0;
    lo += hit * step;
    n = min(step, n - hit * step);
  }
  return lo;
}

// Where row t of the token axis stands. seq < 0: it belongs to no sequence. bad: its position or page lies
// outside what the batch describes (the caller raises kStatusBadIndex and leaves the row out).
struct Kv4Where {
  int seq;
  int pos;
  int64_t page;
  bool bad;
};

__device__ __forceinline__ Kv4Where kv4_where(const Kv4Batch& b, int t) {
  Kv4Where w{-1, 0, 0, false};
  if (b.B == 0) return w;
  const int s = kv4_find_seq(b.q_start, b.B, t);
  const int q0 = b.q_start[s], q1 = b.q_start[s + 1], len = b.lengths[s];
  if (t < q0 || t >= q1) return w;
  w.seq = s;
  const int64_t pos = static_cast<int64_t>(len) - (q1 - static_cast<int64_t>(t));
  const int64_t pi = pos >> b.ps_log2;
  w.bad = pos < 0 || pi >= b.P;
  if (!w.bad) {
    w.pos = static_cast<int>(pos);
    w.page = b.table[static_cast<int64_t>(s) * b.ld_table + pi];
    w.bad = w.page < 0 || w.page >= b.pages;
  }
  return w;
}

struct Kv4AppendParams {
  Kv4Batch b;
  const void *q, *k, *v, *cos, *sin;
  void* q_out;               // [T, hq, D] contiguous
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;  // element strides of tokens and heads
  int T, hq, table_rows;
};

template <int D>
struct Kv4Rows {
  static constexpr int kLanes = D / 16;           // lanes per row: 8 elements of each half of the row
  static constexpr int kPerCta = 256 / kLanes;    // rows a CTA takes
};

template <typename T>
__device__ __forceinline__ void kv4_unpack8(const uint4& w, float (&f)[8]) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = unpack2<T>(a[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

template <bool F32, typename T>
__device__ __forceinline__ void kv4_table8(const void* tab, int64_t at, float (&f)[8]) {
  if constexpr (F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(tab) + at);
    const float4 a = p[0], b = p[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    kv4_unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(tab) + at), f);
  }
}

// Code of y in [low, ...] with the given step (> 0, finite). The quotient in 32 bits decides except within
// 2^-10 of the border of two codes (the quotient's error is below 2^-19), where the sign of the exact
// difference in 64 bits does; a tie goes to the even code.
template <typename Y>
__device__ __forceinline__ uint32_t kv4_code(Y y, float low, float step, float inv) {
  const float t = static_cast<float>(y - static_cast<Y>(low)) * inv;
  float c = rintf(t);
  if (fabsf(fabsf(t - c) - 0.5f) < 0x1p-10f) {
    const double below = floor(static_cast<double>(t));
    const double d = (static_cast<double>(y) - low) - (below + 0.5) * static_cast<double>(step);
    const bool odd = (static_cast<int>(below) & 1) != 0;
    c = static_cast<float>(below) + ((d > 0 || (d == 0 && odd)) ? 1.f : 0.f);
  }
  return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));
}

// Quantises the row whose elements this lane group holds (ya: 8 of the first half, yb: 8 of the second) and
// stores it. Every lane of the warp takes part in the shuffles.
template <typename T, int D, typename Y>
__device__ __forceinline__ void kv4_store_row(const Y (&ya)[8], const Y (&yb)[8], uint8_t* codes, uint32_t* affine,
                                              int64_t row, int j0, bool store) {
  Y mn = ya[0], mx = ya[0];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mn = min(mn, min(ya[i], yb[i]));
    mx = max(mx, max(ya[i], yb[i]));
    nan |= ya[i] != ya[i] || yb[i] != yb[i];  // min and max drop a NaN
  }
#pragma unroll
  for (int o = Kv4Rows<D>::kLanes / 2; o; o >>= 1) {
    mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    nan |= __shfl_xor_sync(0xffffffffu, static_cast<int>(nan), o) != 0;
  }
  const float low = to_float<T>(from_float<T>(static_cast<float>(mn)));
  const float step = to_float<T>(from_float<T>(static_cast<float>((static_cast<double>(mx) - low) / 15.0)));
  const bool bad = nan || !isfinite(low) || !isfinite(step);
  uint32_t wa = 0, wb = 0;
  if (!bad && step != 0.f) {
    const float inv = 1.f / step;
    if (isfinite(inv)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        wa |= kv4_code<Y>(ya[i], low, step, inv) << (4 * i);
        wb |= kv4_code<Y>(yb[i], low, step, inv) << (4 * i);
      }
    } else {  // a step so small that its reciprocal overflows: divide in 64 bits
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double a = rint((static_cast<double>(ya[i]) - low) / step), b = rint((static_cast<double>(yb[i]) - low) / step);
        wa |= static_cast<uint32_t>(fmin(fmax(a, 0.0), 15.0)) << (4 * i);
        wb |= static_cast<uint32_t>(fmin(fmax(b, 0.0), 15.0)) << (4 * i);
      }
    }
  }
  if (!store) return;
  uint8_t* c = codes + row * (D / 2) + j0 / 2;
  *reinterpret_cast<uint32_t*>(c) = wa;
  *reinterpret_cast<uint32_t*>(c + D / 4) = wb;
  const float nanv = __int_as_float(0x7fc00000);
  if (j0 == 0) affine[row] = pack2<T>(bad ? nanv : step, bad ? nanv : low);
}

// grid (T, ceil((hq + 2 hk) / rows per CTA)), 256 threads. A group of D/16 lanes takes one row: q rows are
// rotated in 32 bits and rounded once; k rows are rotated in 64 bits (the products and their sum are exact
// there, so codes do not depend on how a compiler contracts them) and quantised; v rows are quantised.
// Bound by HBM at many rows: q in and out, k and v in, an eighth of that out as codes.
template <typename T, int D, bool F32>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p) {
  using R = Kv4Rows<D>;
  constexpr int H = D / 2;
  const int t = blockIdx.x;
  const int r = blockIdx.y * R::kPerCta + threadIdx.x / R::kLanes;
  const int j0 = (threadIdx.x % R::kLanes) * 8;
  const int hk = p.b.hk;
  const int kind = r < p.hq ? 0 : r < p.hq + hk ? 1 : r < p.hq + 2 * hk ? 2 : 3;
  const int h = kind == 0 ? r : kind == 1 ? r - p.hq : r - p.hq - hk;
  uint4 xa = make_uint4(0, 0, 0, 0), xb = xa;
  if (kind < 3) {
    const T* src = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                   t * (kind == 0 ? p.q_t : kind == 1 ? p.k_t : p.v_t) +
                   h * (kind == 0 ? p.q_h : kind == 1 ? p.k_h : p.v_h) + j0;
    xa = *reinterpret_cast<const uint4*>(src);
    xb = *reinterpret_cast<const uint4*>(src + H);
  }
  Kv4Where w = kv4_where(p.b, t);
  if (w.seq >= 0 && !w.bad && w.pos >= p.table_rows) w.bad = true;
  if (w.bad && threadIdx.x == 0) raise_status(kStatusBadIndex);
  const bool real = w.seq >= 0 && !w.bad;
  float a[8], b[8], ca[8], cb[8], sa[8], sb[8];
  kv4_unpack8<T>(xa, a);
  kv4_unpack8<T>(xb, b);
  const int64_t at = static_cast<int64_t>(real ? w.pos : 0) * D + j0;
  if (kind < 2 && real) {
    kv4_table8<F32, T>(p.cos, at, ca);
    kv4_table8<F32, T>(p.cos, at + H, cb);
    kv4_table8<F32, T>(p.sin, at, sa);
    kv4_table8<F32, T>(p.sin, at + H, sb);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) ca[i] = cb[i] = sa[i] = sb[i] = 0.f;
  }
  if (kind == 0) {
    uint32_t oa[4], ob[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 2 * i;
      oa[i] = real ? pack2<T>(a[e] * ca[e] - b[e] * sa[e], a[e + 1] * ca[e + 1] - b[e + 1] * sa[e + 1]) : 0u;
      ob[i] = real ? pack2<T>(b[e] * cb[e] + a[e] * sb[e], b[e + 1] * cb[e + 1] + a[e + 1] * sb[e + 1]) : 0u;
    }
    T* o = static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.hq + h) * D + j0;
    *reinterpret_cast<uint4*>(o) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
    *reinterpret_cast<uint4*>(o + H) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
  }
  const bool store = real && (kind == 1 || kind == 2);
  const int64_t row = ((w.page * hk + h) << p.b.ps_log2) + (w.pos & ((1 << p.b.ps_log2) - 1));
  if (__any_sync(0xffffffffu, store && kind == 1)) {
    double ya[8], yb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double x1 = a[i], x2 = b[i];
      ya[i] = x1 * static_cast<double>(ca[i]) - x2 * static_cast<double>(sa[i]);
      yb[i] = x2 * static_cast<double>(cb[i]) + x1 * static_cast<double>(sb[i]);
    }
    kv4_store_row<T, D, double>(ya, yb, p.b.kc, p.b.ka, row, j0, store && kind == 1);
  }
  if (__any_sync(0xffffffffu, store && kind == 2))
    kv4_store_row<T, D, float>(a, b, p.b.vc, p.b.va, row, j0, store && kind == 2);
}

// The values the cache holds for the rows of the token axis, [T, hk, D] each; zero rows where a row belongs
// to no sequence. Same grid and lane groups over 2 hk rows a token.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Batch b, T* k_out, T* v_out) {
  using R = Kv4Rows<D>;
  const int t = blockIdx.x;
  const int r = blockIdx.y * R::kPerCta + threadIdx.x / R::kLanes;
  const int j0 = (threadIdx.x % R::kLanes) * 8;
  const Kv4Where w = kv4_where(b, t);
  if (w.bad && threadIdx.x == 0) raise_status(kStatusBadIndex);
  if (r >= 2 * b.hk) return;
  const bool is_v = r >= b.hk;
  const int h = is_v ? r - b.hk : r;
  uint32_t oa[4] = {0, 0, 0, 0}, ob[4] = {0, 0, 0, 0};
  if (w.seq >= 0 && !w.bad) {
    const int64_t row = ((w.page * b.hk + h) << b.ps_log2) + (w.pos & ((1 << b.ps_log2) - 1));
    const uint8_t* c = (is_v ? b.vc : b.kc) + row * (D / 2) + j0 / 2;
    const uint32_t wa = *reinterpret_cast<const uint32_t*>(c), wb = *reinterpret_cast<const uint32_t*>(c + D / 4);
    const float2 f = unpack2<T>((is_v ? b.va : b.ka)[row]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 8 * i;
      oa[i] = pack2<T>(fmaf(static_cast<float>((wa >> e) & 15u), f.x, f.y),
                       fmaf(static_cast<float>((wa >> (e + 4)) & 15u), f.x, f.y));
      ob[i] = pack2<T>(fmaf(static_cast<float>((wb >> e) & 15u), f.x, f.y),
                       fmaf(static_cast<float>((wb >> (e + 4)) & 15u), f.x, f.y));
    }
  }
  T* o = (is_v ? v_out : k_out) + (static_cast<int64_t>(t) * b.hk + h) * D + j0;
  *reinterpret_cast<uint4*>(o) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
  *reinterpret_cast<uint4*>(o + D / 2) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
}

}  // namespace dscq
