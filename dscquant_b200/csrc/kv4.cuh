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
#include <type_traits>

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

// The sequence and position of row t, for a whole warp. Up to 32 sequences take one trip to memory.
__device__ __forceinline__ Kv4Where kv4_position(const Kv4Batch& b, int t) {
  Kv4Where w{-1, 0, 0, false};
  if (b.B == 0) return w;
  int s, q1, len;
  if (b.B <= 32) {
    const int lane = threadIdx.x & 31, i = min(lane, b.B - 1);
    const int lo = b.q_start[i], hi = b.q_start[i + 1], n = b.lengths[i];
    const unsigned in = __ballot_sync(0xffffffffu, lane < b.B && t >= lo && t < hi);
    if (!in) return w;
    s = __ffs(in) - 1;
    q1 = __shfl_sync(0xffffffffu, hi, s);
    len = __shfl_sync(0xffffffffu, n, s);
  } else {
    s = kv4_find_seq(b.q_start, b.B, t);
    const int q0 = b.q_start[s];
    q1 = b.q_start[s + 1], len = b.lengths[s];
    if (t < q0 || t >= q1) return w;
  }
  w.seq = s;
  const int64_t pos = static_cast<int64_t>(len) - (q1 - static_cast<int64_t>(t));
  w.bad = pos < 0 || pos >> b.ps_log2 >= b.P;
  if (!w.bad) w.pos = static_cast<int>(pos);
  return w;
}
// The page of that position.
__device__ __forceinline__ void kv4_page(const Kv4Batch& b, Kv4Where& w) {
  if (w.seq < 0 || w.bad) return;
  w.page = b.table[static_cast<int64_t>(w.seq) * b.ld_table + (w.pos >> b.ps_log2)];
  w.bad = w.page < 0 || w.page >= b.pages;
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

// Eight entries of an angle table, kept as they are stored.
template <typename T, bool F32>
struct Kv4Angles {
  uint4 w[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* table, int64_t at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(table) + at * (F32 ? 4 : 2));
    w[0] = p[0];
    if constexpr (F32) w[1] = p[1];
  }
  __device__ __forceinline__ float get(int i) const {  // i is a constant once unrolled
    const uint4 v = w[F32 ? i / 4 : 0];
    const int j = F32 ? i % 4 : i / 2;
    const uint32_t x = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
    if constexpr (F32) return __uint_as_float(x);
    const float2 f = unpack2<T>(x);
    return i % 2 ? f.y : f.x;
  }
};

// The rows' definition in 64 bits, for the whole warp: low, step and the codes of the 16 elements of this lane, x[0..7]
// and x[D/2 ..], rotated with the angles at `at` unless cos is null.
struct Kv4Row {
  float low, step;
  uint32_t wa, wb;
};
template <typename T, int D, bool F32>
__device__ __forceinline__ Kv4Row kv4_quantise_exact(const T* x, const void* cos, const void* sin, int64_t at) {
  constexpr int H = D / 2;
  double y[16];
  {
    float a[8], b[8];
    kv4_unpack8<T>(*reinterpret_cast<const uint4*>(x), a);
    kv4_unpack8<T>(*reinterpret_cast<const uint4*>(x + H), b);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = a[i], y[i + 8] = b[i];
    if (cos) {
      Kv4Angles<T, F32> c, s;
      c.load(cos, at);
      s.load(sin, at);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[i] = static_cast<double>(a[i]) * c.get(i) - static_cast<double>(b[i]) * s.get(i);
      c.load(cos, at + H);
      s.load(sin, at + H);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[i + 8] = static_cast<double>(b[i]) * c.get(i) + static_cast<double>(a[i]) * s.get(i);
    }
  }
  double mn = y[0], mx = y[0];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    mn = y[i] < mn ? y[i] : mn;
    mx = y[i] > mx ? y[i] : mx;
    nan |= y[i] != y[i];
  }
#pragma unroll
  for (int o = Kv4Rows<D>::kLanes / 2; o; o >>= 1) {
    const double n = __shfl_xor_sync(0xffffffffu, mn, o), x2 = __shfl_xor_sync(0xffffffffu, mx, o);
    mn = n < mn ? n : mn;
    mx = x2 > mx ? x2 : mx;
    nan |= __shfl_xor_sync(0xffffffffu, static_cast<int>(nan), o) != 0;
  }
  Kv4Row r;
  r.low = to_float<T>(from_float<T>(static_cast<float>(mn)));
  r.step = to_float<T>(from_float<T>(static_cast<float>((mx - r.low) / 15.0)));
  r.wa = r.wb = 0;
  if (nan || !isfinite(r.low) || !isfinite(r.step)) {
    r.low = r.step = __int_as_float(0x7fc00000);
  } else if (r.step != 0.f) {
    const double low = r.low, step = r.step, inv = 1.0 / step;
    bool close = false;
    auto pack = [&](auto quotient) {
      r.wa = r.wb = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r.wa |= static_cast<uint32_t>(quotient(y[i] - low)) << (4 * i);
        r.wb |= static_cast<uint32_t>(quotient(y[i + 8] - low)) << (4 * i);
      }
    };
    pack([&](double d) {
      const double t = d * inv, c = rint(t);
      close |= fabs(fabs(t - c) - 0.5) < 0x1p-40;
      return c < 0.0 ? 0.0 : c > 15.0 ? 15.0 : c;
    });
    if (close)  // next to a border the quotient itself decides
      pack([&](double d) { return fmin(fmax(rint(d / step), 0.0), 15.0); });
  }
  return r;
}

// Largest (smallest) of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The same in 32 bits for the 16 elements of this lane. `exact`: they are 16-bit numbers; otherwise they are off by
// at most `rel` times the larger of their own size and `big`. False where that, or the rounding of the arithmetic,
// could decide low, step or a code otherwise than 64 bits do, and where a row is not plain numbers.
//
// Borders of two codes. Inexact rows: no quotient may lie within a window of one. Exact rows are full of ties, which
// rint sends to the even code as it should once the quotient is rounded correctly (one Newton step). A quotient that
// is not a tie stays clear of the border: elements of at least 2^-C of the row's largest are multiples of a power of
// two for which the distance is over 2^-19 (C = 14 for 8 mantissa bits; 11 bits leave 10), and smaller elements sit
// within 2^(4 - C) of the quotient of 0, which must not be near a border itself.
// Codes come out of the rounding addition: the low bits of 1.5 2^23 + t are rint(t).
template <typename T, int D>
__device__ __forceinline__ bool kv4_quantise_fast(const float (&ya)[8], const float (&yb)[8], bool exact, float big,
                                                  float rel, Kv4Row& out) {
  constexpr float kMagic = 12582912.f;
  float mn = ya[0], mx = ya[0];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mn = min3(mn, ya[i], yb[i]);
    mx = max3(mx, ya[i], yb[i]);
  }
#pragma unroll
  for (int o = Kv4Rows<D>::kLanes / 2; o; o >>= 1) {
    const float n = __shfl_xor_sync(0xffffffffu, mn, o), x = __shfl_xor_sync(0xffffffffu, mx, o);
    mn = min3(mn, n, n);
    mx = max3(mx, x, x);
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  }
  const float low = to_float<T>(from_float<T>(mn)), range = mx - low;
  const float step = to_float<T>(from_float<T>(__fdiv_rn(range, 15.f))), inv = 1.f / step;
  out.low = low;
  out.step = step;
  // false for NaN and infinities, a step of 0 or one whose reciprocal overflows, and codes outside 0 .. 15
  bool ok = range * inv < 15.4f && (mn - low) * inv > -0.4f && inv < INFINITY;
  uint32_t wa = 0, wb = 0;
  if (exact) {
    const float back = range - mx;  // the range must not have been rounded
    ok = ok && (mx - (range - back)) + (-low - back) == 0.f;
    auto quotient = [&](float y) {
      const float d = y - low, t = d * inv;
      return fmaf(fmaf(-t, step, d), inv, t);
    };
    constexpr float kNear = std::is_same<T, __half>::value ? 0x1p-6f : 0x1p-10f;
    const float zero = quotient(0.f);
    ok = ok && (mn > 0.f || mx < 0.f || 0.5f - fabsf(zero - rintf(zero)) > kNear);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wa += __float_as_uint(quotient(ya[i]) + kMagic) << (4 * i);
      wb += __float_as_uint(quotient(yb[i]) + kMagic) << (4 * i);
    }
  } else {
    const float err = fmaxf(big, fmaxf(fabsf(mn), fabsf(mx))) * rel, slack = err + fabsf(range) * 0x1p-22f;
    ok = ok && low == to_float<T>(from_float<T>(mn - err)) && low == to_float<T>(from_float<T>(mn + err)) &&
         step == to_float<T>(from_float<T>((range - slack) * (1.f / 15.f))) &&
         step == to_float<T>(from_float<T>((range + slack) * (1.f / 15.f)));
    const float shift = -low * inv;
    // y inv + shift is off by the element's error, that of inv and the roundings of shift and of the result
    const float window = 0x1p-19f + (2.f * err + 0x1p-22f * fmaxf(fabsf(mn), fabsf(mx))) * fabsf(inv);
    float far = 0.f;
    auto code = [&](float y) {
      const float t = fmaf(y, inv, shift), r = t + kMagic;
      far = fmaxf(far, fabsf(t - (r - kMagic)));
      return __float_as_uint(r);
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wa += code(ya[i]) << (4 * i);
      wb += code(yb[i]) << (4 * i);
    }
    ok = ok && far < 0.5f - window;
  }
  constexpr uint32_t kBias = 0x4B400000u + (0x4B400000u << 4) + (0x4B400000u << 8);  // the rest shifts out
  out.wa = wa - kBias;
  out.wb = wb - kBias;
  return ok;
}

// One CTA per token and 256-thread slice of its hq + 2 hk rows (gridDim.y slices; fewer, with more rows a thread,
// once the tokens alone fill the GPU). A group of D/16 lanes takes one row: q rows are rotated in 32 bits and
// rounded once; k rows are rotated and quantised in 32 bits with a bound on the error, and again in 64 bits where
// that could change a bit, so codes are those of the definition; v rows likewise, from exact values.
// Bound by HBM at many rows: q in and out, k and v in, an eighth of that out as codes. Measured on a B200: 10158 tokens
// of 32 + 32 + 32 heads of 128 in 112 us (3.4 TB/s, 0.53 of the copy rate; 101 us without the checks on the error), one
// token in 5 us. 64 registers and four CTAs an SM beat 80 and three (129 us), despite a few spills: what is left is the
// chain from a token's place in the batch to its angles.
template <typename T, int D, bool F32>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const Kv4AppendParams p) {
  using R = Kv4Rows<D>;
  constexpr int H = D / 2;
  const int t = blockIdx.x, hk = p.b.hk, rows = p.hq + 2 * hk;
  const int j0 = (threadIdx.x % R::kLanes) * 8;
  // every lane of a warp runs the same rounds: the shuffles need them all
  const int first = blockIdx.y * R::kPerCta + threadIdx.x / R::kLanes;
  int r = first;
  const int rounds = (rows - static_cast<int>(blockIdx.y) * R::kPerCta + gridDim.y * R::kPerCta - 1) /
                     static_cast<int>(gridDim.y * R::kPerCta);
  uint4 xa, xb;  // the round's row, and the next one's on their way
  uint4 na, nb;
  auto row_of = [&](int row) {
    return j0 + (row < p.hq        ? static_cast<const T*>(p.q) + t * p.q_t + row * p.q_h
                 : row < p.hq + hk ? static_cast<const T*>(p.k) + t * p.k_t + (row - p.hq) * p.k_h
                                   : static_cast<const T*>(p.v) + t * p.v_t + (row - p.hq - hk) * p.v_h);
  };
  auto load = [&](int row) {
    na = nb = make_uint4(0, 0, 0, 0);
    if (row >= rows) return;
    const T* src = row_of(row);
    na = *reinterpret_cast<const uint4*>(src);
    nb = *reinterpret_cast<const uint4*>(src + H);
  };
  load(r);
  Kv4Where w = kv4_position(p.b, t);
  if (w.seq >= 0 && !w.bad && w.pos >= p.table_rows) w.bad = true;
  Kv4Angles<T, F32> cos_a, cos_b, sin_a, sin_b;
  if (w.seq >= 0 && !w.bad) {  // the angles travel while the page is looked up
    const int64_t at = static_cast<int64_t>(w.pos) * D + j0;
    cos_a.load(p.cos, at);
    cos_b.load(p.cos, at + H);
    sin_a.load(p.sin, at);
    sin_b.load(p.sin, at + H);
  }
  kv4_page(p.b, w);
  if (w.bad && threadIdx.x == 0) raise_status(kStatusBadIndex);
  const bool real = w.seq >= 0 && !w.bad;
  const int64_t slot = w.pos & ((1 << p.b.ps_log2) - 1);
  auto store = [&](int row, const Kv4Row& y) {
    const bool is_k = row < p.hq + hk;
    const int64_t at = ((w.page * hk + (row - p.hq - (is_k ? 0 : hk))) << p.b.ps_log2) + slot;
    uint8_t* c = (is_k ? p.b.kc : p.b.vc) + at * (D / 2) + j0 / 2;
    *reinterpret_cast<uint32_t*>(c) = y.wa;
    *reinterpret_cast<uint32_t*>(c + D / 4) = y.wb;
    if (j0 == 0) (is_k ? p.b.ka : p.b.va)[at] = pack2<T>(y.step, y.low);
  };
  bool again = false;
  for (int round = 0; round < rounds; ++round, r += gridDim.y * R::kPerCta) {
    xa = na, xb = nb;
    if (round + 1 < rounds) load(r + gridDim.y * R::kPerCta);
    const bool is_q = r < p.hq, is_k = !is_q && r < p.hq + hk, is_v = r >= p.hq + hk && r < rows;
    if (!real) {  // the whole CTA: nothing to cache, zero queries
      if (is_q) {
        T* o = static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.hq + r) * D + j0;
        *reinterpret_cast<uint4*>(o) = *reinterpret_cast<uint4*>(o + H) = make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    float ya[8], yb[8], big = 0.f;
    kv4_unpack8<T>(xa, ya);
    kv4_unpack8<T>(xb, yb);
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = ya[i], ua = yb[i] * sin_a.get(i), ub = x * sin_b.get(i);
        ya[i] = fmaf(x, cos_a.get(i), -ua);
        yb[i] = fmaf(yb[i], cos_b.get(i), ub);
        if constexpr (F32) big = fmaxf(big, fmaxf(fabsf(ua), fabsf(ub)));
      }
    }
    if (is_q) {
      T* o = static_cast<T*>(p.q_out) + (static_cast<int64_t>(t) * p.hq + r) * D + j0;
      *reinterpret_cast<uint4*>(o) = make_uint4(pack2<T>(ya[0], ya[1]), pack2<T>(ya[2], ya[3]), pack2<T>(ya[4], ya[5]),
                                                pack2<T>(ya[6], ya[7]));
      *reinterpret_cast<uint4*>(o + H) = make_uint4(pack2<T>(yb[0], yb[1]), pack2<T>(yb[2], yb[3]),
                                                    pack2<T>(yb[4], yb[5]), pack2<T>(yb[6], yb[7]));
    }
    if (!__any_sync(0xffffffffu, is_k || is_v)) continue;
    Kv4Row y;
    // the sum rounds by 2^-24 of itself; products of 16-bit numbers are exact, those with a 32-bit angle are not
    const bool ok = kv4_quantise_fast<T, D>(ya, yb, is_v, big, F32 ? 0x1p-23f : 0x1p-24f, y);
    again |= !ok && (is_k || is_v);
    if (is_k || is_v) store(r, y);
  }
  // Seldom: 64 bits for the warp's rows. Behind the loop, where nothing else needs the registers.
  if (real && __any_sync(0xffffffffu, again)) {
    r = first;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round, r += gridDim.y * R::kPerCta) {
      const bool is_k = r >= p.hq && r < p.hq + hk, cached = r >= p.hq && r < rows;
      if (!__any_sync(0xffffffffu, cached)) continue;
      const Kv4Row y = kv4_quantise_exact<T, D, F32>(row_of(min(r, rows - 1)), is_k ? p.cos : nullptr, p.sin,
                                                     static_cast<int64_t>(w.pos) * D + j0);
      if (cached) store(r, y);
    }
  }
}

// The values the cache holds for the rows of the token axis, [T, hk, D] each; zero rows where a row belongs
// to no sequence. Same grid and lane groups over 2 hk rows a token.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Batch b, T* k_out, T* v_out) {
  using R = Kv4Rows<D>;
  const int t = blockIdx.x;
  const int r = blockIdx.y * R::kPerCta + threadIdx.x / R::kLanes;
  const int j0 = (threadIdx.x % R::kLanes) * 8;
  Kv4Where w = kv4_position(b, t);
  kv4_page(b, w);
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
