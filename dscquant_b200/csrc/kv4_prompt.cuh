// Attention of many rows per sequence (prompts and their chunks) over the 4-bit paged cache: bound by the tensor cores
// and the exponentials. See kv4_attention.cuh for the operator.
//
// A CTA takes 256 rows (tokens x query heads of one key head) of a sequence as two tiles of 128 and runs over the
// keys they see, 64 at a time (128 to a stage of operands), with tcgen05 (kind::f16, M = 128):
//   S_i = Q_i K^T   (TMEM, two buffers of 64 columns)     P_i = exp2(S_i - max) over S_i     O_i += P_i V   (TMEM)
// The scores of the next 64 keys are made while a softmax runs (one buffer of 128 keys, whose softmax then waits for
// its own products: 1.10 ms instead of 0.98 for 1000-1500-row chunks over 8k, 64/8 heads). TMEM: two tiles of two S/P
// buffers, O_0, O_1 = 512 columns.
//
// Operands are fp16 whatever the cache's type. Codes become numbers on the way into shared memory, four warps, one key
// a thread: a code in the low bits of an fp16 is the subnormal n 2^-24, so an AND and a fused multiply-add give
// round(n step' + low') for two elements, with (step', low') scaled by a power of two that puts the tile's largest
// element under 2^-6. That rounds keys and values to 11 bits; queries, scaled by a power of two a row, are exact. Scores,
// statistics and sums are 32-bit.
// For f16, whose outputs would show that rounding (7e-4 of the result against 64 bits instead of 3e-4), keys and values are
// split into two fp16 parts, each multiplied, which together are within 2^-18 of a row's largest element: twice the
// products, and stages of 64 keys instead of 128 for the same memory. The weights' rounding is the one that stays.
//
// What a row does not see, or hardly weighs, must not cost it bits. With s_j the score of key j and v_j = V_j 2^(E_j) its
// scaled value row, the weights handed to the product are W_j = fp16(2^(T_j - M)), T_j = s_j + E_j, M a running maximum of
// the T_j that the row sees, and
//   out = 2^M sum W_j V_j / sum 2^(s_j).
// E_j is the tile's exponent, but for bf16 a key whose largest element is under 1/16 of the tile's has its own (and keys
// their own scale likewise), so that fp16 keeps 2^-13 of every row's largest element at least. Tiles with such keys, and
// those whose exponent is 20 below an earlier one, so that the sum of the 2^(s_j) cannot be had from the weights in 32
// bits, are marked wide and take a slower path. (All of f16's range fits two parts under one scale: the largest element
// goes under 2^15, and 2^-40 of it stays.) M is a whole number and only moves when it would be passed by 2^8; then the
// row's sums in TMEM are scaled, by the warps that own them. Weights keep 11 bits down to 2^-21 of the largest. (The slower
// path is a loop over TMEM: a second copy of the unrolled one cost the other tiles 9% for its length alone.)
//
// Keys no row may see (behind the end, on pages out of range) are zeros with their scores masked. A value row that is
// not finite is zeros too and flagged; rows that see its key become NaN, the others must not.
//
// Measured on a B200 (with the launch for short sequences before it): chunks of 1000 to 1500 rows over 8 to 10 thousand
// keys, 64 heads on 8: bf16 1000 us, 747 TFLOP/s (0.44 of the cuBLAS rate), f16 1180 us; three prompts of 900 to 2048
// tokens, 32 heads: bf16 151 us, f16 188 us. What binds is the softmax's own chain (read 64 scores, maximum, exponentials, write)
// and its handshakes, two tiles' worth at a time, on 128 registers a thread: 14 warps leave no more, and at D = 128 120
// bytes (f16 212) are spilled. For f16 it is the split of the codes besides: in 32 bits, leaving out half of it took 160 us
// off, half of the products 33. Short prompts add 3 us of setting up and draining to each CTA's few tiles. One
// warp issuing both tiles' products made the chunks 3% slower.
//
// Warps 0-3, 4-7: softmax of tile 0 and 1 (a thread a row); 8-11: codes to operands (split: 8, 9 the even, 10, 11 the odd
// 64 keys, independently); 12, 13: the products of tile 0
// and 1, a warp each so that neither waits for the other's weights. All waits bounded.
#pragma once
#include "kv4_decode.cuh"

namespace dscq {

struct Kv4PromptParams {
  Kv4AttnParams a;
  int64_t min_rows;  // sequences with fewer rows * group than this are not this kernel's
};

constexpr int kKv4PromptThreads = 14 * 32;
constexpr int64_t kKv4AllRows = INT64_MAX;

// A whole number; what 32 bits do not count singly any more stays in range.
__device__ __forceinline__ int whole(float x) { return static_cast<int>(fminf(fmaxf(x, -0x1p28f), 0x1p28f)); }
// x 2^e in two steps, for |e| up to 250.
__device__ __forceinline__ float times_pow2(float x, int e) { return x * pow2f(e / 2) * pow2f(e - e / 2); }

// kind::f16 with fp16 A and B, f32 D; A K-major, B K-major or MN-major (bit 16).
__host__ __device__ constexpr uint32_t umma_idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// D[tmem] (+)= A[tmem] B[smem], A: a lane a row, two consecutive k a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

// 32 lanes x 32 bit, 8 consecutive columns per thread.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int D>
struct Kv4PromptConfig {
  static constexpr int kHalf = 128 * 128;               // 128 rows of 64 fp16, 128-byte swizzled
  static constexpr int kTile = D / 64 * kHalf;          // an operand of 128 rows
  static constexpr int kSmem = 1024 + 6 * kTile + 2048; // Q_0, Q_1, two stages of K and of V; barriers, tile facts
};

template <typename T, int D>
__global__ void __launch_bounds__(kKv4PromptThreads, 1) kv4_prompt_kernel(const Kv4PromptParams p) {
  using C = Kv4PromptConfig<D>;
  constexpr bool kSplit = std::is_same<T, __half>::value;
  const Kv4AttnParams& a = p.a;
  extern __shared__ uint8_t kv4_prompt_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv4_prompt_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = smem;                  // [2]
  uint8_t* ks = smem + 2 * C::kTile;   // [2] tiles, or the two parts of one
  uint8_t* vs = smem + 4 * C::kTile;   // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 6 * C::kTile);
  uint64_t *qfull = bars, *kfull = bars + 1, *kempty = bars + 3, *vfull = bars + 5, *vempty = bars + 7;
  uint64_t *sfull = bars + 9, *pfull = bars + 13, *odone = bars + 17, *done = bars + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* item = reinterpret_cast<int*>(tmem_slot + 2);       // sequence, head, row tile
  int* kexp = item + 4;                                    // [2][2] exponents of the scales of 64 keys
  int* vexp = kexp + 4;
  uint32_t* hide = reinterpret_cast<uint32_t*>(vexp + 4);  // [2][4] keys on pages out of range
  uint32_t* poison = hide + 8;                             // [2][4] keys whose values are not finite
  uint32_t* wide = poison + 8;                             // [2][4] keys with scales of their own
  uint32_t* shift = wide + 8;                              // [2][128] their exponents below the tile's: keys | values << 16
  float* tile_max = reinterpret_cast<float*>(shift + 256); // [2][4][2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // A stage of operands holds 128 keys, split 64: where those of 64 keys `sub` go, and how often it was filled before.
  auto stage_of = [](int sub) { return (kSplit ? sub : sub >> 1) & 1; };
  auto use_of = [](int sub) { return static_cast<uint32_t>(kSplit ? sub >> 1 : sub >> 2); };

  if (warp == 12) {
    // this CTA's 256 rows; of a sequence the last ones, which see the most keys, first
    int64_t left = blockIdx.x;
    int seq = -1, head = 0, tile = 0;
    auto tiles_of = [&](int s) -> int64_t {
      const Kv4Seq r = kv4_seq<128, 256>(a, kKv4AllRows, s);
      return static_cast<int64_t>(r.n) * a.group < p.min_rows ? 0 : static_cast<int64_t>(r.blocks) * a.b.hk;
    };
    auto scan32 = [&](int64_t v) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      return v;
    };
    // a lane adds up a stretch of sequences, then the warp looks through the stretch that holds this CTA
    const int per = (a.b.B + 31) / 32;
    int64_t mine = 0;
#pragma unroll 4
    for (int s = min(lane * per, a.b.B); s < min(lane * per + per, a.b.B); ++s) mine += tiles_of(s);
    const int64_t upto = scan32(mine);
    const unsigned past = __ballot_sync(0xffffffffu, upto > left);
    if (past) {
      const int who = __ffs(past) - 1, end = min(who * per + per, a.b.B);
      left -= __shfl_sync(0xffffffffu, upto - mine, who);
      for (int s0 = who * per; s0 < end && seq < 0; s0 += 32) {
        const int64_t n = s0 + lane < end ? tiles_of(s0 + lane) : 0, sum = scan32(n);
        const unsigned in = __ballot_sync(0xffffffffu, sum > left);
        if (in) {
          const int src = __ffs(in) - 1;
          const int at = static_cast<int>(left - __shfl_sync(0xffffffffu, sum - n, src));
          seq = s0 + src;
          tile = static_cast<int>(__shfl_sync(0xffffffffu, n, src)) / a.b.hk - 1 - at / a.b.hk;
          head = at % a.b.hk;
        } else {
          left -= __shfl_sync(0xffffffffu, sum, 31);
        }
      }
    }
    int halves = 1;
    if (seq >= 0) {
      const Kv4Seq r = kv4_seq<128, 256>(a, kKv4AllRows, seq);
      halves = tile * 256 + 128 < r.n * a.group ? 2 : 1;
    }
    if (lane == 0) {
      item[0] = seq, item[1] = head, item[2] = tile;
      mbar_init(qfull, 8);
      for (int i = 0; i < 2; ++i) {
        mbar_init(kfull + i, kSplit ? 2 : 4);
        mbar_init(vfull + i, kSplit ? 2 : 4);
        mbar_init(kempty + i, halves);
        mbar_init(vempty + i, halves);
        mbar_init(sfull + 2 * i, 1);
        mbar_init(sfull + 2 * i + 1, 1);
        mbar_init(pfull + 2 * i, 4);
        mbar_init(pfull + 2 * i + 1, 4);
        mbar_init(odone + 2 * i, 1);
        mbar_init(odone + 2 * i + 1, 1);
      }
      mbar_init(done, 1);
      mbar_init(done + 1, 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int seq = item[0], head = item[1], r0 = item[2] * 256;
  if (seq >= 0) {
    const Kv4Seq sq = kv4_seq<128, 256>(a, kKv4AllRows, seq);
    const int rows = sq.n * a.group;
    const int halves = r0 + 128 < rows ? 2 : 1;
    // up to the last row's position; 64 keys each
    const int reach = min(sq.keys, sq.len - sq.n + a.row_token(min(r0 + 256, rows) - 1) + 1);
    const int subs = max((reach + 63) / 64, 1);
    const int tiles = (subs + 1) / 2;

    if (warp < 8) {
      // ------------------------------------------------ queries, softmax, output: a thread a row
      const int half = warp >> 2, row = (warp & 3) * 32 + lane, r = r0 + half * 128 + row;
      const bool live = half < halves, real = live && r < rows;
      const int tok = a.row_token(real ? r : 0);
      const int64_t hd = head * a.group + (real ? r - tok * a.group : 0);
      float c1 = 0.f;
      if (live) {
        uint4 x[D / 8];
        float big = 0.f;
        const T* src = static_cast<const T*>(a.q) + (sq.q0 + static_cast<int64_t>(tok)) * a.q_t + hd * a.q_h;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          x[c] = real ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0, 0, 0, 0);
          float f[8];
          kv4_unpack8<T>(x[c], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(f[e]));
        }
        // as in kv4_decode.cuh: the row's largest element in [2^14, 2^15), a negative scale turns the queries around
        const int k = big > 0.f && big < INFINITY ? min(max(14 - log2i(big), -90), 120) : 0;
        const float f = a.scale_log2 == 0.f ? 0.f : copysignf(pow2f(k), a.scale_log2);
        c1 = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2) * pow2f(-k);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          float y[8];
          kv4_unpack8<T>(x[c], y);
          // element order 0 4 1 5 2 6 3 7, as the codes come apart
          const uint4 o = make_uint4(pack2<__half>(y[0] * f, y[4] * f), pack2<__half>(y[1] * f, y[5] * f),
                                     pack2<__half>(y[2] * f, y[6] * f), pack2<__half>(y[3] * f, y[7] * f));
          *reinterpret_cast<uint4*>(qs + half * C::kTile + (c >> 3) * C::kHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = o;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(qfull);

      if (live) {
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + half * 128 + lanes, o_at = tmem + 256 + half * 128 + lanes;
        const int lim = real ? sq.sees(tok) : INT_MAX;  // a row of nothing masks nothing
        float m = -INFINITY, l = 0.f;  // M, a whole number
        int unit = -(1 << 29);         // sum 2^(s_j) = l 2^unit; lower than any score
        bool ok = true, nan = false;
        for (int sub = 0; sub < subs; ++sub) {
          const int t = sub >> 1, u = sub & 1, s = t & 1;
          ok = mbar_wait(&sfull[2 * half + u], t & 1u, abort_flag) &&
               mbar_wait(&vfull[stage_of(sub)], use_of(sub) & 1u, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t at = s_at + u * 64;
          const int see = min(lim - sub * 64, 64);  // columns this row sees
          const uint32_t hidden[2] = {hide[s * 4 + 2 * u], hide[s * 4 + 2 * u + 1]};
          const uint32_t bad[2] = {poison[s * 4 + 2 * u], poison[s * 4 + 2 * u + 1]};
          const float ev = static_cast<float>(vexp[s * 2 + u]);
          float ce = fmaxf(times_pow2(c1, kexp[s * 2 + u]), 0x1p-126f);  // never 0: a masked score of -inf stays one
          float own_sum = 0.f, own_top = -INFINITY;
          const bool own = !kSplit && (wide[s * 4 + 2 * u] | wide[s * 4 + 2 * u + 1]) != 0;
          if (own) {
            // keys with exponents of their own: T_j - E takes the place of their scores, and the s_j are summed up here
            const uint32_t* sh = shift + s * 128 + u * 64;
#pragma unroll 1
            for (int c = 0; c < 64; c += 8) {
              uint32_t x[8];
              tmem_ld8(at + c, x);
              tmem_ld_wait();
              float top = own_top, y[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t e = sh[c + j];
                const bool seen = c + j < see && !(hidden[c >> 5] >> ((c & 31) + j) & 1u);
                y[j] = times_pow2(__uint_as_float(x[j]), -static_cast<int>(e & 0xffffu)) * ce;
                x[j] = __float_as_uint(y[j] - static_cast<float>(e >> 16));
                y[j] = seen ? y[j] : -INFINITY;
                top = fmaxf(top, y[j]);
              }
              tmem_st8(at + c, x);
              top = top == -INFINITY ? top : ceilf(top);
              own_sum *= top == own_top ? 1.f : ex2(own_top - top);
              own_top = top;
#pragma unroll
              for (int j = 0; j < 8; ++j) own_sum += y[j] == -INFINITY ? 0.f : ex2(y[j] - top);
            }
            tmem_st_wait();
            ce = 1.f;
          }
          uint32_t v[2][32];
          tmem_ld32(at, v[0]);
          tmem_ld32(at + 32, v[1]);
          tmem_ld_wait();
          if (bad[0] | bad[1])
            for (int j = 0; j < see; ++j)
              if ((bad[j >> 5] & ~hidden[j >> 5]) >> (j & 31) & 1u) nan = true;
          // ---- the maximum
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (__any_sync(0xffffffffu, see < (c + 1) * 32 || hidden[c])) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c * 32 + j >= see || (hidden[c] >> j & 1u)) v[c][j] = 0xff800000u;
            }
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            mx[0] = fmax3(mx[0], __uint_as_float(v[0][j]), __uint_as_float(v[0][j + 1]));
            mx[1] = fmax3(mx[1], __uint_as_float(v[1][j]), __uint_as_float(v[1][j + 1]));
          }
          float mt = fmaxf(mx[0], mx[1]);
          mt = mt == -INFINITY ? mt : fmaf(mt, ce, ev);
          float f = 1.f;
          if (mt > m + 8.f || (m == -INFINITY && mt > m)) {
            f = pow2f(static_cast<int>(fmaxf(m - ceilf(mt), -126.f)));
            m = ceilf(mt);
          }
          if (sub > 0 && __any_sync(0xffffffffu, f != 1.f)) {
            // the sums up to here must be complete (those before the last were when these scores came)
            ok = mbar_wait(&odone[2 * half + (u ^ 1)], ((sub - 1) >> 1) & 1u, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16(o_at + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(o_at + c, o);
            }
          }
          // ---- weights, over the scores they come from: up to 2^15, so small ones stay normal fp16 numbers down to
          // 2^-21 of the largest
          const float base = m == -INFINITY ? 0.f : m - 7.f - ev;
          float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float p0 = ex2(fmaf(__uint_as_float(v[c][j]), ce, -base));
              const float p1 = ex2(fmaf(__uint_as_float(v[c][j + 1]), ce, -base));
              sums[j & 2] += p0;
              sums[(j & 2) + 1] += p1;
              w[j / 2] = pack2<__half>(p0, p1);
            }
            tmem_st16(at + c * 16, w);
          }
          // ---- the sum of 2^(s_j) is that of 2^(T_j - M + 7) in units of 2^base, where the keys share an exponent
          const float sum = own ? own_sum : (sums[0] + sums[1]) + (sums[2] + sums[3]);
          int in = whole(own ? own_top : base);
          if (mt == -INFINITY) in = unit;  // (a sum over nothing, 0 or NaN)
          const int to = max(unit, in);
          l = fmaf(l, pow2f(max(unit - to, -126)), sum * pow2f(max(in - to, -126)));
          unit = to;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          // from here on the tile's facts may give way to those of the next tile in this stage
          if (lane == 0) mbar_arrive(&pfull[2 * half + u]);
        }
        // A barrier for the sums of even and one for those of odd subs: its phase before the awaited one is then two subs
        // old and surely over, and the one after it cannot come before this warp's next weights, so parity says which.
        ok = ok && mbar_wait(&odone[2 * half + ((subs - 1) & 1)], ((subs - 1) >> 1) & 1u, abort_flag);
        if (__all_sync(0xffffffffu, ok)) {
          tc_fence_after();
          const float inv = nan ? __int_as_float(0x7fc00000) : l == 0.f ? 0.f : 1.f / l;
          const int ev = m == -INFINITY ? 0 : min(max(whole(m) - 7 - unit, -250), 250);
          T* out = static_cast<T*>(a.out) + ((sq.q0 + static_cast<int64_t>(tok)) * a.hq + hd) * D;
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld32(o_at + c, v);
            tmem_ld_wait();
            if (real) {
#pragma unroll
              for (int j = 0; j < 32; j += 8) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = times_pow2(__uint_as_float(v[j + i]) * inv, ev);
                *reinterpret_cast<uint4*>(out + c + j) = make_uint4(pack2<T>(y[0], y[2]), pack2<T>(y[4], y[6]),
                                                                    pack2<T>(y[1], y[3]), pack2<T>(y[5], y[7]));
              }
            }
          }
        }
      }
    } else if (warp < 12) {
      // ------------------------------------------------ codes to operands: a thread a key
      const int key = threadIdx.x - 256, part = warp - 8, odd = part >> 1;  // odd: its 64 keys of the tile
      uint4 kc[D / 32], vc[D / 32];
      uint32_t ka = 0, va = 0;
      bool have = false, lost = false;
      int page = -1;
      auto look = [&](int t) {  // the page of this thread's key in tile t; -1 behind the end
        const int at = t * 128 + key;
        page = t < tiles && at < sq.keys ? a.b.table[seq * a.b.ld_table + (at >> a.b.ps_log2)] : -1;
      };
      auto row_of = [&](int t) {
        return ((static_cast<int64_t>(page) * a.b.hk + head) << a.b.ps_log2) + ((t * 128 + key) & ((1 << a.b.ps_log2) - 1));
      };
      auto load = [&](int t) {
        have = page >= 0 && page < a.b.pages;
        lost = !have && t < tiles && t * 128 + key < sq.keys;
        ka = va = 0;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) kc[c] = vc[c] = make_uint4(0, 0, 0, 0);
        if (!have) return;
        const int64_t row = row_of(t);
        ka = a.b.ka[row];
        va = a.b.va[row];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          kc[c] = reinterpret_cast<const uint4*>(a.b.kc + row * (D / 2))[c];
          vc[c] = reinterpret_cast<const uint4*>(a.b.vc + row * (D / 2))[c];
        }
      };
      // (step 2^24, step 2^20, low) under a scale of 2^-x as pairs of fp16
      auto expand = [&](uint8_t* dst, const uint4 (&codes)[D / 32], float2 f, int x) {
        const float st = times_pow2(f.x, -x), lo = times_pow2(f.y, -x);
        const __half2 s24 = __float2half2_rn(st * 0x1p24f), s20 = __float2half2_rn(st * 0x1p20f), l2 = __float2half2_rn(lo);
        auto two = [&](uint32_t w, const __half2& by) {
          __half2 h;
          memcpy(&h, &w, 4);
          h = __hfma2(h, by, l2);
          memcpy(&w, &h, 4);
          return w;
        };
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 q4 = codes[c / 4];
          const uint32_t w = c % 4 == 0 ? q4.x : c % 4 == 1 ? q4.y : c % 4 == 2 ? q4.z : q4.w, u = w >> 8;
          *reinterpret_cast<uint4*>(dst + (c >> 3) * C::kHalf + key * 128 + (((c & 7) ^ (key & 7)) << 4)) =
              make_uint4(two(w & kCode0, s24), two(w & kCode1, s20), two(u & kCode0, s24), two(u & kCode1, s20));
        }
      };
      // The same in two parts, code * step_a + low_a and code * step_b + low_b. step_a and low_a are the multiples of g
      // nearest to step and low, with g the power of two that makes every element less than 1024 g: the first part is exact, and
      // the second, at most 8 g, rounds by 2^-18 of the row's largest element. (In 32 bits, ten instructions for two
      // elements instead of five, chunks of 1000 to 1500 rows over 8k took 1.34 ms instead of 1.18.) 32 elements a
      // turn: unrolled, the length of the code alone would bind.
      auto split = [&](uint8_t* dst, uint4 (&codes)[D / 32], float2 f, int x) {
        const float st = times_pow2(f.x, -x), lo = times_pow2(f.y, -x);
        const int e = max(log2i(fmaxf(fabsf(lo), fabsf(fmaf(15.f, st, lo)))), -30) - 9;
        const float g = pow2f(e), per = pow2f(-e), sa = rintf(st * per) * g, la = rintf(lo * per) * g;
        const __half2 sa2 = __float2half2_rn(sa), la2 = __float2half2_rn(la);
        const __half2 sb2 = __float2half2_rn(st - sa), lb2 = __float2half2_rn(lo - la);
        const __half2 zero = __float2half2_rn(1024.f);
        auto two = [&](uint32_t w, uint32_t& hi, uint32_t& rest) {
          w = (w & kCode0) | 0x64006400u;  // a code in the low bits of 1024
          __half2 n;
          memcpy(&n, &w, 4);
          n = __hsub2(n, zero);
          const __half2 h = __hfma2(n, sa2, la2), r = __hfma2(n, sb2, lb2);
          memcpy(&hi, &h, 4);
          memcpy(&rest, &r, 4);
        };
#pragma unroll 1
        for (int c = 0; c < D / 8; c += 4) {
          const uint32_t words[4] = {codes[0].x, codes[0].y, codes[0].z, codes[0].w};
#pragma unroll
          for (int i = 0; i + 1 < D / 32; ++i) codes[i] = codes[i + 1];
          uint8_t* row = dst + (c >> 3) * C::kHalf + key * 128;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint4 hi, rest;
            two(words[k], hi.x, rest.x);
            two(words[k] >> 4, hi.y, rest.y);
            two(words[k] >> 8, hi.z, rest.z);
            two(words[k] >> 12, hi.w, rest.w);
            uint8_t* to = row + ((((c + k) & 7) ^ (key & 7)) << 4);
            *reinterpret_cast<uint4*>(to) = hi;
            *reinterpret_cast<uint4*>(to + C::kTile) = rest;
          }
        }
      };
      look(0);
      load(0);
      look(1);
      bool ok = true;
      int run = -1000;  // the largest exponent of values so far
      // the exponent that puts a largest element of x under 2^-6, split 2^15
      auto exponent = [](float x) { return kSplit ? log2i(fmaxf(x, 0x1p-24f)) - 14 : log2i(x) + 7; };
      for (int t = 0; t < tiles; ++t) {
        const int s = t & 1, st = stage_of(2 * t + odd);
        const uint32_t use = use_of(2 * t + odd);
        float2 kf = unpack2<T>(ka), vf = unpack2<T>(va);
        const bool sick = !isfinite(vf.x) || !isfinite(vf.y);
        if (sick) vf = make_float2(0.f, 0.f);
        float km = fmaxf(fabsf(kf.y), fabsf(fmaf(15.f, kf.x, kf.y)));
        float vm = fmaxf(fabsf(vf.y), fabsf(fmaf(15.f, vf.x, vf.y)));
        if (!(km < INFINITY)) km = 0.f;
        if (!(vm < INFINITY)) vm = 0x1.fffffep127f;
        const float kown = km, vown = vm;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, o));
          vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
        }
        if (lane == 0) tile_max[(s * 4 + part) * 2] = km, tile_max[(s * 4 + part) * 2 + 1] = vm;
        const unsigned gone = __ballot_sync(0xffffffffu, lost), ill = __ballot_sync(0xffffffffu, sick && have);
        // a warp whose wait ran out still comes here, so that none of the others stays behind
        if (!named_bar_and(kSplit ? 1 + odd : 1, kSplit ? 64 : 128, ok)) break;
#pragma unroll
        for (int i = 1; i < (kSplit ? 2 : 4); ++i) {
          km = fmaxf(km, tile_max[(s * 4 + (part ^ i)) * 2]);
          vm = fmaxf(vm, tile_max[(s * 4 + (part ^ i)) * 2 + 1]);
        }
        const int kx = exponent(km), vx = exponent(vm);
        // keys far below the tile's largest have exponents of their own; a seen value row of zeros has the lowest, so that
        // its T_j moves no maximum
        auto apart = [&](float x, int tile) {
          return !kSplit && x > 0.f && tile - exponent(x) > 4 ? tile - exponent(x) : 0;
        };
        const int ksh = apart(kown, kx), vsh = !kSplit && vown == 0.f && have && !sick ? 254 : apart(vown, vx);
        run = max(run, vx);
        const unsigned far = __ballot_sync(0xffffffffu, ksh | vsh || vx < run - 20);
        if (lost) raise_status(kStatusBadIndex);

        ok = __all_sync(0xffffffffu, use == 0 || mbar_wait(&kempty[st], (use & 1u) ^ 1u, abort_flag));
        if (!ok) continue;
        if constexpr (kSplit)
          split(ks, kc, kf, kx);
        else
          expand(ks + s * C::kTile, kc, kf, kx - ksh);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[st]);
        ok = __all_sync(0xffffffffu, use == 0 || mbar_wait(&vempty[st], (use & 1u) ^ 1u, abort_flag));
        if (!ok) continue;
        if constexpr (kSplit)
          split(vs, vc, vf, vx);
        else
          expand(vs + s * C::kTile, vc, vf, vx - vsh);
        if constexpr (!kSplit) shift[s * 128 + key] = static_cast<uint32_t>(ksh) | static_cast<uint32_t>(vsh) << 16;
        if (lane == 0) {  // the tile's facts: their last user read them before its values were multiplied
          hide[s * 4 + part] = gone;
          poison[s * 4 + part] = ill;
          wide[s * 4 + part] = far;
          if (!(part & 1)) kexp[s * 2 + odd] = kx, vexp[s * 2 + odd] = vx;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&vfull[st]);
        load(t + 1);
        look(t + 2);
      }
    } else {
      // ------------------------------------------------ MMA: the warp walks together, so addresses stay uniform
      constexpr uint32_t id_qk = umma_idesc_f16(128, 64, false), id_pv = umma_idesc_f16(128, D, true);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(qs)), k_desc = umma_desc_sw128(smem_u32(ks));
      const uint64_t v_desc = umma_desc_sw128_mn_atoms(smem_u32(vs), C::kHalf);
      // S of tile i, keys 64 sub ..: into its buffer sub & 1
      const int i = warp - 12;  // the tile
      constexpr int kParts = kSplit ? 2 : 1;
      // where the operands of keys 64 sub .. begin
      auto keys_at = [&](int sub) {
        return static_cast<uint32_t>(((kSplit ? 0 : stage_of(sub) * C::kTile) + (sub & 1) * 64 * 128) >> 4);
      };
      // whether no later keys of this stage's filling follow
      auto last_of = [&](int sub) { return kSplit || (sub & 1) || sub + 1 == subs; };
      // S of keys 64 sub .. into its buffer sub & 1
      auto scores = [&](int sub) {
        const int st = stage_of(sub), u = sub & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&kfull[st], use_of(sub) & 1u, abort_flag))) return false;
        tc_fence_after();
        const uint64_t qd = q_desc + static_cast<uint32_t>(i * C::kTile >> 4);
        const uint64_t kd = k_desc + keys_at(sub);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kParts * D / 16; ++k) {
            const int part = k / (D / 16), in = k % (D / 16);
            const uint32_t off = static_cast<uint32_t>((in >> 2) * C::kHalf + (in & 3) * 32) >> 4;
            umma_f16_ss(tmem + i * 128 + u * 64, qd + off, kd + off + (part * C::kTile >> 4), id_qk, k > 0 ? 1u : 0u);
          }
          umma_commit(&sfull[2 * i + u]);
          if (last_of(sub)) umma_commit(&kempty[st]);
        }
        __syncwarp();
        return true;
      };
      bool ok = __all_sync(0xffffffffu, i < halves && mbar_wait(qfull, 0, abort_flag));
      for (int sub = 0; ok && sub < min(subs, 2); ++sub) ok = scores(sub);
      for (int sub = 0; ok && sub < subs; ++sub) {
        const int st = stage_of(sub), u = sub & 1;
        const uint64_t vd = v_desc + keys_at(sub);
        ok = mbar_wait(&vfull[st], use_of(sub) & 1u, abort_flag) &&
             mbar_wait(&pfull[2 * i + u], (sub >> 1) & 1u, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kParts * 4; ++k)
            umma_f16_ts(tmem + 256 + i * 128, tmem + i * 128 + u * 64 + k % 4 * 8,
                        vd + ((k / 4 * C::kTile + k % 4 * 2048) >> 4), id_pv, sub > 0 || k > 0 ? 1u : 0u);
          umma_commit(&odone[2 * i + u]);
          if (last_of(sub)) umma_commit(&vempty[st]);
        }
        __syncwarp();
        if (sub + 2 < subs) ok = scores(sub + 2);
      }
      if (elect_one()) umma_commit(&done[i]);
      mbar_wait(&done[i], 0, nullptr);  // nothing is in flight when the memory goes
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace dscq
