// Attention of few rows per sequence (single tokens, drafts) over the 4-bit paged cache: bound by reading the
// cache once. See kv4_attention.cuh for the operator.
//
// Mathematics. With n the 4-bit code, (step, low) of a row and c' = 1 + n/16 (one shift and one LOP3 put two
// codes into the mantissas of two 16-bit numbers, exactly):
//   q.k = 16 step (q.c') + (low - 16 step) sum(q)          -- q.c' on the tensor cores, the rest per key
//   o   = 16/F (sum_t P'_t c'_t - sum_t P'_t) + sum_t p_t low_t,   P'_t = round16(F p_t step_t)
// so no element is ever dequantised; step and low cost a few operations per key, not per element. Scores,
// softmax statistics and sums are 32-bit; only the weights P' are rounded to 16 bits, as the tensor cores
// take them (F = 16 for bf16; 4 for f16, whose range F step must not leave).
//
// Fragments (mma.m16n8k16). Scores: A = 16 keys x 16 dims, B = 8 query rows; a lane's 32 dims (16 for D = 64)
// of a key are one 16-byte load, any dim order works as long as the queries use the same. Output: A = 16
// dims x 16 keys, B = weights; a lane needs pairs of adjacent KEYS for one dim, which a byte permute of two
// keys' words gives. The weights move from the score layout (key, row) to B's (row, key) by movmatrix.
//
// Work split. All (sequence, key head, block of 8 NT rows) runs are laid end to end as tiles of TILE keys and cut into
// equal shares, one a warp, whatever the lengths; the cut points come from the lengths on the device, so a captured
// launch follows them. A warp streams its share through its own ring of bulk copies, across run borders. It
// finishes runs that lie inside its share; pieces of cut runs meet in shared memory once all warps of the
// CTA are done, pieces of runs cut by CTA borders in a second kernel, in order: no atomics, the same bits every time.
#pragma once
#include "kv4_attention.cuh"

namespace dscq {

struct Kv4DecodeParams {
  Kv4AttnParams a;
  int64_t max_rows;  // sequences with more rows * group than this are not this kernel's
  float* ws;         // [G][2][8 NT][D + 2]: rows' sums, then their maxima and weights' sums
  int* desc;         // [G][8]: slot 0 {valid, ends}, slot 1 {valid, b, h, block}
};

template <typename T>
struct Kv4Mma;
template <>
struct Kv4Mma<__nv_bfloat16> {
  static constexpr uint32_t kOne = 0x3F803F80u, kMask = 0x00780078u;
  static constexpr int kShift = 3;  // code's place in the mantissa
  static constexpr float kF = 16.f;
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Kv4Mma<__half> {
  static constexpr uint32_t kOne = 0x3C003C00u, kMask = 0x03C003C0u;
  static constexpr int kShift = 6;
  static constexpr float kF = 4.f;
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Codes I and I + 4 of `w` as the pair (1 + n/16, 1 + n'/16).
template <typename T, int I>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w) {
  constexpr int s = Kv4Mma<T>::kShift - 4 * I;
  const uint32_t x = s >= 0 ? w << (s >= 0 ? s : 0) : w >> (s < 0 ? -s : 0);
  return (x & Kv4Mma<T>::kMask) | Kv4Mma<T>::kOne;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// One sequence as the decode kernel sees it.
struct Kv4Seq {
  int q0, n, len, tiles, blocks;  // first row, rows, cached tokens (as given), tiles of a run, row blocks
  int keys;                       // cached tokens the page table can hold
};

template <int TILE, int RB>
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnParams& a, int64_t max_rows, int s) {
  Kv4Seq r;
  int q0 = a.b.q_start[s], q1 = a.b.q_start[s + 1];
  r.len = a.b.lengths[s];
  r.q0 = max(q0, 0);
  r.n = max(min(q1, a.T) - r.q0, 0);
  const int cap = a.b.P << a.b.ps_log2;
  r.keys = min(max(r.len, 0), cap);
  const int64_t rows = static_cast<int64_t>(r.n) * a.group;
  r.blocks = rows > max_rows ? 0 : static_cast<int>((rows + RB - 1) / RB);
  r.tiles = max((r.keys + TILE - 1) / TILE, 1);
  if (r.n > 0 && (r.len > cap || q0 < 0 || q1 > a.T)) raise_status(kStatusBadIndex);
  return r;
}

template <int D_, int NT_, int WARPS_, int STAGES_, int TILE_>
struct Kv4DecodeConfig {
  static constexpr int D = D_, NT = NT_, WARPS = WARPS_, STAGES = STAGES_, TILE = TILE_;
  static constexpr int RB = 8 * NT;                       // rows of a block
  static constexpr int kCodes = TILE * D / 2;             // bytes of one side's codes in a stage
  static constexpr int kStage = 2 * kCodes + 2 * TILE * 4;
  static constexpr int kRing = STAGES * kStage;
  static constexpr int kPiece = RB * (D + 2) * 4;         // a cut run's piece
  static constexpr int kSmem = WARPS * (kRing + kPiece) + WARPS * STAGES * 12 + 1024;
  static_assert(kRing >= kPiece, "the last piece of a warp goes into its ring");
  static_assert(2 * WARPS <= 32 && kStage % 16 == 0 && kPiece % 16 == 0, "layout");
};

template <typename T, class C>
__global__ void __launch_bounds__(C::WARPS * 32, 1) kv4_decode_kernel(const Kv4DecodeParams p) {
  using M = Kv4Mma<T>;
  constexpr int D = C::D, NT = C::NT, TILE = C::TILE, WARPS = C::WARPS, STAGES = C::STAGES, RB = C::RB;
  constexpr int KB = TILE / 16;  // 16-key blocks of a tile
  constexpr int W4 = D / 32;     // words of codes a lane takes of a key
  const Kv4AttnParams& a = p.a;
  extern __shared__ __align__(128) uint8_t kv4_smem[];
  uint8_t* first_all = kv4_smem + WARPS * C::kRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(first_all + WARPS * C::kPiece);
  uint32_t* vmask_all = reinterpret_cast<uint32_t*>(bars + WARPS * STAGES);
  __shared__ int64_t scan[WARPS + 1];
  __shared__ int where[WARPS][4];    // sequence, head, block, tile a warp starts at
  __shared__ int piece[2 * WARPS][6];  // valid, starts, ends, b, h, block; pieces 2w (cut at its start), 2w + 1

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  uint8_t* ring = kv4_smem + warp * C::kRing;
  uint64_t* full = bars + warp * STAGES;
  uint32_t* vmask = vmask_all + warp * STAGES;
  if (lane < STAGES) {
    mbar_init(&full[lane], 1);
    fence_mbar_init();
  }
  if (tid < 2 * WARPS) piece[tid][0] = 0;

  // Rows of no sequence are zero.
  const int B = a.b.B;
  {
    const int lo = B ? min(max(a.b.q_start[0], 0), a.T) : 0, hi = B ? min(max(a.b.q_start[B], lo), a.T) : 0;
    const int64_t row16 = static_cast<int64_t>(a.hq) * D / 8;  // 16-byte pieces of a row
    const int64_t none = (lo + a.T - hi) * row16;
    for (int64_t i = blockIdx.x * (WARPS * 32ll) + tid; i < none; i += gridDim.x * (WARPS * 32ll)) {
      const int64_t r = i < lo * row16 ? i : i - lo * row16 + hi * row16;
      reinterpret_cast<uint4*>(a.out)[r] = make_uint4(0, 0, 0, 0);
    }
  }

  // Every CTA adds up the tiles of all sequences; whoever holds a warp's first tile says where it is.
  const int per = (B + WARPS * 32 - 1) / (WARPS * 32);
  const int s_lo = min(tid * per, B), s_hi = min(s_lo + per, B);
  int64_t mine = 0;
  for (int s = s_lo; s < s_hi; ++s) {
    const Kv4Seq r = kv4_seq<TILE, RB>(a, p.max_rows, s);
    mine += static_cast<int64_t>(r.blocks) * r.tiles * a.b.hk;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w == warp) before = total;
    total += scan[w];
  }
  before += incl - mine;
  // a warp has at least one tile where there are enough; CTAs beyond that have none
  const int64_t parts = max(min(total / WARPS, static_cast<int64_t>(gridDim.x)), static_cast<int64_t>(1));
  const int64_t shares = parts * WARPS;
  for (int w = 0; w < WARPS; ++w) {
    const int64_t at = total * (static_cast<int64_t>(blockIdx.x) * WARPS + w) / shares;
    if (at >= before && at < before + mine) {
      int64_t left = at - before;
      for (int s = s_lo; s < s_hi; ++s) {
        const Kv4Seq r = kv4_seq<TILE, RB>(a, p.max_rows, s);
        const int64_t units = static_cast<int64_t>(r.blocks) * r.tiles * a.b.hk;
        if (left < units) {
          const int64_t run = left / r.tiles;
          where[w][0] = s;
          where[w][1] = static_cast<int>(run / r.blocks);
          where[w][2] = static_cast<int>(run % r.blocks);
          where[w][3] = static_cast<int>(left % r.tiles);
          break;
        }
        left -= units;
      }
    }
  }
  __syncthreads();

  const int64_t gw = static_cast<int64_t>(blockIdx.x) * WARPS + warp;
  const int64_t count = gw < shares ? total * (gw + 1) / shares - total * gw / shares : 0;
  struct Cursor {
    int b, h, blk, t;
    Kv4Seq s;
  };
  Cursor c{where[warp][0], where[warp][1], where[warp][2], where[warp][3], {}};
  if (count > 0) c.s = kv4_seq<TILE, RB>(a, p.max_rows, c.b);
  Cursor pr = c;  // the tile to fetch next
  auto advance = [&](Cursor& x, bool more) {
    if (++x.t < x.s.tiles) return;
    x.t = 0;
    if (++x.blk < x.s.blocks) return;
    x.blk = 0;
    if (++x.h < a.b.hk || !more) return;
    x.h = 0;
    do {
      x.s = kv4_seq<TILE, RB>(a, p.max_rows, ++x.b);
    } while (x.s.blocks == 0 && x.b + 1 < B);
  };
  const int pl2 = min(a.b.ps_log2, TILE == 64 ? 6 : TILE == 32 ? 5 : 4);  // log2 of the keys one copy brings
  const int pieces = TILE >> pl2;
  // Fetches tile `pr` into `stage`: lane i < pieces copies the i-th run of keys that lie in one page.
  auto fetch = [&](int stage) {
    const int key = pr.t * TILE + (lane << pl2);
    const bool want = lane < pieces && key < pr.s.keys;
    int64_t page = -1;
    if (want) page = a.b.table[pr.b * a.b.ld_table + (key >> a.b.ps_log2)];
    const bool ok = want && page >= 0 && page < a.b.pages;
    const unsigned got = __ballot_sync(0xffffffffu, ok), wanted = __ballot_sync(0xffffffffu, want);
    if (lane == 0) {
      vmask[stage] = got | (got != wanted ? 0x80000000u : 0u);
      if (got != wanted) raise_status(kStatusBadIndex);
      mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(__popc(got)) * (static_cast<uint32_t>(D + 8) << pl2));
    }
    __syncwarp();
    if (ok) {
      const int64_t row = ((page * a.b.hk + pr.h) << a.b.ps_log2) + (key & ((1 << a.b.ps_log2) - 1));
      uint8_t* st = ring + stage * C::kStage;
      const uint32_t cb = static_cast<uint32_t>(D / 2) << pl2, ab = 4u << pl2;
      bulk_load_g2s(st + lane * cb, a.b.kc + row * (D / 2), cb, &full[stage]);
      bulk_load_g2s(st + C::kCodes + lane * cb, a.b.vc + row * (D / 2), cb, &full[stage]);
      bulk_load_g2s(st + 2 * C::kCodes + lane * ab, a.b.ka + row, ab, &full[stage]);
      bulk_load_g2s(st + 2 * C::kCodes + TILE * 4 + lane * ab, a.b.va + row, ab, &full[stage]);
    }
  };
  int64_t fetched = 0;
  for (; fetched < STAGES && fetched < count; ++fetched) {
    fetch(static_cast<int>(fetched));
    advance(pr, fetched + 1 < count);
  }

  float o[NT][D / 16][4], ones[NT][4], mx[NT][2], l[NT][2], low[NT][2], sumq[NT][2];
  uint32_t qf[NT][W4][4];
  int lim[NT][2], min_lim = 0, t0 = 0;
  bool failed = false;
  int stage = 0;
  uint32_t parity = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int rows = c.s.n * a.group;  // at most max_rows, or of a sequence whose rows fit 31 bits
    const int r0 = c.blk * RB;
    if (i == 0 || c.t == 0) {
      // ---- a run (or the rest of one) begins: its queries, in the lane order of the codes
      t0 = c.t;
      min_lim = INT_MAX;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + g;
        float sum = 0.f;
        const T* src = static_cast<const T*>(a.q) + (c.s.q0 + static_cast<int64_t>(r / a.group)) * a.q_t +
                       (static_cast<int64_t>(c.h) * a.group + r % a.group) * a.q_h + q * (D / 4);
#pragma unroll
        for (int w = 0; w < W4; ++w) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r < rows) v = *reinterpret_cast<const uint4*>(src + 8 * w);
          const float2 f0 = unpack2<T>(v.x), f1 = unpack2<T>(v.y), f2 = unpack2<T>(v.z), f3 = unpack2<T>(v.w);
          sum += ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
          qf[nt][w][0] = __byte_perm(v.x, v.z, 0x5410);  // elements 0, 4
          qf[nt][w][1] = __byte_perm(v.x, v.z, 0x7632);  // 1, 5
          qf[nt][w][2] = __byte_perm(v.y, v.w, 0x5410);  // 2, 6
          qf[nt][w][3] = __byte_perm(v.y, v.w, 0x7632);  // 3, 7
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sumq[nt][j] = __shfl_sync(0xffffffffu, sum, (2 * q + j) * 4);
          const int rr = r0 + nt * 8 + 2 * q + j;
          // keys the row sees: positions up to its own
          lim[nt][j] = rr < rows ? min(c.s.keys, c.s.len - c.s.n + rr / a.group + 1) : c.s.keys;
          min_lim = min(min_lim, lim[nt][j]);
          mx[nt][j] = -INFINITY;
          l[nt][j] = low[nt][j] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) ones[nt][e] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][d][e] = 0.f;
      }
      min_lim = min(min_lim, __shfl_xor_sync(0xffffffffu, min_lim, 1));
      min_lim = min(min_lim, __shfl_xor_sync(0xffffffffu, min_lim, 2));
    }

    if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], parity, nullptr))) {
      failed = true;
      break;
    }
    const uint8_t* st = ring + stage * C::kStage;
    const uint32_t* kaff = reinterpret_cast<const uint32_t*>(st + 2 * C::kCodes);
    const uint32_t* vaff = kaff + TILE;
    const uint32_t have = vmask[stage];
    const int key0 = c.t * TILE;
    const bool masked = key0 + TILE > min_lim || (have & 0x80000000u);

    // ---- scores of the tile: s[nt][kb][.]: keys 16 kb + g (0, 1) and + 8 (2, 3), rows 2q (0, 2) and 2q + 1
    float s[NT][KB][4];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      uint32_t w0[W4], w1[W4];
      const uint8_t* kr = st + (16 * kb + g) * (D / 2) + q * (D / 8);
      if constexpr (D == 128) {
        const uint4 x = *reinterpret_cast<const uint4*>(kr), y = *reinterpret_cast<const uint4*>(kr + 8 * (D / 2));
        w0[0] = x.x, w0[1] = x.y, w0[2] = x.z, w0[3] = x.w;
        w1[0] = y.x, w1[1] = y.y, w1[2] = y.z, w1[3] = y.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(kr), y = *reinterpret_cast<const uint2*>(kr + 8 * (D / 2));
        w0[0] = x.x, w0[1] = x.y;
        w1[0] = y.x, w1[1] = y.y;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][kb][e] = 0.f;
#pragma unroll
      for (int w = 0; w < W4; ++w) {
        const uint32_t a0[4] = {kv4_pair<T, 0>(w0[w]), kv4_pair<T, 0>(w1[w]), kv4_pair<T, 1>(w0[w]), kv4_pair<T, 1>(w1[w])};
        const uint32_t a1[4] = {kv4_pair<T, 2>(w0[w]), kv4_pair<T, 2>(w1[w]), kv4_pair<T, 3>(w0[w]), kv4_pair<T, 3>(w1[w])};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          M::mma(s[nt][kb], a0, qf[nt][w][0], qf[nt][w][1]);
          M::mma(s[nt][kb], a1, qf[nt][w][2], qf[nt][w][3]);
        }
      }
      const float2 k0 = unpack2<T>(kaff[16 * kb + g]), k1 = unpack2<T>(kaff[16 * kb + 8 + g]);
      const float m0 = 16.f * a.scale_log2 * k0.x, m1 = 16.f * a.scale_log2 * k1.x;
      const float c0 = fmaf(a.scale_log2, k0.y, -m0), c1 = fmaf(a.scale_log2, k1.y, -m1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s[nt][kb][0] = fmaf(s[nt][kb][0], m0, c0 * sumq[nt][0]);
        s[nt][kb][1] = fmaf(s[nt][kb][1], m0, c0 * sumq[nt][1]);
        s[nt][kb][2] = fmaf(s[nt][kb][2], m1, c1 * sumq[nt][0]);
        s[nt][kb][3] = fmaf(s[nt][kb][3], m1, c1 * sumq[nt][1]);
      }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = 16 * kb + 8 * j + g;
          const bool here = (have >> (at >> pl2)) & 1u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (!here || key0 + at >= lim[nt][x]) s[nt][kb][2 * j + x] = -INFINITY;
        }
      }
    }

    // ---- running maximum; earlier sums follow it
    float base[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float al[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float m = fmaxf(s[nt][0][x], s[nt][0][2 + x]);
#pragma unroll
        for (int kb = 1; kb < KB; ++kb) m = fmaxf(m, fmaxf(s[nt][kb][x], s[nt][kb][2 + x]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        m = fmaxf(m, mx[nt][x]);
        base[nt][x] = m == -INFINITY ? 0.f : m;
        al[x] = ex2(mx[nt][x] - base[nt][x]);
        mx[nt][x] = m;
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          l[nt][x] *= al[x];
          low[nt][x] *= al[x];
          ones[nt][x] *= al[x];
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[nt][d][x] *= al[x];
            o[nt][d][2 + x] *= al[x];
          }
        }
      }
    }

    // ---- weights, and the output's products
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const float2 v0 = unpack2<T>(vaff[16 * kb + g]), v1 = unpack2<T>(vaff[16 * kb + 8 + g]);
      uint32_t bf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pe = ex2(s[nt][kb][e] - base[nt][e & 1]);
          const float2 va = e < 2 ? v0 : v1;
          l[nt][e & 1] += pe;
          w[e] = pe * (M::kF * va.x);
          float lo = pe * va.y;
          // a key the row does not see may hold anything, NaN included
          if (masked && s[nt][kb][e] == -INFINITY) w[e] = lo = 0.f;
          low[nt][e & 1] += lo;
        }
        bf[nt][0] = movmatrix_trans(pack2<T>(w[0], w[1]));
        bf[nt][1] = movmatrix_trans(pack2<T>(w[2], w[3]));
        const uint32_t one[4] = {M::kOne, M::kOne, M::kOne, M::kOne};
        M::mma(ones[nt], one, bf[nt][0], bf[nt][1]);
      }
      // keys 2q, 2q + 1 and 2q + 8, 2q + 9 of the block; D/8 dims from D/8 * g
      const uint8_t* vr = st + C::kCodes + (16 * kb + 2 * q) * (D / 2) + g * (D / 16);
      uint32_t x[4][D / 64];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* vk = vr + ((j & 1) + 8 * (j >> 1)) * (D / 2);
        if constexpr (D == 128) {
          const uint2 y = *reinterpret_cast<const uint2*>(vk);
          x[j][0] = y.x, x[j][1] = y.y;
        } else {
          x[j][0] = *reinterpret_cast<const uint32_t*>(vk);
        }
      }
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {
        // elements 0..3 (then 4..7) of the word, keys 2q | 2q + 1 and 2q + 8 | 2q + 9
        const uint32_t e0 = __byte_perm(x[0][w], x[1][w], 0x5410), e1 = __byte_perm(x[2][w], x[3][w], 0x5410);
        const uint32_t f0 = __byte_perm(x[0][w], x[1][w], 0x7632), f1 = __byte_perm(x[2][w], x[3][w], 0x7632);
        const uint32_t a0[4] = {kv4_pair<T, 0>(e0), kv4_pair<T, 1>(e0), kv4_pair<T, 0>(e1), kv4_pair<T, 1>(e1)};
        const uint32_t a1[4] = {kv4_pair<T, 2>(e0), kv4_pair<T, 3>(e0), kv4_pair<T, 2>(e1), kv4_pair<T, 3>(e1)};
        const uint32_t a2[4] = {kv4_pair<T, 0>(f0), kv4_pair<T, 1>(f0), kv4_pair<T, 0>(f1), kv4_pair<T, 1>(f1)};
        const uint32_t a3[4] = {kv4_pair<T, 2>(f0), kv4_pair<T, 3>(f0), kv4_pair<T, 2>(f1), kv4_pair<T, 3>(f1)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          M::mma(o[nt][4 * w + 0], a0, bf[nt][0], bf[nt][1]);
          M::mma(o[nt][4 * w + 1], a1, bf[nt][0], bf[nt][1]);
          M::mma(o[nt][4 * w + 2], a2, bf[nt][0], bf[nt][1]);
          M::mma(o[nt][4 * w + 3], a3, bf[nt][0], bf[nt][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (fetched < count) {
      fetch(stage);
      ++fetched;
      advance(pr, fetched < count);
    }
    if (++stage == STAGES) stage = 0, parity ^= 1;

    const bool run_ends = c.t + 1 == c.s.tiles;
    if (run_ends || i + 1 == count) {
      // ---- a run (or a piece of one) is done
      const bool whole = t0 == 0 && run_ends;
      const int slot = t0 > 0 ? 0 : 1;
      float* dst = reinterpret_cast<float*>(slot == 0 ? first_all + warp * C::kPiece : ring);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float ls = l[nt][x], lw = low[nt][x];
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) {
            ls += __shfl_xor_sync(0xffffffffu, ls, sh);
            lw += __shfl_xor_sync(0xffffffffu, lw, sh);
          }
          const int row = nt * 8 + 2 * q + x, rr = r0 + row;
          constexpr float f = 16.f / M::kF;
          const float inv = whole ? (ls == 0.f ? 0.f : 1.f / ls) : 1.f;
          float y[D / 8];
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            y[2 * d] = fmaf(f, o[nt][d][x] - ones[nt][x], lw) * inv;
            y[2 * d + 1] = fmaf(f, o[nt][d][2 + x] - ones[nt][x], lw) * inv;
          }
          if (whole) {
            if (rr < rows) {
              T* out = static_cast<T*>(a.out) +
                       ((c.s.q0 + static_cast<int64_t>(rr / a.group)) * a.hq + c.h * a.group + rr % a.group) * D + g * (D / 8);
#pragma unroll
              for (int d = 0; d < D / 8; d += 8)
                *reinterpret_cast<uint4*>(out + d) = make_uint4(pack2<T>(y[d], y[d + 1]), pack2<T>(y[d + 2], y[d + 3]),
                                                                pack2<T>(y[d + 4], y[d + 5]), pack2<T>(y[d + 6], y[d + 7]));
            }
          } else {
#pragma unroll
            for (int d = 0; d < D / 8; d += 4)
              *reinterpret_cast<float4*>(dst + row * D + g * (D / 8) + d) = make_float4(y[d], y[d + 1], y[d + 2], y[d + 3]);
            if (g == 0) {
              dst[RB * D + row] = mx[nt][x];
              dst[RB * D + RB + row] = ls;
            }
          }
        }
      if (!whole && lane == 0) {
        int* pc = piece[2 * warp + slot];
        pc[1] = t0 == 0;
        pc[2] = run_ends;
        pc[3] = c.b, pc[4] = c.h, pc[5] = c.blk;
        pc[0] = 1;
      }
    }
    advance(c, i + 1 < count);
  }
  if (failed) {  // a copy never came: let the others land (or give up on them too) before the memory goes
    for (int k = 0; k < STAGES; ++k) {
      if (++stage == STAGES) stage = 0, parity ^= 1;
      mbar_wait(&full[stage], parity, nullptr);
    }
  }
  __syncthreads();

  // ---- pieces of cut runs: lane i holds piece i; equal neighbours are one run
  const bool have = lane < 2 * WARPS && piece[lane][0];
  const unsigned all = __ballot_sync(0xffffffffu, have);
  const unsigned lower = all & ((1u << lane) - 1);
  bool opens = have;
  if (have && lower) {
    const int* x = piece[lane];
    const int* y = piece[31 - __clz(lower)];
    opens = x[3] != y[3] || x[4] != y[4] || x[5] != y[5];
  }
  const unsigned open = __ballot_sync(0xffffffffu, opens);
  const int runs = __popc(open);
  if (tid == 0) {
    int* d = p.desc + blockIdx.x * 8;
    d[0] = d[2] = 0;
  }
  __syncthreads();
  for (int item = warp; item < runs * RB; item += WARPS) {
    const int row = item % RB;
    unsigned rest = open;
    for (int k = item / RB; k; --k) rest &= rest - 1;
    const int head = __ffs(rest) - 1;
    const unsigned later = rest & (rest - 1);
    const unsigned group = all & ~((1u << head) - 1) & (later ? (later & -later) - 1 : ~0u);
    const int tail = 31 - __clz(group);
    auto data = [&](int i) {
      return reinterpret_cast<const float*>(i & 1 ? kv4_smem + (i >> 1) * C::kRing : first_all + (i >> 1) * C::kPiece);
    };
    float m = -INFINITY;
    for (unsigned x = group; x; x &= x - 1) m = fmaxf(m, data(__ffs(x) - 1)[RB * D + row]);
    const float mb = m == -INFINITY ? 0.f : m;
    float ls = 0.f, y[W4];
#pragma unroll
    for (int d = 0; d < W4; ++d) y[d] = 0.f;
    for (unsigned x = group; x; x &= x - 1) {
      const float* src = data(__ffs(x) - 1);
      const float f = ex2(src[RB * D + row] - mb);
      ls = fmaf(src[RB * D + RB + row], f, ls);
#pragma unroll
      for (int d = 0; d < W4; ++d) y[d] = fmaf(src[row * D + lane * W4 + d], f, y[d]);
    }
    const int* hd = piece[head];
    const bool starts = hd[1], ends = piece[tail][2];
    if (starts && ends) {
      const Kv4Seq sq = kv4_seq<TILE, RB>(a, p.max_rows, hd[3]);
      const int rr = hd[5] * RB + row;
      if (rr < sq.n * a.group) {
        T* out = static_cast<T*>(a.out) +
                 ((sq.q0 + static_cast<int64_t>(rr / a.group)) * a.hq + hd[4] * a.group + rr % a.group) * D + lane * W4;
        const float inv = ls == 0.f ? 0.f : 1.f / ls;
#pragma unroll
        for (int d = 0; d < W4; d += 2) *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(y[d] * inv, y[d + 1] * inv);
      }
    } else {
      const int slot = starts ? 1 : 0;
      float* dst = p.ws + (blockIdx.x * 2 + slot) * static_cast<int64_t>(RB * (D + 2));
#pragma unroll
      for (int d = 0; d < W4; ++d) dst[row * D + lane * W4 + d] = y[d];
      if (lane == 0) {
        dst[RB * D + row] = m;
        dst[RB * D + RB + row] = ls;
        if (row == 0) {
          int* ds = p.desc + blockIdx.x * 8;
          if (slot == 0) {
            ds[1] = ends;
            ds[0] = 1;
          } else {
            ds[3] = hd[3], ds[4] = hd[4], ds[5] = hd[5];
            ds[2] = 1;
          }
        }
      }
    }
  }
}

// Joins the pieces of the runs cut by CTA borders: CTA i takes the run that starts in (and runs out of) CTA
// i of the first kernel. A warp per row, pieces in order.
template <typename T, int D, int RB, int TILE>
__global__ void __launch_bounds__(256) kv4_decode_join(const Kv4DecodeParams p, int parts) {
  constexpr int W4 = D / 32;
  const Kv4AttnParams& a = p.a;
  const int* d0 = p.desc + blockIdx.x * 8;
  if (!d0[2]) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int last = blockIdx.x;
  for (int i = blockIdx.x + 1; i < parts; ++i) {
    if (!p.desc[i * 8]) break;
    last = i;
    if (p.desc[i * 8 + 1]) break;
  }
  auto data = [&](int i) {
    return p.ws + (i * 2 + (i == static_cast<int>(blockIdx.x) ? 1 : 0)) * static_cast<int64_t>(RB * (D + 2));
  };
  const int b = d0[3], h = d0[4], blk = d0[5];
  const Kv4Seq sq = kv4_seq<TILE, RB>(a, p.max_rows, b);
  for (int row = warp; row < RB; row += 8) {
    const int rr = blk * RB + row;
    if (rr >= sq.n * a.group) break;
    float m = -INFINITY;
    for (int i = blockIdx.x + lane; i <= last; i += 32) m = fmaxf(m, data(i)[RB * D + row]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float mb = m == -INFINITY ? 0.f : m;
    float ls = 0.f, y[W4];
#pragma unroll
    for (int d = 0; d < W4; ++d) y[d] = 0.f;
#pragma unroll 4
    for (int i = blockIdx.x; i <= last; ++i) {
      const float* src = data(i);
      const float f = ex2(src[RB * D + row] - mb);
      ls = fmaf(src[RB * D + RB + row], f, ls);
#pragma unroll
      for (int d = 0; d < W4; ++d) y[d] = fmaf(src[row * D + lane * W4 + d], f, y[d]);
    }
    const float inv = ls == 0.f ? 0.f : 1.f / ls;
    T* out = static_cast<T*>(a.out) +
             ((sq.q0 + static_cast<int64_t>(rr / a.group)) * a.hq + h * a.group + rr % a.group) * D + lane * W4;
#pragma unroll
    for (int d = 0; d < W4; d += 2) *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(y[d] * inv, y[d + 1] * inv);
  }
}

}  // namespace dscq
