// Attention of few rows per sequence (single tokens, drafts) over the 4-bit paged cache: bound by reading the
// cache once. See kv4_attention.cuh for the operator.
//
// Mathematics. A 4-bit code n in the low bits of an fp16 number is the subnormal n 2^-24 (n 2^-20 four bits up), which
// tensor cores multiply exactly; so an AND (and one shift for every other pair) makes two operands of two codes:
//   q.k = step (q.n) + low sum(q)
//   o   = sum_t P'_t n_t / F + sum_t p_t low_t,   P'_t = fp16(F p_t step_t), F of each row
// and for f16 outputs, which would show the rounding of P' (4e-4 of the result), about the middle code, where it counts
// a third: sum_t P'_t (n_t - 8) / F + sum_t p_t (low_t + 8 step_t), sum_t P'_t from one more product with ones.
// No element is ever dequantised; step and low cost a few operations per key, not per element. Queries
// enter as fp16, each row scaled by a power of two to the top of its range (exact but for elements 2^-29 below
// the row's largest); F is a power of two, a row's own, that falls when one of the row's weights times its step would
// leave fp16: what the row does not see, or hardly weighs, costs it nothing. P' keeps 11 bits down to 2^-26 of the row's
// largest contribution. Scores, softmax statistics and sums are 32-bit; only the weights P' are rounded.
//
// Fragments (mma.m16n8k16). Scores: A = 16 keys x 16 dims, B = 8 query rows; a lane's 32 dims (16 for D = 64)
// of a key are one 16-byte load, any dim order works as long as the queries use the same. Output: A = 16
// dims x 16 keys, B = weights; a lane needs pairs of adjacent KEYS for one dim, which a byte permute of two
// keys' words gives. The weights move from the score layout (key, row) to B's (row, key) by movmatrix.
//
// Work split. All (sequence, key head, block of 8 NT rows) runs are laid end to end as tiles of TILE keys and cut into
// equal shares, one a warp, whatever the lengths; the cut points come from the lengths on the device, so a captured
// launch follows them. A warp streams its share through its own ring of asynchronous copies, across run borders. It
// finishes runs that lie inside its share; pieces of cut runs meet in shared memory once all warps of the
// CTA are done, pieces of runs cut by CTA borders in a second kernel, in order: no atomics, the same bits every time.
//
// Measured on a B200: 64 contexts of 0 to 8191 tokens, 64 heads on 8: 80 us for 287 MB (3.6 TB/s, 0.55 of the copy rate; 78
// with one F for all rows); three of 50 to 65 thousand: 52 us (3.2 TB/s). Twelve warps an SM keep the issue slots and
// the integer pipe half busy with the ANDs, permutes and copies of codes, and a tile's chain of products and exponentials
// does not overlap further: 16 warps (32-key tiles, 128 registers) took 96 us, 8 warps 90, 12 with 32-key tiles 91.
#pragma once
#include "kv4_attention.cuh"
#include "rotq_tc.cuh"

namespace dscq {

struct Kv4DecodeParams {
  Kv4AttnParams a;
  int64_t max_rows;  // sequences with more rows * group than this are not this kernel's
  // A piece of a cut run is [8 NT][D] sums of its rows, then their maxima and weights' sums (32-bit).
  float* cta;        // [G][2] pieces of runs cut by CTA borders
  float* warp;       // [G][WARPS] pieces of runs cut at a warp's start
  int* desc;         // [G][8]: slot 0 {valid, ends}, slot 1 {valid, b, h, block}
  int whole;         // a CTA takes a whole run (the grid holds all of them): no run is cut by a CTA border
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^e as a float, -126 <= e <= 127.
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// floor(log2 x) of a positive normal x.
__device__ __forceinline__ int log2i(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

constexpr uint32_t kEight = 0x00080008u;                          // code 8 twice
constexpr uint32_t kCode0 = 0x000F000Fu, kCode1 = 0x00F000F0u;  // two codes of a word: weights 2^-24 and 2^-20

// One sequence as the decode kernel sees it.
struct Kv4Seq {
  int q0, n, len, tiles, blocks;  // first row, rows, cached tokens (as given), tiles of a run, row blocks
  int keys;                       // cached tokens the page table can hold
  // Keys row i sees: positions up to its own; none (0 or less) where that lies before the first or behind the page table.
  __device__ __forceinline__ int sees(int i) const {
    const int n_keys = len - n + i + 1;
    return n_keys > keys ? 0 : n_keys;
  }
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

// Four rows of a run being put together from its pieces, by one warp: lane's dims are D/32 from lane * D/32.
template <int D>
struct Kv4Joined {
  static constexpr int E = D / 32;
  float m[4], l[4], y[4][E];
  // Pieces `which` (bits), at(i) giving piece i: lane i weighs piece i, then all add them up.
  template <class At>
  __device__ __forceinline__ void join(unsigned which, At at, int RB, int row0, int lane) {
    float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, pl[4] = {0.f, 0.f, 0.f, 0.f}, f[4];
    if (which >> lane & 1u) {
      const float* piece = at(lane);
      const float4 a = *reinterpret_cast<const float4*>(piece + RB * D + row0);
      const float4 b = *reinterpret_cast<const float4*>(piece + RB * D + RB + row0);
      pm[0] = a.x, pm[1] = a.y, pm[2] = a.z, pm[3] = a.w;
      pl[0] = b.x, pl[1] = b.y, pl[2] = b.z, pl[3] = b.w;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = pm[r];
#pragma unroll
      for (int o = 16; o; o >>= 1) m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], o));
      f[r] = ex2(pm[r] - (m[r] == -INFINITY ? 0.f : m[r]));
      l[r] = pl[r] * f[r];
#pragma unroll
      for (int o = 16; o; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
#pragma unroll
      for (int e = 0; e < E; ++e) y[r][e] = 0.f;
    }
    for (unsigned x = which; x; x &= x - 1) {
      const int i = __ffs(x) - 1;
      const float* src = at(i) + row0 * D + lane * E;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float g = __shfl_sync(0xffffffffu, f[r], i);
        float v[E];
        if constexpr (E == 4) {
          const float4 u = *reinterpret_cast<const float4*>(src + r * D);
          v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else {
          const float2 u = *reinterpret_cast<const float2*>(src + r * D);
          v[0] = u.x, v[1] = u.y;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) y[r][e] = fmaf(v[e], g, y[r][e]);
      }
    }
  }
  // The same with `other`, earlier pieces first.
  __device__ __forceinline__ void add(const Kv4Joined& other) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float n = fmaxf(m[r], other.m[r]), nb = n == -INFINITY ? 0.f : n;
      const float f = ex2(m[r] - nb), g = ex2(other.m[r] - nb);
      m[r] = n;
      l[r] = fmaf(l[r], f, other.l[r] * g);
#pragma unroll
      for (int e = 0; e < E; ++e) y[r][e] = fmaf(y[r][e], f, other.y[r][e] * g);
    }
  }
  __device__ __forceinline__ void store(float* piece, int RB, int row0, int lane) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int e = 0; e < E; ++e) piece[(row0 + r) * D + lane * E + e] = y[r][e];
      if (lane == r) {
        piece[RB * D + row0 + r] = m[r];
        piece[RB * D + RB + row0 + r] = l[r];
      }
    }
  }
  // Rows rr .. rr + 3 of sequence sq and key head h.
  template <typename T>
  __device__ __forceinline__ void write(const Kv4AttnParams& a, const Kv4Seq& sq, int h, int rr, int lane) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (rr + r >= sq.n * a.group) break;
      T* out = static_cast<T*>(a.out) + ((sq.q0 + static_cast<int64_t>(a.row_token(rr + r))) * a.hq + h * a.group +
                                         rr + r - a.row_token(rr + r) * a.group) * D + lane * E;
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
      for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(out + e) = pack2<T>(y[r][e] * inv, y[r][e + 1] * inv);
    }
  }
};

template <int D_, int NT_, int WARPS_, int STAGES_, int TILE_>
struct Kv4DecodeConfig {
  static constexpr int D = D_, NT = NT_, WARPS = WARPS_, STAGES = STAGES_, TILE = TILE_;
  static constexpr int RB = 8 * NT;                       // rows of a block
  static constexpr int kCodes = TILE * D / 2;             // bytes of one side's codes in a stage
  static constexpr int kStage = 2 * kCodes + 2 * TILE * 4;
  static constexpr int kRing = STAGES * kStage;
  static constexpr int kPiece = RB * (D + 2);             // floats of a cut run's piece
  static constexpr int kSmem = WARPS * kRing + WARPS * STAGES * 12;
  static constexpr int64_t workspace(int64_t parts) { return parts * ((2 + WARPS) * kPiece * 4 + 32); }
  static_assert(kRing >= kPiece * 4, "the last piece of a warp goes into its ring");
  static_assert(2 * WARPS <= 32 && kStage % 16 == 0 && kPiece % 4 == 0, "layout");
};

template <typename T, class C>
__global__ void __launch_bounds__(C::WARPS * 32, 1) kv4_decode_kernel(const Kv4DecodeParams p) {
  constexpr int D = C::D, NT = C::NT, TILE = C::TILE, WARPS = C::WARPS, STAGES = C::STAGES, RB = C::RB;
  constexpr int KB = TILE / 16;  // 16-key blocks of a tile
  constexpr int W4 = D / 32;     // words of codes a lane takes of a key
  constexpr bool kMid = std::is_same<T, __half>::value;  // codes about 8
  const Kv4AttnParams& a = p.a;
  extern __shared__ __align__(128) uint8_t kv4_smem[];
  float* first_all = p.warp + blockIdx.x * static_cast<int64_t>(WARPS * C::kPiece);
  uint64_t* bars = reinterpret_cast<uint64_t*>(kv4_smem + WARPS * C::kRing);
  uint32_t* vmask_all = reinterpret_cast<uint32_t*>(bars + WARPS * STAGES);
  __shared__ int64_t scan[WARPS];
  __shared__ int64_t tiles_before[WARPS * 32];  // of each thread's sequences
  __shared__ int piece[2 * WARPS][6];  // where (0: none), starts, ends, b, h, block; pieces 2w (cut at its start), 2w + 1

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  uint8_t* ring = kv4_smem + warp * C::kRing;
  uint64_t* full = bars + warp * STAGES;
  uint32_t* vmask = vmask_all + warp * STAGES;
  if (lane < STAGES) {
    mbar_init(&full[lane], 32);
    fence_mbar_init();
  }
  if (tid < 2 * WARPS) piece[tid][0] = 0;

  const int B = a.b.B;
  // Adds up what all sequences hold (tiles, or runs where a CTA takes a whole one) and finds the warp's share: the
  // sequences [s_lo, s_hi) its first tile is in, `left` tiles (runs) from the start of the first. Up to 256 sequences
  // every warp does it alone, more are added up by the whole CTA.
  auto units_of = [&](const Kv4Seq& r) {
    return static_cast<int64_t>(r.blocks) * a.b.hk * (p.whole ? 1 : r.tiles);
  };
  auto scan32 = [&](int64_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  const bool alone = B <= 256;
  const int adders = alone ? 32 : WARPS * 32, adder = alone ? lane : tid;
  const int per = (B + adders - 1) / adders;
  int64_t mine = 0;
  Kv4Seq held{};  // the adder's (last) sequence
  for (int s = min(adder * per, B); s < min(adder * per + per, B); ++s) {
    held = kv4_seq<TILE, RB>(a, p.max_rows, s);
    mine += units_of(held);
  }
  const int64_t incl = scan32(mine);
  int64_t total, before = incl - mine;
  if (alone) {
    total = __shfl_sync(0xffffffffu, incl, 31);
  } else {
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w == warp) before += total;
      total += scan[w];
    }
    tiles_before[tid] = before;
    __syncthreads();
  }
  // Equal shares: warp g of the launch begins at tile g * base + min(g, extra). A warp has at least one tile
  // where there are enough; CTAs beyond that have none.
  const int parts = static_cast<int>(max(min(total / WARPS, static_cast<int64_t>(gridDim.x)), static_cast<int64_t>(1)));
  const int shares = parts * WARPS;
  const int64_t base = total >> 32 ? total / shares : static_cast<uint32_t>(total) / static_cast<uint32_t>(shares);
  const int extra = static_cast<int>(total - base * shares);
  const int gw = blockIdx.x * WARPS + warp;
  int count = gw < shares ? static_cast<int>(base) + (gw < extra) : 0;
  struct Cursor {
    int b, h, blk, t;
    Kv4Seq s;
  };
  Cursor c{};
  if (p.whole ? static_cast<int64_t>(blockIdx.x) < total : count > 0) {
    int64_t left = p.whole ? static_cast<int64_t>(blockIdx.x) : gw * base + min(gw, extra);
    int th;
    if (alone) {
      th = 31 - __clz(__ballot_sync(0xffffffffu, before <= left));
      left -= __shfl_sync(0xffffffffu, before, th);
    } else {
      unsigned le = __ballot_sync(0xffffffffu, tiles_before[lane * WARPS] <= left);
      th = (31 - __clz(le)) * WARPS;
      le = __ballot_sync(0xffffffffu, lane < WARPS && tiles_before[th + (lane < WARPS ? lane : 0)] <= left);
      th += 31 - __clz(le);
      left -= tiles_before[th];
    }
    const int s_hi = min(th * per + per, B);
    auto take = [&](const Kv4Seq& r, int src) {
      c.s.q0 = __shfl_sync(0xffffffffu, r.q0, src);
      c.s.n = __shfl_sync(0xffffffffu, r.n, src);
      c.s.len = __shfl_sync(0xffffffffu, r.len, src);
      c.s.tiles = max(__shfl_sync(0xffffffffu, r.tiles, src), 1);
      c.s.blocks = max(__shfl_sync(0xffffffffu, r.blocks, src), 1);
      c.s.keys = __shfl_sync(0xffffffffu, r.keys, src);
    };
    if (alone && per == 1) {
      c.b = th;
      take(held, th);
    }
    for (int s0 = th * per; !(alone && per == 1); s0 += 32) {
      Kv4Seq r{};
      if (s0 + lane < s_hi) r = kv4_seq<TILE, RB>(a, p.max_rows, s0 + lane);
      const int64_t units = units_of(r), upto = scan32(units);
      const unsigned past = __ballot_sync(0xffffffffu, upto > left);
      if (!past && s0 + 32 < s_hi) {
        left -= __shfl_sync(0xffffffffu, upto, 31);
        continue;
      }
      const int src = past ? __ffs(past) - 1 : 31;
      left -= __shfl_sync(0xffffffffu, upto - units, src);
      c.b = s0 + src;
      take(r, src);
      break;
    }
    int64_t run = left;
    if (p.whole) {
      const int n = c.s.tiles / WARPS, more = c.s.tiles % WARPS;
      count = n + (warp < more);
      c.t = warp * n + min(warp, more);
    } else {
      run = left >> 32 ? left / c.s.tiles : static_cast<uint32_t>(left) / static_cast<uint32_t>(c.s.tiles);
      c.t = static_cast<int>(left - run * c.s.tiles);
    }
    c.h = static_cast<int>(run >> 32 ? run / c.s.blocks : static_cast<uint32_t>(run) / static_cast<uint32_t>(c.s.blocks));
    c.blk = static_cast<int>(run - static_cast<int64_t>(c.h) * c.s.blocks);
  } else {
    count = 0;
  }
  // sequences that share rows can have more runs than the grid was made for
  if (p.whole && total > gridDim.x && tid == 0) raise_status(kStatusBadIndex);
  if (alone) __syncthreads();  // the barriers and pieces set up above
  Cursor pr = c;  // the tile to fetch next
  auto advance = [&](Cursor& x, bool more) {  // more: there is a tile behind this one
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
  // A tile's keys lie in `pieces` runs of one page each. Lane i < pieces looks up the page of run i of the next tile
  // while the current one is worked on; then all lanes copy, 16 bytes each (one bulk copy per run and array instead, whose
  // operands a divergent lane hands over one lane at a time: 78.8 us for 64 contexts of 4100 tokens, against 78.3).
  constexpr int kRows = 512 / (D / 2);  // keys a copy of the warp brings
  int page = -1;
  bool want = false;
  auto look = [&] {
    const int key = pr.t * TILE + (lane << pl2);
    want = lane < pieces && key < pr.s.keys;
    page = want ? a.b.table[pr.b * a.b.ld_table + (key >> a.b.ps_log2)] : -1;
  };
  auto fetch = [&](int stage) {
    const bool ok = want && page >= 0 && page < a.b.pages;
    const unsigned got = __ballot_sync(0xffffffffu, ok);
    const bool all = got == __ballot_sync(0xffffffffu, want);
    if (lane == 0) {
      vmask[stage] = got | (all ? 0u : 0x80000000u);
      if (!all) raise_status(kStatusBadIndex);
    }
    const uint32_t st = smem_u32(ring + stage * C::kStage) + lane * 16;
    for (int i = 0; i < pieces; ++i) {
      const int pg = __shfl_sync(0xffffffffu, page, i);
      if (!(got >> i & 1u)) continue;
      const int in_page = (pr.t * TILE + (i << pl2)) & ((1 << a.b.ps_log2) - 1);
      const int64_t row = ((static_cast<int64_t>(pg) * a.b.hk + pr.h) << a.b.ps_log2) + in_page;
      const uint8_t *k = a.b.kc + row * (D / 2) + lane * 16, *v = a.b.vc + row * (D / 2) + lane * 16;
      const uint32_t to = st + (i << pl2) * (D / 2);
      if (pl2 == 6) {
#pragma unroll
        for (int j = 0; j < 64 / kRows; ++j) {
          copy16(to + j * 512, k + j * 512);
          copy16(to + C::kCodes + j * 512, v + j * 512);
        }
      } else {
        for (int j = 0; j < (1 << pl2) / kRows; ++j) {
          copy16(to + j * 512, k + j * 512);
          copy16(to + C::kCodes + j * 512, v + j * 512);
        }
      }
      // steps and lows: the low half of the warp for the keys, the high half for the values
      const int l16 = lane & 15;
      if (l16 < (1 << pl2) / 4)
        copy16(st - lane * 16 + 2 * C::kCodes + (lane < 16 ? 0 : TILE * 4) + (i << pl2) * 4 + l16 * 16,
               (lane < 16 ? a.b.ka : a.b.va) + row + l16 * 4);
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[stage])) : "memory");
    __syncwarp();
  };
  int fetched = 0;
  if (count > 0) look();
  auto fetch_next = [&](int stage) {
    fetch(stage);
    if (++fetched < count) {
      advance(pr, true);
      look();
    }
  };
  if (count > 0) fetch_next(0);

  // Rows of no sequence are zero.
  {
    const int lo = B ? min(max(a.b.q_start[0], 0), a.T) : 0, hi = B ? min(max(a.b.q_start[B], lo), a.T) : 0;
    const int64_t row16 = static_cast<int64_t>(a.hq) * D / 8;  // 16-byte pieces of a row
    const int64_t none = (lo + a.T - hi) * row16;
    for (int64_t i = blockIdx.x * (WARPS * 32ll) + tid; i < none; i += gridDim.x * (WARPS * 32ll)) {
      const int64_t r = i < lo * row16 ? i : i - lo * row16 + hi * row16;
      reinterpret_cast<uint4*>(a.out)[r] = make_uint4(0, 0, 0, 0);
    }
  }

  // mx is the running maximum of the scores in their rows' own units, c1 turns those into powers of two
  float o[NT][D / 16][4], ones[NT][4], mx[NT][2], l[NT][2], low[NT][2], sumq[NT][2], c1[NT][2];
  uint32_t qf[NT][W4][4];
  int lim[NT][2], min_lim = 0, max_lim = 0, t0 = 0;
  float F[NT][2], cap = 0.f;  // F of the rows, powers of two; steps below cap cannot leave fp16 under any of them
  bool failed = false;
  int stage = 0;
  uint32_t parity = 0;
  for (int i = 0; i < count; ++i) {
    const int rows = c.s.n * a.group;  // at most max_rows, or of a sequence whose rows fit 31 bits
    const int r0 = c.blk * RB;
    if (i == 0 || c.t == 0) {
      // ---- a run (or the rest of one) begins: its queries, in the lane order of the codes
      t0 = c.t;
      min_lim = INT_MAX;
      max_lim = 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + g;
        const int tok = a.row_token(r);
        const T* src = static_cast<const T*>(a.q) + (c.s.q0 + static_cast<int64_t>(tok)) * a.q_t +
                       (static_cast<int64_t>(c.h) * a.group + (r - tok * a.group)) * a.q_h + q * (D / 4);
        float x[W4][8], sum = 0.f, big = 0.f;
#pragma unroll
        for (int w = 0; w < W4; ++w) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r < rows) v = *reinterpret_cast<const uint4*>(src + 8 * w);
          kv4_unpack8<T>(v, x[w]);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum += x[w][e];
            big = fmaxf(big, fabsf(x[w][e]));
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // the row's largest element goes to [2^14, 2^15); a negative scale turns the queries around
        const int k = big > 0.f && big < INFINITY ? min(max(14 - log2i(big), -90), 120) : 0;
        const float qs = a.scale_log2 == 0.f ? 0.f : copysignf(pow2f(k), a.scale_log2);
#pragma unroll
        for (int w = 0; w < W4; ++w)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = e & 1 ? qs * 0.0625f : qs;  // codes four bits up count sixteenfold
            qf[nt][w][e] = pack2<__half>(x[w][e] * f, x[w][e + 4] * f);
          }
        // never 0: a masked score of -inf stays one
        const float sq = sum * qs * 0x1p-24f;
        const float cc = a.scale_log2 == 0.f ? 1.f : fmaxf(fabsf(a.scale_log2) * pow2f(24 - k), 0x1p-126f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sumq[nt][j] = __shfl_sync(0xffffffffu, sq, (2 * q + j) * 4);
          c1[nt][j] = __shfl_sync(0xffffffffu, cc, (2 * q + j) * 4);
          const int rr = r0 + nt * 8 + 2 * q + j;
          lim[nt][j] = rr < rows ? c.s.sees(a.row_token(rr)) : 0;
          min_lim = min(min_lim, rr < rows ? lim[nt][j] : c.s.keys);
          max_lim = max(max_lim, lim[nt][j]);
          mx[nt][j] = -INFINITY;
          l[nt][j] = low[nt][j] = 0.f;
          F[nt][j] = lim[nt][j] > 0 ? 0x1p100f : 0x1p-100f;  // the first tile brings it down
        }
        cap = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) ones[nt][e] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][d][e] = 0.f;
      }
#pragma unroll
      for (int sh = 1; sh < 4; sh <<= 1) {
        min_lim = min(min_lim, __shfl_xor_sync(0xffffffffu, min_lim, sh));
        max_lim = max(max_lim, __shfl_xor_sync(0xffffffffu, max_lim, sh));
      }
    }

    // the first tiles of all warps before the others
    if (i == 0)
      while (fetched < STAGES && fetched < count) fetch_next(fetched);

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

    // ---- the values' steps, of either sign
    uint32_t va[KB][2];
    float vmax = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int j = 0; j < 2; ++j) va[kb][j] = vaff[16 * kb + 8 * j + g];
    bool poison = false;  // keys some rows see and others do not, with values that are no numbers
    if (masked) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = 16 * kb + 8 * j + g;
          // what no row sees may hold anything
          if (key0 + at >= max_lim || !((have >> (at >> pl2)) & 1u)) va[kb][j] = 0;
          const float2 f = unpack2<T>(va[kb][j]);
          poison |= !isfinite(f.x) || !isfinite(f.y);
        }
      poison = __any_sync(0xffffffffu, poison);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      vmax = fmax3(vmax, fabsf(unpack2<T>(va[kb][0]).x), fabsf(unpack2<T>(va[kb][1]).x));

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
        const uint32_t u0 = w0[w] >> 8, u1 = w1[w] >> 8;
        const uint32_t a0[4] = {w0[w] & kCode0, w1[w] & kCode0, w0[w] & kCode1, w1[w] & kCode1};
        const uint32_t a1[4] = {u0 & kCode0, u1 & kCode0, u0 & kCode1, u1 & kCode1};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(s[nt][kb], a0, qf[nt][w][0], qf[nt][w][1]);
          mma_f16(s[nt][kb], a1, qf[nt][w][2], qf[nt][w][3]);
        }
      }
      const float2 k0 = unpack2<T>(kaff[16 * kb + g]), k1 = unpack2<T>(kaff[16 * kb + 8 + g]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        s[nt][kb][0] = fmaf(s[nt][kb][0], k0.x, k0.y * sumq[nt][0]);
        s[nt][kb][1] = fmaf(s[nt][kb][1], k0.x, k0.y * sumq[nt][1]);
        s[nt][kb][2] = fmaf(s[nt][kb][2], k1.x, k1.y * sumq[nt][0]);
        s[nt][kb][3] = fmaf(s[nt][kb][3], k1.x, k1.y * sumq[nt][1]);
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
        float m = mx[nt][x];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) m = fmax3(m, s[nt][kb][x], s[nt][kb][2 + x]);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        base[nt][x] = m == -INFINITY ? 0.f : m * c1[nt][x];
        al[x] = mx[nt][x] == m ? 1.f : ex2(fmaf(mx[nt][x], c1[nt][x], -base[nt][x]));
        mx[nt][x] = m;
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          l[nt][x] *= al[x];
          low[nt][x] *= al[x];
          if constexpr (kMid) ones[nt][x] *= al[x];
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[nt][d][x] *= al[x];
            o[nt][d][2 + x] *= al[x];
          }
        }
      }
    }

    // ---- steps larger than any before under some row's F (seldom behind the first tile): rows whose weights they would
    // take out of fp16 lower theirs, so that the largest is in [2^12, 2^13) and steps may still grow fourfold
    if (__any_sync(0xffffffffu, vmax >= cap)) {
      float top = 0.f;  // the largest F
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float w = 0.f;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              w = fmaxf(w, ex2(fmaf(s[nt][kb][2 * j + x], c1[nt][x], -base[nt][x])) * fabsf(unpack2<T>(va[kb][j]).x));
          w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 4));
          w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 8));
          w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 16));
          if (w * F[nt][x] >= 0x1p15f) {
            const float less = pow2f(12 - log2i(w)), f = less / F[nt][x];
            F[nt][x] = less;
            if constexpr (kMid) ones[nt][x] *= f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[nt][d][x] *= f;
              o[nt][d][2 + x] *= f;
            }
          }
          top = fmaxf(top, F[nt][x]);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      cap = 0x1p15f / top;  // a weight is at most 1 (2^-22 more): under 2^16
    }

    // ---- weights, and the output's products
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const float2 v0 = unpack2<T>(va[kb][0]), v1 = unpack2<T>(va[kb][1]);
      const float mid0 = kMid ? fmaf(8.f, v0.x, v0.y) : v0.y, mid1 = kMid ? fmaf(8.f, v1.x, v1.y) : v1.y;
      uint32_t bf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
        float pe[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pe[e] = ex2(fmaf(s[nt][kb][e], c1[nt][e & 1], -base[nt][e & 1]));
          l[nt][e & 1] += pe[e];
          w[e] = pe[e] * (e < 2 ? v0.x : v1.x) * F[nt][e & 1];
        }
        if (!poison) {
#pragma unroll
          for (int e = 0; e < 4; ++e) low[nt][e & 1] = fmaf(pe[e], e < 2 ? mid0 : mid1, low[nt][e & 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s[nt][kb][e] == -INFINITY)
              w[e] = 0.f;
            else
              low[nt][e & 1] = fmaf(pe[e], e < 2 ? mid0 : mid1, low[nt][e & 1]);
        }
        bf[nt][0] = movmatrix_trans(pack2<__half>(w[0], w[1]));
        bf[nt][1] = movmatrix_trans(pack2<__half>(w[2], w[3]));
        if constexpr (kMid) {
          const uint32_t eights[4] = {kEight, kEight, kEight, kEight};
          mma_f16(ones[nt], eights, bf[nt][0], bf[nt][1]);
        }
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
        const uint32_t g0 = e0 >> 8, g1 = e1 >> 8, h0 = f0 >> 8, h1 = f1 >> 8;
        const uint32_t a0[4] = {e0 & kCode0, e0 & kCode1, e1 & kCode0, e1 & kCode1};
        const uint32_t a1[4] = {g0 & kCode0, g0 & kCode1, g1 & kCode0, g1 & kCode1};
        const uint32_t a2[4] = {f0 & kCode0, f0 & kCode1, f1 & kCode0, f1 & kCode1};
        const uint32_t a3[4] = {h0 & kCode0, h0 & kCode1, h1 & kCode0, h1 & kCode1};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_f16(o[nt][4 * w + 0], a0, bf[nt][0], bf[nt][1]);
          mma_f16(o[nt][4 * w + 1], a1, bf[nt][0], bf[nt][1]);
          mma_f16(o[nt][4 * w + 2], a2, bf[nt][0], bf[nt][1]);
          mma_f16(o[nt][4 * w + 3], a3, bf[nt][0], bf[nt][1]);
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (fetched < count) fetch_next(stage);
    if (++stage == STAGES) stage = 0, parity ^= 1;

    const bool run_ends = c.t + 1 == c.s.tiles;
    if (run_ends || i + 1 == count) {
      // ---- a run (or a piece of one) is done
      const bool whole = t0 == 0 && run_ends;
      const int slot = t0 > 0 ? 0 : 1;
      const bool last = i + 1 == count;  // the ring is free then, an earlier piece goes through the cache
      float* dst = last ? reinterpret_cast<float*>(ring) : first_all + warp * C::kPiece;
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
          const float inv = whole ? (ls == 0.f ? 0.f : 1.f / ls) : 1.f;
          const float back = 1.f / F[nt][x];  // and the codes' 2^-24 or 2^-20
          float y[D / 8];
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            y[2 * d] = fmaf((o[nt][d][x] - ones[nt][x]) * 0x1p24f, back, lw) * inv;
            y[2 * d + 1] = fmaf((o[nt][d][2 + x] - 16.f * ones[nt][x]) * 0x1p20f, back, lw) * inv;
          }
          if (whole) {
            if (rr < rows) {
              T* out = static_cast<T*>(a.out) +
                       ((c.s.q0 + static_cast<int64_t>(a.row_token(rr))) * a.hq + c.h * a.group + (rr - a.row_token(rr) * a.group)) * D + g * (D / 8);
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
              dst[RB * D + row] = mx[nt][x] == -INFINITY ? -INFINITY : mx[nt][x] * c1[nt][x];
              dst[RB * D + RB + row] = ls;
            }
          }
        }
      if (!whole && lane == 0) {
        int* pc = piece[2 * warp + slot];
        pc[1] = t0 == 0;
        pc[2] = run_ends;
        pc[3] = c.b, pc[4] = c.h, pc[5] = c.blk;
        pc[0] = last ? 2 : 1;
      }
    }
    advance(c, i + 1 < count);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may be set up
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
  // A warp takes four rows of a run: a lane D/32 consecutive dims of each, pieces in order.
  for (int item = warp; item < runs * (RB / 4); item += WARPS) {
    const int row0 = item % (RB / 4) * 4;
    unsigned rest = open;
    for (int k = item / (RB / 4); k; --k) rest &= rest - 1;
    const int head = __ffs(rest) - 1;
    const unsigned later = rest & (rest - 1);
    const unsigned group = all & ~((1u << head) - 1) & (later ? (later & -later) - 1 : ~0u);
    Kv4Joined<D> y;
    y.join(group, [&](int i) {
      return piece[i][0] == 2 ? reinterpret_cast<const float*>(kv4_smem + (i >> 1) * C::kRing)
                              : first_all + (i >> 1) * C::kPiece;
    }, RB, row0, lane);
    const int* hd = piece[head];
    const bool starts = hd[1], ends = piece[31 - __clz(group)][2];
    if (starts && ends) {
      y.template write<T>(a, kv4_seq<TILE, RB>(a, p.max_rows, hd[3]), hd[4], hd[5] * RB + row0, lane);
    } else {
      const int slot = starts ? 1 : 0;
      y.store(p.cta + (blockIdx.x * 2 + slot) * static_cast<int64_t>(C::kPiece), RB, row0, lane);
      if (lane == 0 && row0 == 0) {
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

// Joins the pieces of the runs cut by CTA borders: CTA i takes the run that starts in (and runs out of) CTA
// i of the first kernel. A warp takes four rows.
template <typename T, int D, int RB, int TILE>
__global__ void __launch_bounds__(32 * RB / 4) kv4_decode_join(const Kv4DecodeParams p, int parts) {
  constexpr int64_t kPiece = RB * (D + 2);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // until the first kernel is done and its stores are visible
  const int* d0 = p.desc + blockIdx.x * 8;
  if (!d0[2]) return;
  const int row0 = (threadIdx.x >> 5) * 4, lane = threadIdx.x & 31;
  // its pieces: the one it starts with, then the first ones of the CTAs behind, up to the one that ends it; 32 at a time
  Kv4Joined<D> y;
  bool more = true;
  for (int at = blockIdx.x; more; at += 32) {
    const int i = at + lane;
    const bool valid = i < parts && (i == static_cast<int>(blockIdx.x) || p.desc[i * 8]);
    const bool ends = valid && i != static_cast<int>(blockIdx.x) && p.desc[i * 8 + 1];
    const unsigned stop = __ballot_sync(0xffffffffu, ends || !valid);
    unsigned which = ~0u;
    if (stop) {
      const int k = __ffs(stop) - 1;
      which = (1u << k) - 1;
      if (__shfl_sync(0xffffffffu, static_cast<int>(ends), k)) which |= 1u << k;
      more = false;
    }
    Kv4Joined<D> z;
    z.join(which, [&](int j) {
      return p.cta + ((at + j) * 2 + (at + j == static_cast<int>(blockIdx.x) ? 1 : 0)) * kPiece;
    }, RB, row0, lane);
    if (at == static_cast<int>(blockIdx.x))
      y = z;
    else
      y.add(z);
  }
  y.template write<T>(p.a, kv4_seq<TILE, RB>(p.a, p.max_rows, d0[3]), d0[4], d0[5] * RB + row0, lane);
}

}  // namespace dscq
