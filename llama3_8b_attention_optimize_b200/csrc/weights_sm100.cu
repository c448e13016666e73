// weights_sm100.cu -- accumulated attention weight of every cached slot, on the sm_100a
// tensor core.
//
// For the chunk of attend_sm100.cu (same q_start, lens, slots and mask) and its lse,
//   acc_out[b, h, j] = (j < lens[b] - n ? acc[b, h, j] : 0)
//                      + sum over the group's heads and the chunk's tokens that see slot j
//                        of exp(q . K[b, h, j] * scale - lse),
// for j < lens[b]; entries at lens[b] and above are left alone.  Slots that the chunk
// itself wrote start from zero.
//
// With the lse known nothing has to be normalised, so the scores are computed transposed:
// S^T = K Q^T puts a slot on a TMEM lane and the (token, head) rows on columns, and a
// slot's sum stays in one thread's registers.  K is read once, no score is written, and
// the order of every sum is fixed: runs repeat bit for bit.
//
// Unit of work: (sequence, kv head, block of 256 slots), two 128-slot K tiles side by side
// that share the query tiles (128 rows: G heads of 128 / G tokens) it walks as steps.  Where
// a sequence brings at most 64 rows, a block has 512 slots, two steps of 256 with one query
// tile: a unit's beginning and end cost as much as loading 256 slots takes.  The
// steps of all units are cut into equal parts, one per CTA and SM (ragged.cuh).  Parts of
// one unit leave 256 sums each, which a second kernel adds in order.
//
// Pipeline: a producer warp (K tiles in a ring of 5, query tiles in one of 2), one
// MMA-issuing warp per K tile (two S^T buffers each: all 512 TMEM columns), a helper warp
// that stages each query tile's lse, and eight softmax warps per K tile (a thread: one
// slot, 64 of the 128 rows).
//
// Measured (Hq 32, Hkv 8, both launches, replayed from a graph): 64 single tokens over
// 128..8191 slots (572 MB) 100 us, 5.7 TB/s, bound by memory; 1024 tokens behind 7168 slots
// (64 GFLOP, 250 M exponentials) 98 us, bound by the exponentials: their unit is busy for two
// thirds of the cycles, waits and the scores' way from TMEM fill the rest.  The approximate
// exponential puts the chunk's sums at 3.9e-8 from 64 bits, where 32-bit torch is at 3.0e-8.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "gqa_internal.h"
#include "ragged.cuh"

namespace gqa {
namespace weights {

using ragged::Boxes;
using ragged::Desc;
using ragged::kMaxB;
using ragged::kMaxCtas;
using ragged::Part;
using ragged::Seq;
using ragged::Walk;

constexpr int kD = 128;
constexpr int kBlock = 256;                // slots of a unit: two K tiles
constexpr int kTileBytes = 128 * 128 * 2;  // K and Q tiles: 32 KB
constexpr int kHalf = kTileBytes / 2;
constexpr int kQStages = 2;
constexpr int kKStages = 5;  // K tiles in flight; tile i of the CTA (two a unit) lies in stage i % 5
// Tiles land on barriers of their own, i % 10: even tiles are one issuer's and odd ones the
// other's, so a stage changes hands at each use.  An issuer that waited on a stage's barrier
// would skip every other phase, and where tile i - 5 is late (loads may land out of order)
// the parity of the phase before it would pass for tile i's.
constexpr int kKBars = 2 * kKStages;
constexpr float kLog2e = 1.4426950408889634f;

constexpr int kSoftmaxWarps = 16;
constexpr int kWarpProducer = 16;
constexpr int kWarpMma = 17;  // and 18: one per K tile
constexpr int kWarpHelper = 19;
constexpr int kThreads = 640;

constexpr int kOffQ = 0;
constexpr int kOffK = kOffQ + kQStages * kTileBytes;
constexpr int kOffBar = kOffK + kKStages * kTileBytes;
constexpr int kNumBars = 34;
constexpr int kOffLse = kOffBar + kNumBars * 8;     // [2][128] -lse * log2(e)
constexpr int kOffSum = kOffLse + 2 * 128 * 4;      // [K tile][128] sums of the rows' second half
constexpr int kOffTok = kOffSum + 2 * 128 * 4;      // [128] token of a row in its tile
constexpr int kOffTmemPtr = kOffTok + 128;
constexpr int kOffStart = kOffTmemPtr + 16;
constexpr int kSmemBytes = kOffStart + 48;
static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");
static_assert(ragged::kPlanBytes <= kOffBar, "the plan's scratch lies in the tiles");
static_assert(sizeof(Walk) <= 48, "room for the start");

enum : int {
  B_QFULL = 0,    // [2]
  B_QEMPTY = 2,   // [2] one arrival per issuer
  B_KFULL = 4,    // [10]
  B_KEMPTY = 14,  // [5]
  B_SFULL = 19,   // [K tile][2]
  B_SFREE = 23,   // [K tile][2] one arrival per softmax warp
  B_LFULL = 27,   // [2] lse of a query tile staged
  B_LEMPTY = 29,  // [2] one arrival per softmax warp
  B_DRAIN = 31,   // [2]
};

enum : int {
  SITE_PRODUCER = 0x711,
  SITE_MMA = 0x712,
  SITE_SOFTMAX = 0x713,
  SITE_HELPER = 0x714,
  SITE_DRAIN = 0x716,
  SITE_SMEM_ALIGN = 0x717,
  SITE_Q_START = 0x630,   // q_start not ascending or outside [0, T]
  SITE_LENGTH = 0x631,    // lens[b] outside [0, capacity]
  SITE_BAD_PAGE = 0x632,  // block-table entry outside [0, num_pages)
};

static_assert(B_DRAIN + 2 <= kNumBars && kOffLse % 16 == 0, "barriers, and 16-byte reads behind them");

struct Params {
  ragged::Batch batch;
  const float *lse, *acc;
  float* acc_out;
  float* part;  // [2 * grid][kBlock]
  Desc* desc;   // [grid]
  int G, Hq, causal, tpt, box;
  int wide_n;  // most tokens of a sequence with blocks of 512 slots (64 rows)
  float scale_log2;
};

// Units: blocks of 256 slots.  Steps: the query tiles of which some row sees the block.  Wide
// units (of 512 slots) are one step; sequences without tokens have such too, to pass their sums on.
struct Line {
  static constexpr int extra = 2;  // what a unit's beginning and end cost, in query tiles
  int tpt, causal, wide_n;
  __device__ __forceinline__ Line(const Params& p) : tpt(p.tpt), causal(p.causal), wide_n(p.wide_n) {}
  __device__ __forceinline__ bool wide(const Seq& s) const { return s.n <= wide_n; }
  __device__ __forceinline__ int block(const Seq& s) const { return wide(s) ? 2 * kBlock : kBlock; }
  __device__ __forceinline__ bool has(const Seq& s) const { return s.L > 0; }
  __device__ __forceinline__ int units(const Seq& s) const { return (s.L + block(s) - 1) / block(s); }
  __device__ __forceinline__ bool ends(const Seq& s, int u) const { return (u + 1) * block(s) >= s.L; }
  __device__ __forceinline__ int tiles(const Seq& s) const { return (s.n + tpt - 1) / tpt; }
  // first query tile that sees slot kBlock * u: floor((kBlock u - (L - n)) / tpt), at least 0
  __device__ __forceinline__ int first(const Seq& s, int u) const {
    const int x = u * kBlock - (s.L - s.n);
    return !causal || x < tpt || wide(s) ? 0 : x / tpt;
  }
  __device__ __forceinline__ int count(const Seq& s, int u) const { return wide(s) ? 1 : tiles(s) - first(s, u); }
  __device__ __forceinline__ uint32_t before(const Seq& s, int k) const {
    if (wide(s)) return k * (1 + extra);
    uint32_t sum = static_cast<uint32_t>(k) * (tiles(s) + extra);
    const int base = s.L - s.n;
    const int u1 = base > 0 ? (base + kBlock - 1) / kBlock : 0;  // first unit past the old slots
    if (causal && k > u1) sum -= ragged::floor_sum(k - u1, tpt, kBlock, u1 * kBlock - base);
    return sum;
  }
};

// 16 columns of this lane's row of TMEM; tmem_wait_ld_dep16 before they are used.
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// p = 2^(s * sl2 + nl) of 16 rows that all see the slot.  The exponentials bound a chunk of
// many tokens (a share of them on the FMA pipe, by a quintic, took as long to 9 % longer).
__device__ __forceinline__ void add_all(const uint32_t (&s)[16], const float* nl, float2 sl2, float2& a0, float2& a1) {
#pragma unroll
  for (int c = 0; c < 16; c += 4) {
    const float4 l = *reinterpret_cast<const float4*>(nl + c);
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl2, make_float2(l.x, l.y));
    const float2 y =
        __ffma2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), sl2, make_float2(l.z, l.w));
    a0 = __fadd2_rn(a0, make_float2(ex2_approx(x.x), ex2_approx(x.y)));
    a1 = __fadd2_rn(a1, make_float2(ex2_approx(y.x), ex2_approx(y.y)));
  }
}

// The same where not all of the 16 rows see the slot: only the first nv, and of those the
// ones whose token is at least `from` within the tile.
__device__ __forceinline__ void add_masked(const uint32_t (&s)[16], const float* nl, const uint8_t* tok, int nv, int from,
                                           float sl2, float2& a0) {
#pragma unroll
  for (int c = 0; c < 16; c += 4) {
    const float4 l = *reinterpret_cast<const float4*>(nl + c);
    const uchar4 t = *reinterpret_cast<const uchar4*>(tok + c);
    const float e[4] = {ex2_approx(fmaf(__uint_as_float(s[c]), sl2, l.x)), ex2_approx(fmaf(__uint_as_float(s[c + 1]), sl2, l.y)),
                        ex2_approx(fmaf(__uint_as_float(s[c + 2]), sl2, l.z)),
                        ex2_approx(fmaf(__uint_as_float(s[c + 3]), sl2, l.w))};
    const int k[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < nv && k[i] >= from) a0.x += e[i];  // anything else may be NaN
  }
}

// The same for a few rows, eight at a time: units of single tokens are so short that the
// fetching of more code would bound them (163 -> 115 us for 64 tokens when this was written).
__device__ __forceinline__ void add_some(uint32_t taddr, const float* nl, const uint8_t* tok, int nv, int from, float sl2,
                                         float2& a0) {
#pragma unroll 1
  for (int c0 = 0; c0 < nv; c0 += 8) {
    uint32_t v[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr + c0));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])
                 :
                 : "memory");
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float e = ex2_approx(fmaf(__uint_as_float(v[c]), sl2, nl[c0 + c]));
      if (c0 + c < nv && static_cast<int>(tok[c0 + c]) >= from) a0.x += e;  // anything else may be NaN
    }
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) record_error(SITE_SMEM_ALIGN);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };

  if (warp == kWarpHelper) {  // a barrier a lane
    for (int i = lane; i < B_DRAIN + 2; i += 32) {
      int count = 1;
      if (i >= B_QEMPTY && i < B_KFULL) count = 2;
      if (i >= B_SFREE && i < B_LFULL) count = 8;
      if (i >= B_LFULL && i < B_LEMPTY) count = 32;
      if (i >= B_LEMPTY && i < B_DRAIN) count = kSoftmaxWarps;
      mbar_init(bar(i), count);
    }
    fence_mbar_init();
  }
  if (threadIdx.x < 128) smem[kOffTok + threadIdx.x] = static_cast<uint8_t>(threadIdx.x / p.G);
  if (warp == kWarpMma) {
    tmem_alloc(sbase + kOffTmemPtr, 512);
    tmem_relinquish();
  }
  if (warp == kWarpProducer && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
  }
  const Line line(p);
  const Line lines[1] = {line};
  const int cost[1] = {1};
  ragged::plan<kThreads>(p.batch, lines, cost, reinterpret_cast<uint32_t*>(smem),
                         reinterpret_cast<Walk*>(smem + kOffStart), p.desc, SITE_Q_START, SITE_LENGTH);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kOffTmemPtr);
  Walk walk = *reinterpret_cast<const Walk*>(smem + kOffStart);
  // The plan's scratch (generic writes) lies where TMA will write.
  fence_proxy_async_smem();
  __syncthreads();
  Part s;

  if (warp == kWarpProducer) {
    // ------------------------------------------------------------ TMA producer (whole warp)
    bool ok = true;
    uint32_t g = 0, m = 0;  // query tiles and K tiles loaded
    const Boxes boxes(p.box, lane);
    auto load_q = [&](int head, int tok) {
      const int st = static_cast<int>(g % kQStages);
      if (g >= kQStages)
        ok = __all_sync(0xffffffffu, mbar_wait(bar(B_QEMPTY + st), (g / kQStages - 1) & 1u, SITE_PRODUCER));
      if (!ok) return;
      if (lane == 0) {
        mbar_expect_tx(bar(B_QFULL + st), 2 * 128 * p.G * p.tpt);
        for (int e = 0; e < 2; ++e)
          tma_load_4d(sbase + kOffQ + st * kTileBytes + e * kHalf, &tmQ, bar(B_QFULL + st), 64 * e, head, tok, 0);
      }
      ++g;
    };
    // the next unit with tokens and its pages, looked up a unit ahead
    int page[4] = {-1, -1, -1, -1}, tiles = 0;
    auto advance = [&]() -> bool {
      do {
        if (!ragged::next_part(p.batch, line, walk, s)) return false;
      } while (s.s.n == 0);
      const int32_t* table = p.batch.table + static_cast<size_t>(s.b) * p.batch.max_pages;
      tiles = line.block(s.s) / 128;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < tiles) page[i] = boxes.page(p.batch, table, s.u * 128 * tiles + 128 * i, s.s.L);
      return true;
    };
    bool more = advance();
    while (ok && more) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!ok || i >= tiles) continue;
        const int st = static_cast<int>(m % kKStages);
        const int row = boxes.row(p.batch, page[i], s.h, s.u * 128 * tiles + 128 * i, s.s.L, SITE_BAD_PAGE);
        if (m >= kKStages)
          ok = __all_sync(0xffffffffu, mbar_wait(bar(B_KEMPTY + st), (m / kKStages - 1) & 1u, SITE_PRODUCER));
        if (!ok) continue;
        const uint32_t mine = __ballot_sync(0xffffffffu, row >= 0), full = bar(B_KFULL + static_cast<int>(m % kKBars));
        if (lane == 0) mbar_expect_tx(full, __popc(mine) * p.box * 128);
        __syncwarp();
        if (row >= 0)
          tma_load_3d(sbase + kOffK + st * kTileBytes + boxes.offset, &tmK, full, boxes.half * 64, row, 0);
        ++m;
        if (i == 0 && tiles == 4) load_q(s.h * p.G, s.s.a);  // its one query tile, ahead of most of K
      }
      if (!ok) break;
      if (tiles == 4) {
        more = advance();  // while the loads are under way
        continue;
      }
      const int steps = s.k1 - s.k0, head = s.h * p.G;
      int tok = s.s.a + (line.first(s.s, s.u) + s.k0) * p.tpt;
      for (int k = 0; ok && k < steps; ++k, tok += p.tpt) {
        load_q(head, tok);
        if (k == 0) more = advance();
      }
    }
    // Drain: every load this warp issued must land before the CTA may exit.
    for (uint32_t i = g > kQStages ? g - kQStages : 0u; i < g; ++i)
      mbar_wait_drain(bar(B_QFULL + static_cast<int>(i % kQStages)), (i / kQStages) & 1u, SITE_DRAIN);
    for (uint32_t i = m > kKStages ? m - kKStages : 0u; i < m; ++i)
      mbar_wait_drain(bar(B_KFULL + static_cast<int>(i % kKBars)), (i / kKBars) & 1u, SITE_DRAIN);
    __syncwarp();
  } else if (warp == kWarpMma || warp == kWarpMma + 1) {
    // ------------------------------------------------------------ MMA issuers, one per K tile
    const int kt = warp - kWarpMma;
    if (lane == 0) {
      constexpr uint32_t kHi = sdesc_hi_sw128(1024);
      const uint32_t k_lo = sdesc_lo(sbase + kOffK, 16);
      const uint32_t q_lo = sdesc_lo(sbase + kOffQ, 16);
      constexpr uint32_t kTile16 = kTileBytes / 16;
      bool ok = true;
      uint32_t g = 0, qn = 0, m = kt;  // steps, query tiles, and the K tile
      while (ok && ragged::next_part(p.batch, line, walk, s)) {
        if (s.s.n == 0) continue;
        const bool wide = line.wide(s.s);
        const int first = line.first(s.s, s.u) + s.k0, steps = wide ? 2 : s.k1 - s.k0;
        for (int k = 0; ok && k < steps; ++k, ++g) {
          const int ks = static_cast<int>(m % kKStages), st = static_cast<int>(qn % kQStages), bb = static_cast<int>(g & 1);
          const bool k_first = wide || k == 0, k_last = wide || k + 1 == steps;  // of the K tile, of the query tile
          const bool q_first = !wide || k == 0, q_last = !wide || k + 1 == steps;
          if (k_first) ok = mbar_wait_spin(bar(B_KFULL + static_cast<int>(m % kKBars)), (m / kKBars) & 1u, SITE_MMA);
          if (ok && q_first) ok = mbar_wait_spin(bar(B_QFULL + st), (qn / kQStages) & 1u, SITE_MMA);
          if (ok && g >= 2) ok = mbar_wait_spin(bar(B_SFREE + 2 * kt + bb), (g / 2 - 1) & 1u, SITE_MMA);
          if (!ok) break;
          // only as many columns as the tile has rows, in the MMA's steps of 16
          const int nv = (wide ? s.s.n : min(p.tpt, s.s.n - (first + k) * p.tpt)) * p.G;
          const uint32_t id = idesc_bf16_f32(128, (nv + 15) / 16 * 16, false);
          const uint32_t a0 = k_lo + ks * kTile16, b0 = q_lo + st * kTile16;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = ((kk >> 2) * kHalf + (kk & 3) * 32) / 16;
            umma_ss_lohi(tmem + 256 * kt + 128 * bb, a0 + off, b0 + off, kHi, id, kk > 0 ? 1u : 0u);
          }
          umma_commit(bar(B_SFULL + 2 * kt + bb));
          if (q_last) {
            umma_commit(bar(B_QEMPTY + st));
            ++qn;
          }
          if (k_last) {
            umma_commit(bar(B_KEMPTY + ks));
            m += 2;
          }
        }
      }
      umma_commit(bar(B_DRAIN + kt));
      mbar_wait_drain(bar(B_DRAIN + kt), 0, SITE_DRAIN);
    }
    __syncwarp();
  } else if (warp == kWarpHelper) {
    // ------------------------------------------------------------ lse of each query tile
    bool ok = true;
    uint32_t g = 0;
    int tok[4], head[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      tok[i] = (lane + 32 * i) / p.G;
      head[i] = (lane + 32 * i) % p.G;
    }
    while (ok && ragged::next_part(p.batch, line, walk, s)) {
      if (s.s.n == 0) continue;
      const bool wide = line.wide(s.s);
      const int first = line.first(s.s, s.u) + s.k0, steps = wide ? 2 : s.k1 - s.k0;
      for (int k = 0; ok && k < steps; ++k, ++g) {
        const int t0 = wide ? 0 : (first + k) * p.tpt, bb = static_cast<int>(g & 1);
        float nl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          nl[i] = -INFINITY;  // no row, or one that saw nothing
          if (tok[i] < p.tpt && t0 + tok[i] < s.s.n) {
            const float x = __ldg(p.lse + static_cast<size_t>(s.s.a + t0 + tok[i]) * p.Hq + s.h * p.G + head[i]);
            if (x != -INFINITY) nl[i] = -x * kLog2e;
          }
        }
        if (g >= 2) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_LEMPTY + bb), (g / 2 - 1) & 1u, SITE_HELPER));
        if (!ok) break;
        float* dst = reinterpret_cast<float*>(smem + kOffLse) + 128 * bb;
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[lane + 32 * i] = nl[i];
        mbar_arrive(bar(B_LFULL + bb));
      }
    }
  } else {
    // ------------------------------------------------------------ softmax warps
    const int kt = warp >> 3;          // K tile
    const int ch = (warp >> 2) & 1;    // rows [64 ch, 64 ch + 64) of each query tile
    const int r = (warp & 3) * 32 + lane;  // slot in the K tile == TMEM lane
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 256 * kt;
    const float* lse = reinterpret_cast<const float*>(smem + kOffLse);
    const uint8_t* tok = smem + kOffTok;
    float* xsum = reinterpret_cast<float*>(smem + kOffSum) + 128 * kt;
    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    uint32_t g = 0;
    // A slot's old sum, read a unit ahead: its latency is as long as a unit of a
    // single-token batch.
    auto slot_of = [&](const Part& x) -> int {
      return line.wide(x.s) ? (2 * x.u + ch) * kBlock + 128 * kt + r : x.u * kBlock + 128 * kt + r;
    };
    auto old_of = [&](const Part& x) -> float {
      const int slot = slot_of(x);
      if ((ch != 0 && !line.wide(x.s)) || slot >= x.s.L - x.s.n || !x.whole()) return 0.0f;
      return __ldg(p.acc + (static_cast<size_t>(x.b) * p.batch.Hkv + x.h) * p.batch.capacity + slot);
    };
    Part ahead;
    bool more = ragged::next_part(p.batch, line, walk, s);
    float old = more ? old_of(s) : 0.0f;
    // Every warp meets the named barriers of every unit, even after a failed wait.
    while (more) {
      more = ragged::next_part(p.batch, line, walk, ahead);
      const float old_ahead = more ? old_of(ahead) : 0.0f;
      const int slot = slot_of(s);
      const int warp_last = min(s.s.L, slot - lane + 32) - 1;
      const bool wide = line.wide(s.s);
      const int half = wide ? 0 : 64 * ch;  // first row of this warp's

      float sum = 0.0f;
      if (s.s.n > 0) {
        const int first = line.first(s.s, s.u) + s.k0, steps = wide ? 2 : s.k1 - s.k0;
        for (int k = 0; k < steps; ++k, ++g) {
          const int bb = static_cast<int>(g & 1);
          const int t0 = wide ? 0 : (first + k) * p.tpt;
          // rows of this warp: half of the tile's, or in a wide unit's step all or none
          const int nv = wide && k != ch ? 0 : min(64, min(p.tpt, s.s.n - t0) * p.G - half);
          // the tile's first token sees slots up to see0, each next token one more
          const int see0 = p.causal ? s.s.L - s.s.n + t0 : s.s.L - 1;
          if (ok) {  // both asked before either answer is needed
            const uint32_t parity = (g / 2) & 1u;
            const bool l_now = mbar_try_wait(bar(B_LFULL + bb), parity);
            const bool s_now = mbar_try_wait(bar(B_SFULL + 2 * kt + bb), parity);
            bool both = l_now && s_now;
            if (!both)
              both = mbar_wait(bar(B_LFULL + bb), parity, SITE_SOFTMAX) &&
                     mbar_wait(bar(B_SFULL + 2 * kt + bb), parity, SITE_SOFTMAX);
            ok = __all_sync(0xffffffffu, both);
          }
          if (!ok) continue;
          const bool all = see0 >= warp_last;
          const int from = p.causal ? slot - see0 : 0;  // a row of a token below this does not see the slot
          float2 a0 = make_float2(0.f, 0.f), a1 = make_float2(0.f, 0.f);
          const uint32_t tv = tS + 128 * bb + half;
          const float* nl = lse + 128 * bb + half;
          tc_fence_after();
          if (nv > 8) {
            // 16 rows at a time, the next 16 on their way while these are added up
            uint32_t v[2][16];
            ld16(tv, v[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int left = nv - 16 * c;
              tmem_wait_ld_dep16(v[c & 1]);
              if (c < 3) {
                ld16(tv + 16 * (c + 1), v[(c + 1) & 1]);
              } else {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SFREE + 2 * kt + bb));
              }
              if (all && left >= 16)
                add_all(v[c & 1], nl + 16 * c, sl2, a0, a1);
              else if (left > 0)
                add_masked(v[c & 1], nl + 16 * c, tok + half + 16 * c, left, from, p.scale_log2, a0);
            }
          } else {
            add_some(tv, nl, tok + half, nv, from, p.scale_log2, a0);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_SFREE + 2 * kt + bb));
          }
          sum += (a0.x + a0.y) + (a1.x + a1.y);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_LEMPTY + bb));
        }
      }
      if (!wide) {
        named_bar_sync(3 + kt, 256);  // the previous unit's exchange has been read
        if (ch == 1) xsum[r] = sum;
        named_bar_sync(1 + kt, 256);
        if (ch == 0) sum += xsum[r];
      }
      if (ok && (wide || ch == 0) && slot < s.s.L) {
        if (s.whole())
          p.acc_out[(static_cast<size_t>(s.b) * p.batch.Hkv + s.h) * p.batch.capacity + slot] = old + sum;
        else
          p.part[static_cast<size_t>(2 * blockIdx.x + (s.k0 == 0 ? 1 : 0)) * kBlock + 128 * kt + r] = sum;
      }
      s = ahead;
      old = old_ahead;
    }
  }

  // ---- teardown: everyone done with TMEM and shared memory
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Add a split unit's parts in order: block c takes the unit that CTA c began, if any.
__global__ void __launch_bounds__(kBlock) merge_kernel(const Params p) {
  cudaGridDependencySynchronize();
  const Desc d = p.desc[blockIdx.x];
  if (!d.valid) return;
  const Seq& s = d.s;
  const int slot = d.u * kBlock + threadIdx.x;
  if (slot >= s.L) return;
  float sum = 0.0f;
  for (int c = blockIdx.x; c <= d.last; ++c)
    sum += p.part[static_cast<size_t>(2 * c + (c == static_cast<int>(blockIdx.x) ? 1 : 0)) * kBlock + threadIdx.x];
  const size_t at = (static_cast<size_t>(d.b) * p.batch.Hkv + d.h) * p.batch.capacity + slot;
  p.acc_out[at] = (slot < s.L - s.n ? p.acc[at] : 0.0f) + sum;
}

constexpr size_t kPartBytes = static_cast<size_t>(2 * kMaxCtas) * kBlock * sizeof(float);

}  // namespace weights

GQA_ERROR_FLAG_ACCESSOR(error_flag_weights)

}  // namespace gqa

using namespace gqa;

extern "C" size_t gqa_attn_weight_sums_workspace_size(void) {
  return weights::kPartBytes + weights::kMaxCtas * sizeof(ragged::Desc);
}

extern "C" int gqa_attn_weight_sums_f32(const void* q, long long q_token_stride, long long q_head_stride,
                                        const void* kpages, const int32_t* block_table, int max_pages_per_seq,
                                        int page_size, int num_pages, const int32_t* q_start, const int32_t* lens,
                                        const float* lse, const float* acc, float* acc_out, void* workspace,
                                        size_t workspace_bytes, int B, int T, int Hq, int Hkv, int head_dim, float scale,
                                        int flags, gqa_stream_t stream) {
  using namespace weights;
  if (B <= 0 || T < 0 || Hq <= 0 || Hkv <= 0 || max_pages_per_seq <= 0 || page_size <= 0 || num_pages <= 0)
    return GQA_ERR_INVALID_ARGUMENT;
  if (head_dim != kD || Hq % Hkv || page_size % 16) return GQA_ERR_UNSUPPORTED;
  if (!(scale > 0.0f) || !(scale < 1e30f) || (flags & ~GQA_FLAG_CAUSAL)) return GQA_ERR_INVALID_ARGUMENT;
  if (q_token_stride < 0 || q_head_stride < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (!kpages || !block_table || !q_start || !lens || !acc || !acc_out || (T > 0 && (!q || !lse)))
    return GQA_ERR_INVALID_ARGUMENT;
  auto odd = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 4 != 0; };
  if (!aligned16(q) || !aligned16(kpages) || odd(block_table) || odd(q_start) || odd(lens) || odd(lse) || odd(acc) ||
      odd(acc_out) || !aligned16(workspace))
    return GQA_ERR_MISALIGNED;
  if ((T > 1 && q_token_stride % 8) || (Hq > 1 && q_head_stride % 8)) return GQA_ERR_MISALIGNED;
  const int G = Hq / Hkv;
  const long long capacity = static_cast<long long>(max_pages_per_seq) * page_size;
  const long long pool_rows = static_cast<long long>(num_pages) * Hkv * page_size;
  if (G > 128 || B > kMaxB || capacity > (1LL << 30) || pool_rows > 0x7FFFFFFFLL) return GQA_ERR_UNSUPPORTED;
  // query tiles over all blocks of slots: counted in 32 bits
  const long long steps = (static_cast<long long>(T) + 128 / G - 1) / (128 / G) + 3LL * B;
  if (static_cast<double>(steps) * Hkv * (capacity / kBlock + 1) >= 2147483648.0) return GQA_ERR_UNSUPPORTED;
  // a TMA dimension needs a stride: heads or tokens that share one row are the caller's to expand
  if ((T > 1 && q_token_stride == 0) || (Hq > 1 && q_head_stride == 0)) return GQA_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < gqa_attn_weight_sums_workspace_size()) return GQA_ERR_WORKSPACE;

  Params p;
  p.batch = {block_table, q_start, lens, B, T, Hkv, static_cast<int>(capacity), max_pages_per_seq, page_size, num_pages,
             ragged::whole_log2(page_size)};
  p.lse = lse;
  p.acc = acc;
  p.acc_out = acc_out;
  p.part = static_cast<float*>(workspace);
  p.desc = reinterpret_cast<Desc*>(static_cast<char*>(workspace) + kPartBytes);
  p.G = G;
  p.Hq = Hq;
  p.causal = (flags & GQA_FLAG_CAUSAL) != 0;
  p.tpt = 128 / G;
  p.wide_n = 64 / G;
  p.box = std::min(128, page_size & -page_size);
  p.scale_log2 = scale * kLog2e;

  CUtensorMap tmQ, tmK;
  int rc;
  // without tokens nothing is loaded through the query map, but it needs an address
  const long long ht = Hq > 1 ? q_head_stride : kD, tt = T > 1 ? q_token_stride : static_cast<long long>(Hq) * kD;
  const long long qd[4] = {kD, Hq, std::max(T, 1), 1}, qs[3] = {ht * 2, tt * 2, tt * 2};
  const int qb[4] = {64, G, p.tpt, 1};
  if ((rc = make_tmap_4d(&tmQ, T > 0 ? q : kpages, 2, qd, qs, qb)) != GQA_OK) return rc;
  if ((rc = make_tmap_3d_bf16(&tmK, kpages, kD, pool_rows, 1, 64, p.box, 1)) != GQA_OK) return rc;
  static std::atomic<uint64_t> attr_done{0};
  if ((rc = ensure_smem_attr(weights_kernel, kSmemBytes, attr_done)) != GQA_OK) return rc;
  int dev = 0, sms = kMaxCtas;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int grid = std::min(sms, kMaxCtas);
  weights_kernel<<<grid, kThreads, kSmemBytes, stream>>>(tmQ, tmK, p);
  if (cudaGetLastError() != cudaSuccess) return GQA_ERR_CUDA;
  // The merge starts while the first kernel drains and waits for it on the device.
  return launch_after(merge_kernel, dim3(grid), kBlock, stream, p);
}
