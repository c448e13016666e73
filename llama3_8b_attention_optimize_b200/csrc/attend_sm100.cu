// attend_sm100.cu -- attention of a ragged chunk of new tokens over a paged K/V cache, on
// the sm_100a tensor core.
//
// Sequence b brings tokens q_start[b] .. q_start[b + 1] - 1 (n of them); lens[b] counts
// its cached slots with those tokens included, so its token i sits in slot lens[b] - n + i.
//   o[t, h, :] = sum_j softmax_j(q[t, h] . K[b, h / G, j] * scale) V[b, h / G, j, :]
// over the slots j it sees (j <= its own slot when causal, else j < lens[b]), and
// lse[t, h] = ln sum_j exp(q[t, h] . K[b, h / G, j] * scale).  A row that sees no slot gives
// zeros and -inf.
//
// Unit of work: (sequence, kv head, block of query tokens); its rows are (token, head of the
// group) pairs, packed G to a token into NT tiles of 128 rows, so K and V are read once
// for all heads of the group and for NT * 128 / G tokens.  A unit walks its K/V tiles of
// 128 slots with an online softmax.
//
// Split: all units' K/V tiles form one line, cut into equal parts, one per CTA and SM
// (ragged.cuh).  A part may begin and end inside a unit; such segments leave (O, m, l) in
// the workspace and a second kernel merges them.  So one long sequence of a single token
// keeps every SM busy.
//
// Pipeline (per CTA): a producer warp loads Q by TMA and streams K and V tiles through a ring, one
// box per page (or per part of a page inside a tile); one warp per Q tile issues S = Q K^T
// and O += P V (tcgen05, accumulators in TMEM); eight softmax warps per Q tile (two
// halves of 64 slots) turn S into P in shared memory, rescaling O only when the running
// maximum grows by more than 2^16; a helper warp clears V rows past the last slot that the unit
// sees (P is zero there, but a cache may hold anything, and 0 * NaN would spread).
//
// Two tilings: NT = 2 (256 rows, ring of 3 tiles) where sequences bring more rows than a
// tile holds; NT = 1 (128 rows, ring of 5) for single tokens, which are bound by memory.
#include <cuda.h>

#include <algorithm>

#include "attn_common.cuh"
#include "common.cuh"
#include "gqa_internal.h"
#include "ragged.cuh"

namespace gqa {
namespace attend {

using attn::exp2_poly2;
using attn::fmax3;
using attn::load_idx_k;
using attn::load_idx_v;
using attn::sw128_chunk;
using ragged::Boxes;
using ragged::Desc;
using ragged::kMaxB;
using ragged::kMaxCtas;
using ragged::Part;
using ragged::Seq;
using ragged::seq_of;
using ragged::Walk;

constexpr int kD = 128;
constexpr int kBN = 128;                   // slots per K/V tile
constexpr int kTileBytes = 128 * 128 * 2;  // Q, P, K and V tiles: 32 KB
constexpr int kHalf = kTileBytes / 2;      // one 64-column swizzle block of 128 rows
constexpr float kRescaleLog2 = 16.0f;
constexpr float kLn2 = 0.6931471805599453f;

template <int NT>
struct Cfg {
  static constexpr int kStages = NT == 2 ? 3 : 5;
  static constexpr int kSoftmaxWarps = 8 * NT;
  static constexpr int kWarpProducer = kSoftmaxWarps;
  static constexpr int kWarpMma = kSoftmaxWarps + 1;  // one issuer per Q tile
  static constexpr int kWarpHelper = kSoftmaxWarps + 3;
  static constexpr int kThreads = (kSoftmaxWarps + 4) * 32;
  // Register split of the 640-thread tiling, as in the prefill: the sum must stay within
  // the launch allocation (the host checks the compiled count before the first launch).
  static constexpr bool kSplitRegs = NT == 2;
  static constexpr int kRegsLaunch = 96, kRegsHelper = 64, kRegsSoftmax = 104;
  static_assert(4 * 128 * kRegsSoftmax + 128 * kRegsHelper <= 640 * kRegsLaunch, "register split over budget");
  static constexpr int kOffQ = 0;
  static constexpr int kOffP = kOffQ + NT * kTileBytes;
  static constexpr int kOffKV = kOffP + NT * kTileBytes;
  static constexpr int kOffBar = kOffKV + kStages * kTileBytes;
  static constexpr int kNumBars = 40;
  static constexpr int kOffX = kOffBar + kNumBars * 8;  // row exchange [tile][half][128]
  static constexpr int kOffTmemPtr = kOffX + NT * 2 * 128 * 4;
  static constexpr int kOffStart = kOffTmemPtr + 16;  // this CTA's part: first unit, tile, count
  static constexpr int kSmemBytes = kOffStart + 32;
  static_assert(sizeof(Walk) <= 32, "room for the start");
  static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");
  static_assert(kMaxB * 8 + 64 * 8 <= kStages * kTileBytes, "the plan's scratch lies in the ring");
};

enum : int {
  B_QFULL = 0,     // [2] Q tile t of the current unit landed
  B_QEMPTY = 2,    // [1] last QK^T of the segment complete (one arrival per issuer)
  B_KVFULL = 3,    // [5] K/V stage landed
  B_KVEMPTY = 8,   // [5] MMAs reading the stage completed (issuers + helper)
  B_SFULL = 13,    // [2] S_t = Q_t K^T complete
  B_SFREE = 15,    // [2] S_t copied to registers
  B_PREADY = 17,   // [2] P_t in shared memory, O_t rescaled
  B_PVDONE = 19,   // [2] O_t += P_t V complete
  B_VZERO = 21,    // [4] rows past the last seen slot cleared (event k in slot k % 4)
  B_DRAIN = 25,    // [2] every MMA of issuer t complete
};

enum : int {
  SITE_PRODUCER = 0x701,
  SITE_MMA = 0x702,
  SITE_SOFTMAX = 0x703,
  SITE_HELPER = 0x704,
  SITE_EPILOGUE = 0x705,
  SITE_DRAIN = 0x706,
  SITE_SMEM_ALIGN = 0x707,
  SITE_Q_START = 0x620,   // q_start not ascending or outside [0, T]
  SITE_LENGTH = 0x621,    // lens[b] outside [0, capacity]
  SITE_BAD_PAGE = 0x622,  // block-table entry outside [0, num_pages)
};

struct Params {
  ragged::Batch batch;
  uint16_t* o;
  float* lse;
  float4* part_o;  // [2 * grid][32][part_rows]
  float* part_ml;  // [2 * grid][3][part_rows]
  Desc* desc;      // [grid]
  long long o_t, o_h;
  int G, Hq, causal;
  int tpt, tu;     // query tokens per tile, per unit
  int box;         // rows of one K/V box: the largest power of two dividing page_size, <= 128
  int part_rows;
  float scale_log2;
};

// Units: blocks of tu query tokens.  Steps: K/V tiles over the slots [0, limit) that some
// row of the unit sees; one at least, so that rows without any slot are written too.
struct Line {
  int tu, causal;
  __device__ __forceinline__ Line(const Params& p) : tu(p.tu), causal(p.causal) {}
  __device__ __forceinline__ int units(const Seq& s) const { return (s.n + tu - 1) / tu; }
  __device__ __forceinline__ int limit(const Seq& s, int u) const {
    return causal ? max(0, s.L - s.n + min(s.n, (u + 1) * tu)) : s.L;
  }
  __device__ __forceinline__ int count(const Seq& s, int u) const { return max(1, (limit(s, u) + kBN - 1) / kBN); }
  __device__ __forceinline__ long long before(const Seq& s, int k) const {
    const int n = units(s);
    if (!causal) return static_cast<long long>(k) * count(s, 0);
    const int m = min(k, n - 1);  // the last unit may be shorter
    const long long base = s.L - s.n;
    // units whose limit is at most one tile
    const int one = base >= kBN ? 0 : static_cast<int>(min(static_cast<long long>(m), (kBN - base) / tu));
    long long sum = one;
    if (m > one)
      sum += ragged::floor_sum(m - one, kBN, tu, base + static_cast<long long>(one + 1) * tu + kBN - 1);
    if (k == n) sum += count(s, n - 1);
    return sum;
  }
};

struct Seg : Part {
  int tok0, n_tok, base, limit;
  // the unit's last slots lie in this segment and do not fill their tile
  __device__ __forceinline__ bool tail() const { return k1 == count && limit < count * kBN; }
};

__device__ __forceinline__ bool next_seg(const Params& p, Walk& w, Seg& x) {
  const Line line(p);
  if (!ragged::next_part(p.batch, line, w, x)) return false;
  x.tok0 = x.u * p.tu;
  x.n_tok = min(p.tu, x.s.n - x.tok0);
  x.base = x.s.L - x.s.n;
  x.limit = line.limit(x.s, x.u);
  return true;
}

// ------------------------------------------------------------------ exponentials
// One 32-column chunk of S -> p = 2^(s*scale_log2 - m) as bf16, stored straight into the
// K-major SW128 P tile (row r, 16-byte chunks c0..c0+3).  acc sums the rounded p that P V
// multiplies, so that O / l is a mean whose weights add up to one; accf sums them
// unrounded, for the log-sum-exp.
template <bool kEmulate, bool kLse>
__device__ __forceinline__ void exp_chunk_store(const uint32_t (&s)[32], uint8_t* ptile, int r, int c0, float2 sc2,
                                                float2 nm2, float2& acc, float2& accf) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * c + e;
      const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sc2, nm2);
      float2 y;
      if (kEmulate && e == 3) {
        y = exp2_poly2(x);
      } else {
        y.x = ex2_approx(x.x);
        y.y = ex2_approx(x.y);
      }
      if (kLse) accf = __fadd2_rn(accf, y);
      w[e] = pack_bf16x2(y.x, y.y);
      add_bf16x2_to_f32(acc, w[e]);
    }
    *reinterpret_cast<uint4*>(ptile + sw128_chunk(r, c0 + c)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int NT, bool kLse>
__global__ void __launch_bounds__(Cfg<NT>::kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const Params p) {
  using C = Cfg<NT>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // uniform across the CTA: leave before any barrier
    if (threadIdx.x == 0) record_error(SITE_SMEM_ALIGN);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  auto bar = [&](int i) -> uint32_t { return sbase + C::kOffBar + 8 * i; };

  if (threadIdx.x == 0) {
    for (int t = 0; t < NT; ++t) {
      mbar_init(bar(B_QFULL + t), 1);
      mbar_init(bar(B_SFULL + t), 1);
      mbar_init(bar(B_PVDONE + t), 1);
      mbar_init(bar(B_SFREE + t), 256);
      mbar_init(bar(B_PREADY + t), 256);
      mbar_init(bar(B_DRAIN + t), 1);
    }
    mbar_init(bar(B_QEMPTY), NT);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(B_KVFULL + s), 1);
      mbar_init(bar(B_KVEMPTY + s), NT + 1);
    }
    for (int k = 0; k < 4; ++k) mbar_init(bar(B_VZERO + k), 32);
    fence_mbar_init();
  }
  if (warp == C::kWarpMma) {
    tmem_alloc(sbase + C::kOffTmemPtr, 256 * NT);
    tmem_relinquish();
  }
  if (warp == C::kWarpProducer && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }

  ragged::plan<C::kThreads>(p.batch, Line(p), reinterpret_cast<long long*>(smem + C::kOffKV),
                            reinterpret_cast<Walk*>(smem + C::kOffStart), p.desc, SITE_Q_START, SITE_LENGTH);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::kOffTmemPtr);
  Walk walk = *reinterpret_cast<const Walk*>(smem + C::kOffStart);
  auto colS = [](int t) -> uint32_t { return static_cast<uint32_t>(t * 128); };
  auto colO = [](int t) -> uint32_t { return static_cast<uint32_t>(NT * 128 + t * 128); };
  // The plan's scratch (generic writes) lies where TMA will write.
  fence_proxy_async_smem();
  __syncthreads();

  if (warp == C::kWarpProducer) {
    // ------------------------------------------------------------ TMA producer (whole warp)
    if constexpr (C::kSplitRegs) regs_dec<C::kRegsHelper>();
    bool ok = true;
    uint32_t L = 0;               // K/V loads issued by this CTA (ring position)
    uint32_t n_q[2] = {0, 0};     // Q tiles loaded
    uint32_t n_seg = 0;
    const Boxes boxes(p.box, lane);
    Seg s;
    while (ok && next_seg(p, walk, s)) {
      // Q tiles are reused once the previous segment's last QK^T is done
      if (n_seg > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_QEMPTY), (n_seg - 1) & 1, SITE_PRODUCER));
      if (!ok) break;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t * p.tpt < s.n_tok) {
          ++n_q[t];
          if (lane == 0) {
            const uint32_t dst = sbase + C::kOffQ + t * kTileBytes;
            mbar_expect_tx(bar(B_QFULL + t), 2 * 128 * p.G * p.tpt);
            for (int e = 0; e < 2; ++e)
              tma_load_4d(dst + e * kHalf, &tmQ, bar(B_QFULL + t), 64 * e, s.h * p.G, s.s.a + s.tok0 + t * p.tpt, 0);
          }
        }
      }
      ++n_seg;
      const int n = s.k1 - s.k0;
      const int32_t* table = p.batch.table + static_cast<size_t>(s.b) * p.batch.max_pages;
      int page_next = boxes.page(p.batch, table, s.k0 * kBN, s.limit);  // read one K tile ahead
      int row_k = -1, row_v = -1;  // rows of the latest K tile and of the tile whose V comes next
      for (int li = 0; ok && li < 2 * n; ++li) {
        const int st = static_cast<int>(L % kStages);
        const uint32_t r = L / kStages;
        // li -> (tile, K or V): K one tile ahead of V
        const bool is_v = (li == 2 * n - 1) || (li >= 2 && (li & 1) == 0);
        int row;
        if (is_v) {
          row = li == 2 * n - 1 ? row_k : row_v;
        } else {
          const int slot0 = (s.k0 + (li == 0 ? 0 : (li + 1) >> 1)) * kBN;
          row_v = row_k;
          row_k = boxes.row(p.batch, page_next, s.h, slot0, s.limit, SITE_BAD_PAGE);
          page_next = boxes.page(p.batch, table, slot0 + kBN, s.limit);
          row = row_k;
        }
        if (r > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_KVEMPTY + st), (r - 1) & 1u, SITE_PRODUCER));
        if (!ok) break;
        const uint32_t mine = __ballot_sync(0xffffffffu, row >= 0);
        if (lane == 0) mbar_expect_tx(bar(B_KVFULL + st), __popc(mine) * p.box * 128);
        __syncwarp();
        if (row >= 0)
          tma_load_3d(sbase + C::kOffKV + st * kTileBytes + boxes.offset, is_v ? &tmV : &tmK, bar(B_KVFULL + st),
                      boxes.half * 64, row, 0);
        ++L;
      }
    }
    // Drain: every load this warp issued must land before the CTA may exit.
    for (uint32_t i = L > static_cast<uint32_t>(kStages) ? L - kStages : 0u; i < L; ++i)
      mbar_wait_drain(bar(B_KVFULL + static_cast<int>(i % kStages)), (i / kStages) & 1u, SITE_DRAIN);
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (n_q[t] > 0) mbar_wait_drain(bar(B_QFULL + t), (n_q[t] - 1) & 1, SITE_DRAIN);
    __syncwarp();
  } else if (warp >= C::kWarpMma && warp < C::kWarpMma + NT) {
    // ------------------------------------------------------------ MMA issuers
    // One per Q tile: a single thread starts a 128x128x16 MMA only every ~85 cycles, a
    // third slower than the tensor core runs it.
    if constexpr (C::kSplitRegs) regs_dec<C::kRegsHelper>();
    const int tq = warp - C::kWarpMma;
    if (lane == 0) {
      constexpr uint32_t kIdQK = idesc_bf16_f32(128, kBN, false);
      constexpr uint32_t kIdPV = idesc_bf16_f32(128, kD, true);
      constexpr uint32_t kHi = sdesc_hi_sw128(1024);
      const uint32_t q_lo = sdesc_lo(sbase + C::kOffQ + tq * kTileBytes, 16);
      const uint32_t p_lo = sdesc_lo(sbase + C::kOffP + tq * kTileBytes, 16);
      const uint32_t kv_lo = sdesc_lo(sbase + C::kOffKV, 16);
      const uint32_t v_lo = sdesc_lo(sbase + C::kOffKV, kHalf);
      constexpr uint32_t kTile16 = kTileBytes / 16;
      const uint32_t dS = tmem + colS(tq), dO = tmem + colO(tq);
      auto issue_qk = [&](int st) {  // S_t = Q_t K^T over d = 128
        const uint32_t b0 = kv_lo + st * kTile16;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t off = ((kk >> 2) * kHalf + (kk & 3) * 32) / 16;
          umma_ss_lohi(dS, q_lo + off, b0 + off, kHi, kIdQK, kk > 0 ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int st, uint32_t acc) {  // O_t (+)= P_t V over 128 slots
        const uint32_t b0 = v_lo + st * kTile16;
        umma_ss_lohi(dO, p_lo, b0, kHi, kIdPV, acc);
#pragma unroll
        for (int kk = 1; kk < 8; ++kk) {
          const uint32_t off = ((kk >> 2) * kHalf + (kk & 3) * 32) / 16;
          umma_ss_lohi(dO, p_lo + off, b0 + kk * (2048 / 16), kHi, kIdPV, 1u);
        }
      };
      bool ok = true;
      uint32_t L = 0, Gb = 0, Z = 0;  // ring position, iterations of this tile, clearing events
      uint32_t uc = 0;                // segments with this tile
      Seg s;
      while (ok && next_seg(p, walk, s)) {
        const int n = s.k1 - s.k0;
        auto wait_kv = [&](uint32_t ii) -> bool {
          return mbar_wait_spin(bar(B_KVFULL + ii % kStages), (ii / kStages) & 1u, SITE_MMA);
        };
        if (tq * p.tpt >= s.n_tok) {
          // no rows in this tile: pass the stages on, in step with the ring
          for (int li = 0; ok && li < 2 * n; ++li) {
            ok = wait_kv(L + li);
            if (ok) mbar_arrive(bar(B_KVEMPTY + (L + li) % kStages));
          }
          if (ok) mbar_arrive(bar(B_QEMPTY));
        } else {
          ok = mbar_wait_spin(bar(B_QFULL + tq), uc & 1u, SITE_MMA) && wait_kv(L + load_idx_k(0)) &&
               (Gb == 0 || mbar_wait_spin(bar(B_SFREE + tq), (Gb - 1) & 1u, SITE_MMA));
          if (!ok) break;
          {
            const int sk = static_cast<int>((L + load_idx_k(0)) % kStages);
            tc_fence_after();
            issue_qk(sk);
            umma_commit(bar(B_SFULL + tq));
            umma_commit(bar(B_KVEMPTY + sk));
            if (n == 1) umma_commit(bar(B_QEMPTY));
          }
          for (int j = 0; ok && j < n; ++j) {
            const uint32_t g = Gb + j;
            const uint32_t iv = L + load_idx_v(j, n);
            const int sv = static_cast<int>(iv % kStages);
            if (j + 1 < n) {
              // next S as soon as this tile's softmax holds S(j) in registers
              const uint32_t ik = L + load_idx_k(j + 1);
              ok = wait_kv(ik) && mbar_wait_spin(bar(B_SFREE + tq), g & 1u, SITE_MMA);
              if (!ok) break;
              tc_fence_after();
              issue_qk(static_cast<int>(ik % kStages));
              umma_commit(bar(B_SFULL + tq));
              umma_commit(bar(B_KVEMPTY + ik % kStages));
              if (j + 1 == n - 1) umma_commit(bar(B_QEMPTY));
            }
            ok = wait_kv(iv) && mbar_wait_spin(bar(B_PREADY + tq), g & 1u, SITE_MMA);
            if (ok && j == n - 1 && s.tail()) ok = mbar_wait_spin(bar(B_VZERO + Z % 4), (Z / 4) & 1u, SITE_MMA);
            if (!ok) break;
            tc_fence_after();
            issue_pv(sv, j > 0 ? 1u : 0u);
            umma_commit(bar(B_PVDONE + tq));
            umma_commit(bar(B_KVEMPTY + sv));
          }
          Gb += n;
          ++uc;
        }
        if (s.tail()) ++Z;
        L += 2 * n;
      }
      umma_commit(bar(B_DRAIN + tq));
      mbar_wait_drain(bar(B_DRAIN + tq), 0, SITE_DRAIN);
    }
    __syncwarp();
  } else if (warp == C::kWarpHelper) {
    // ------------------------------------------------------------ V rows past the last slot
    if constexpr (C::kSplitRegs) regs_dec<C::kRegsHelper>();
    bool ok = true;
    uint32_t L = 0, Z = 0;
    Seg s;
    while (ok && next_seg(p, walk, s)) {
      const int n = s.k1 - s.k0;
      for (int li = 0; ok && li < 2 * n; ++li) {  // a reader like the issuers, in step with the ring
        const int st = static_cast<int>((L + li) % kStages);
        ok = __all_sync(0xffffffffu, mbar_wait(bar(B_KVFULL + st), ((L + li) / kStages) & 1u, SITE_HELPER));
        if (!ok) break;
        if (li == 2 * n - 1 && s.tail()) {
          const int first = s.limit - (s.count - 1) * kBN;  // rows [first, 128) of the V tile
          uint8_t* v = smem + C::kOffKV + st * kTileBytes;
          for (int i = first * 8 + lane; i < kBN * 8; i += 32) {
            *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(v + kHalf + i * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          mbar_arrive(bar(B_VZERO + Z % 4));
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(bar(B_KVEMPTY + st));
      }
      if (s.tail()) ++Z;
      L += 2 * n;
    }
  } else if (warp < C::kSoftmaxWarps) {
    // ------------------------------------------------------------ softmax warpgroups
    if constexpr (C::kSplitRegs) regs_inc<C::kRegsSoftmax>();
    const int g = warp >> 2;
    const int t = g >> 1;             // Q tile
    const int h = g & 1;              // slots [64h, 64h+64) of each K tile; O dims [64h, 64h+64)
    const int r = threadIdx.x & 127;  // row in tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + colS(t) + 64 * h;
    const uint32_t tO = tmem + lane_off + colO(t) + 64 * h;
    uint8_t* ptile = smem + C::kOffP + t * kTileBytes;
    float* xchg = reinterpret_cast<float*>(smem + C::kOffX) + t * 256;  // [half][row]
    const int bar_x = 1 + t;     // named barrier: both halves of tile t (256 threads)
    const int bar_free = 3 + t;  // named barrier: exchange slots may be rewritten
    const float sl2 = p.scale_log2;
    const int my_tok = r < p.tpt * p.G ? t * p.tpt + r / p.G : 0x3FFFFFFF;  // token in the unit
    bool ok = true;
    uint32_t Gb = 0;
    Seg s;
    // Every warp of the tile runs every iteration of every segment and meets every named
    // barrier, even after a bounded wait failed (ok == false only skips the work), so
    // the two halves of a tile can never wait on each other forever.
    while (next_seg(p, walk, s)) {
      if (t * p.tpt >= s.n_tok) continue;  // no rows in this tile
      const int n = s.k1 - s.k0;
      // last slot this row sees (a row without a token computes what nobody reads, unmasked,
      // so that its warp takes the masked path only where a real row needs it)
      const int lim = my_tok < s.n_tok ? (p.causal ? s.base + s.tok0 + my_tok : s.s.L - 1) : 0x3FFFFFFF;
      // warps without any token's row only keep the hand-offs going
      const bool work = __any_sync(0xffffffffu, my_tok < s.n_tok);
      float m_run = -INFINITY, l_run = 0.0f, lf_run = 0.0f;
      for (int j = 0; j < n; ++j) {
        const uint32_t gi = Gb + j;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_SFULL + t), gi & 1u, SITE_SOFTMAX));
        uint32_t s0[32], s1[32];
        float mx0 = -INFINITY, mx1 = -INFINITY;
        const int rel = lim - (s.k0 + j) * kBN - 64 * h;  // columns (of this half) > rel are masked
        if (ok && work) {
          tc_fence_after();
          tmem_ld32(tS + 0, s0);
          tmem_ld32(tS + 32, s1);
          tmem_wait_ld_dep(s0);
          reg_dep(s1);
          tc_fence_before();
        }
        if (ok) mbar_arrive(bar(B_SFREE + t));  // S_t may now be overwritten by the next QK^T
        if (ok && work) {
          if (rel < 63) {
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (k > rel) s0[k] = 0xFF800000u;
              if (k + 32 > rel) s1[k] = 0xFF800000u;
            }
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            mx0 = fmax3(mx0, __uint_as_float(s0[k]), __uint_as_float(s0[k + 1]));
            mx1 = fmax3(mx1, __uint_as_float(s1[k]), __uint_as_float(s1[k + 1]));
          }
        }
        // row max over both halves: slot [h][r] <-> [1-h][r]
        named_bar_sync(bar_free, 256);  // everyone has read the previous exchange's slots
        xchg[h * 128 + r] = fmaxf(mx0, mx1);
        named_bar_sync(bar_x, 256);
        const float m_tile = fmaxf(fmaxf(mx0, mx1), xchg[(1 - h) * 128 + r]) * sl2;
        const float m_new = fmaxf(m_run, m_tile);
        const bool need = m_new > m_run + kRescaleLog2;
        const float m_use = need ? m_new : m_run;
        const float alpha = need ? ex2_approx(m_run - m_new) : 1.0f;
        const float moff = (m_use == -INFINITY) ? 0.0f : m_use;
        // P_t's buffer (and O_t) are free once the previous PV finished
        if (ok && j > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_PVDONE + t), (gi - 1) & 1u, SITE_SOFTMAX));
        float2 sum = make_float2(0.f, 0.f), sumf = make_float2(0.f, 0.f);
        if (ok && work) {
          const float2 sc2 = make_float2(sl2, sl2), nm2 = make_float2(-moff, -moff);
          // Chunks with no masked entry may evaluate part of the exponentials on the FMA
          // pipe; its cubic is good to 7.5e-5, enough for a weight that is rounded to
          // bf16 but not for the log-sum-exp.
          if (rel >= 63) {
            exp_chunk_store<!kLse, kLse>(s0, ptile, r, 8 * h, sc2, nm2, sum, sumf);
            exp_chunk_store<!kLse, kLse>(s1, ptile, r, 8 * h + 4, sc2, nm2, sum, sumf);
          } else {
            exp_chunk_store<false, kLse>(s0, ptile, r, 8 * h, sc2, nm2, sum, sumf);
            exp_chunk_store<false, kLse>(s1, ptile, r, 8 * h + 4, sc2, nm2, sum, sumf);
          }
          fence_proxy_async_smem();
          if (j > 0 && __any_sync(0xffffffffu, need)) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + 32 * c, o);
              tmem_wait_ld_dep(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st32(tO + 32 * c, o);
            }
            tmem_wait_st();
          }
          tc_fence_before();
        }
        if (ok) mbar_arrive(bar(B_PREADY + t));
        l_run = l_run * alpha + (sum.x + sum.y);
        if (kLse) lf_run = lf_run * alpha + (sumf.x + sumf.y);
        m_run = m_use;
      }

      // ---- epilogue
      const uint32_t last = Gb + n - 1;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_PVDONE + t), last & 1u, SITE_EPILOGUE));
      named_bar_sync(bar_free, 256);
      xchg[h * 128 + r] = l_run;
      named_bar_sync(bar_x, 256);
      const float l_tot = l_run + xchg[(1 - h) * 128 + r];
      float lf_tot = 0.0f;
      if (kLse) {
        named_bar_sync(bar_free, 256);
        xchg[h * 128 + r] = lf_run;
        named_bar_sync(bar_x, 256);
        lf_tot = lf_run + xchg[(1 - h) * 128 + r];
      }
      if (ok && work) {
        tc_fence_after();
        const bool mine = my_tok < s.n_tok;
        const bool whole = s.whole();
        const int hd = r % p.G;
        if (whole) {
          const float inv_l = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
          const long long tok = s.s.a + s.tok0 + my_tok;
          const int head = s.h * p.G + hd;
          uint16_t* dst = p.o + tok * p.o_t + head * p.o_h + 64 * h;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + 32 * c, o);
            tmem_wait_ld_dep(o);
            if (mine) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint4 v;
                v.x = pack_bf16x2(__uint_as_float(o[q * 8 + 0]) * inv_l, __uint_as_float(o[q * 8 + 1]) * inv_l);
                v.y = pack_bf16x2(__uint_as_float(o[q * 8 + 2]) * inv_l, __uint_as_float(o[q * 8 + 3]) * inv_l);
                v.z = pack_bf16x2(__uint_as_float(o[q * 8 + 4]) * inv_l, __uint_as_float(o[q * 8 + 5]) * inv_l);
                v.w = pack_bf16x2(__uint_as_float(o[q * 8 + 6]) * inv_l, __uint_as_float(o[q * 8 + 7]) * inv_l);
                *reinterpret_cast<uint4*>(dst + 32 * c + 8 * q) = v;
              }
            }
          }
          if (kLse && mine && h == 0)
            p.lse[tok * p.Hq + head] = lf_tot > 0.0f ? (m_run + log2f(lf_tot)) * kLn2 : -INFINITY;
        } else {
          // a segment: (O, m, l) to this CTA's slot, 16 bytes of 32 rows side by side
          const int slot = 2 * blockIdx.x + (s.k0 == 0 ? 1 : 0);
          const int row = t * 128 + r;
          float4* dst = p.part_o + (static_cast<size_t>(slot) * 32 + 16 * h) * p.part_rows + row;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + 32 * c, o);
            tmem_wait_ld_dep(o);
            if (mine) {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                dst[static_cast<size_t>(8 * c + q) * p.part_rows] =
                    make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]), __uint_as_float(o[4 * q + 2]),
                                __uint_as_float(o[4 * q + 3]));
            }
          }
          if (mine && h == 0) {
            float* ml = p.part_ml + static_cast<size_t>(slot) * 3 * p.part_rows + row;
            ml[0] = m_run;
            ml[p.part_rows] = l_tot;
            ml[2 * p.part_rows] = lf_tot;
          }
        }
        tc_fence_before();  // O_t may be overwritten by the next segment's first PV
      }
      Gb += n;
    }
  }

  // ---- teardown: everyone done with TMEM and shared memory
  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 256 * NT);
  }
}

// Merge a split unit's segments: block (c, y) takes the unit that CTA c began, if any.
// O = sum_i O_i 2^(m_i - M) / sum_i l_i 2^(m_i - M), segments in order.  A thread holds
// eight dims of one row: 32 lanes read 32 rows' 16 bytes side by side.
constexpr int kMergeThreads = 128;
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const Params p, int nt) {
  cudaGridDependencySynchronize();
  const int c0 = blockIdx.x;
  const Desc d = p.desc[c0];
  if (!d.valid) return;
  const Seq s = seq_of(p.batch, d.b);
  const int n_tok = min(p.tu, s.n - d.u * p.tu);
  const int rows_tile = p.tpt * p.G;
  const int rows = n_tok > p.tpt ? 128 + (n_tok - p.tpt) * p.G : n_tok * p.G;
  const int lane = threadIdx.x & 31;
  const int items = ((rows + 31) / 32) * 16;  // (32 rows, 8 dims) per warp
  for (int it = blockIdx.y * (kMergeThreads / 32) + (threadIdx.x >> 5); it < items;
       it += gridDim.y * (kMergeThreads / 32)) {
    const int row = (it >> 4) * 32 + lane, d8 = it & 15;
    const int t = row >> 7, r = row & 127;
    if (row >= rows || r >= rows_tile) continue;
    auto ml_of = [&](int c, int k) {
      const size_t slot = 2 * static_cast<size_t>(c) + (c == c0 ? 1 : 0);
      return p.part_ml[(slot * 3 + k) * p.part_rows + row];
    };
    float M = -INFINITY;
    for (int c = c0; c <= d.last; ++c) M = fmaxf(M, ml_of(c, 0));
    float l = 0.0f, lf = 0.0f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 2
    for (int c = c0; c <= d.last; ++c) {
      const float m = ml_of(c, 0);
      const float w = m == -INFINITY ? 0.0f : ex2_approx(m - M);
      l += ml_of(c, 1) * w;
      if (p.lse) lf += ml_of(c, 2) * w;
      const size_t slot = 2 * static_cast<size_t>(c) + (c == c0 ? 1 : 0);
      const float4* o = p.part_o + (slot * 32 + 2 * d8) * p.part_rows + row;
      const float4 a = o[0], b = o[p.part_rows];
      acc[0] += a.x * w, acc[1] += a.y * w, acc[2] += a.z * w, acc[3] += a.w * w;
      acc[4] += b.x * w, acc[5] += b.y * w, acc[6] += b.z * w, acc[7] += b.w * w;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const long long tok = s.a + d.u * p.tu + t * p.tpt + r / p.G;
    const int head = d.h * p.G + r % p.G;
    *reinterpret_cast<uint4*>(p.o + tok * p.o_t + head * p.o_h + 8 * d8) =
        make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                   pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
    if (p.lse && d8 == 0) p.lse[tok * p.Hq + head] = lf > 0.0f ? (M + log2f(lf)) * kLn2 : -INFINITY;
  }
}

// ------------------------------------------------------------------ host side
struct Layout {
  size_t o, ml, desc, bytes;
  int rows;
};

// Workspace of segments: a unit has all of T's rows at most.
inline Layout layout_of(int T, int G) {
  Layout w;
  const int tpt = 128 / G;
  w.rows = T <= tpt ? T * G : 256;
  w.o = 0;
  w.ml = w.o + static_cast<size_t>(2 * kMaxCtas) * 32 * w.rows * sizeof(float4);
  w.desc = w.ml + (static_cast<size_t>(2 * kMaxCtas) * 3 * w.rows * sizeof(float) + 15) / 16 * 16;
  w.bytes = w.desc + kMaxCtas * sizeof(Desc);
  return w;
}

template <int NT, bool kLse>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& p, int grid,
           cudaStream_t stream) {
  using C = Cfg<NT>;
  auto* kernel = attend_kernel<NT, kLse>;
  static std::atomic<uint64_t> attr_done{0};
  int rc;
  if ((rc = ensure_smem_attr(kernel, C::kSmemBytes, attr_done)) != GQA_OK) return rc;
  if constexpr (C::kSplitRegs) {  // the register split assumes the compiled count
    static std::atomic<int> regs_ok{0};
    if (regs_ok.load(std::memory_order_acquire) == 0) {
      cudaFuncAttributes fa;
      if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess) return GQA_ERR_CUDA;
      regs_ok.store(fa.numRegs == C::kRegsLaunch ? 1 : -1, std::memory_order_release);
    }
    if (regs_ok.load(std::memory_order_acquire) < 0) return GQA_ERR_UNSUPPORTED;
  }
  kernel<<<grid, C::kThreads, C::kSmemBytes, stream>>>(q, k, v, p);
  return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

}  // namespace attend

GQA_ERROR_FLAG_ACCESSOR(error_flag_attend)

}  // namespace gqa

using namespace gqa;

extern "C" size_t gqa_attend_chunk_workspace_size(int T, int Hq, int Hkv) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 128) return 0;
  return attend::layout_of(T, Hq / Hkv).bytes;
}

extern "C" int gqa_attend_chunk_bf16(const void* q, long long q_token_stride, long long q_head_stride,
                                     const void* kpages, const void* vpages, const int32_t* block_table,
                                     int max_pages_per_seq, int page_size, int num_pages, const int32_t* q_start,
                                     const int32_t* lens, void* o, long long o_token_stride, long long o_head_stride,
                                     float* lse, void* workspace, size_t workspace_bytes, int B, int T, int Hq, int Hkv,
                                     int head_dim, int max_q_len, float scale, int flags, gqa_stream_t stream) {
  using namespace attend;
  if (B <= 0 || T < 0 || Hq <= 0 || Hkv <= 0 || max_pages_per_seq <= 0 || page_size <= 0 || num_pages <= 0)
    return GQA_ERR_INVALID_ARGUMENT;
  if (head_dim != kD || Hq % Hkv || page_size % 16) return GQA_ERR_UNSUPPORTED;
  if (!(scale > 0.0f) || !(scale < 1e30f) || (flags & ~GQA_FLAG_CAUSAL) || max_q_len < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (q_token_stride < 0 || q_head_stride < 0 || o_token_stride < 0 || o_head_stride < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (T == 0) return GQA_OK;
  if (!q || !kpages || !vpages || !block_table || !q_start || !lens || !o) return GQA_ERR_INVALID_ARGUMENT;
  if (!rows_apart(T, Hq, o_token_stride, o_head_stride, kD)) return GQA_ERR_INVALID_ARGUMENT;
  auto odd = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 4 != 0; };
  if (!aligned16(q) || !aligned16(kpages) || !aligned16(vpages) || !aligned16(o) || odd(block_table) || odd(q_start) ||
      odd(lens) || odd(lse) || !aligned16(workspace))
    return GQA_ERR_MISALIGNED;
  if ((T > 1 && (q_token_stride % 8 || o_token_stride % 8)) || (Hq > 1 && (q_head_stride % 8 || o_head_stride % 8)))
    return GQA_ERR_MISALIGNED;
  const int G = Hq / Hkv;
  const long long capacity = static_cast<long long>(max_pages_per_seq) * page_size;
  const long long pool_rows = static_cast<long long>(num_pages) * Hkv * page_size;
  if (G > 128 || B > kMaxB || capacity > 0x7FFFFF00LL || pool_rows > 0x7FFFFFFFLL) return GQA_ERR_UNSUPPORTED;
  // a TMA dimension needs a stride: heads or tokens that share one row are the caller's to expand
  if ((T > 1 && q_token_stride == 0) || (Hq > 1 && q_head_stride == 0)) return GQA_ERR_UNSUPPORTED;
  const Layout w = layout_of(T, G);
  if (!workspace || workspace_bytes < w.bytes) return GQA_ERR_WORKSPACE;

  Params p;
  p.batch = {block_table, q_start, lens, B, T, Hkv, static_cast<int>(capacity), max_pages_per_seq, page_size, num_pages};
  p.o = static_cast<uint16_t*>(o);
  p.lse = lse;
  char* ws = static_cast<char*>(workspace);
  p.part_o = reinterpret_cast<float4*>(ws + w.o);
  p.part_ml = reinterpret_cast<float*>(ws + w.ml);
  p.desc = reinterpret_cast<Desc*>(ws + w.desc);
  p.part_rows = w.rows;
  p.o_t = o_token_stride;
  p.o_h = o_head_stride;
  p.G = G, p.Hq = Hq;
  p.causal = (flags & GQA_FLAG_CAUSAL) != 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.box = std::min(128, page_size & -page_size);
  p.tpt = 128 / G;
  const int longest = max_q_len > 0 ? std::min(max_q_len, T) : T;
  const int nt = longest <= p.tpt ? 1 : 2;
  p.tu = nt * p.tpt;

  CUtensorMap tmQ, tmK, tmV;
  int rc;
  const long long ht = Hq > 1 ? q_head_stride : kD, tt = T > 1 ? q_token_stride : static_cast<long long>(Hq) * kD;
  const long long qd[4] = {kD, Hq, T, 1}, qs[3] = {ht * 2, tt * 2, tt * 2};
  const int qb[4] = {64, G, p.tpt, 1};
  if ((rc = make_tmap_4d(&tmQ, q, 2, qd, qs, qb)) != GQA_OK) return rc;
  if ((rc = make_tmap_3d_bf16(&tmK, kpages, kD, pool_rows, 1, 64, p.box, 1)) != GQA_OK) return rc;
  if ((rc = make_tmap_3d_bf16(&tmV, vpages, kD, pool_rows, 1, 64, p.box, 1)) != GQA_OK) return rc;

  int dev = 0, sms = kMaxCtas;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int grid = std::min(sms, kMaxCtas);
  if (nt == 1)
    rc = lse ? launch<1, true>(tmQ, tmK, tmV, p, grid, stream) : launch<1, false>(tmQ, tmK, tmV, p, grid, stream);
  else
    rc = lse ? launch<2, true>(tmQ, tmK, tmV, p, grid, stream) : launch<2, false>(tmQ, tmK, tmV, p, grid, stream);
  if (rc != GQA_OK) return rc;
  // The merge starts while the first kernel drains and waits for it on the device.
  const int rows = std::min(nt * 128, (longest * G + 31) / 32 * 32);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, std::max(1, rows / 32 * 16 / (kMergeThreads / 32)));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, merge_kernel, static_cast<const Params>(p), nt) == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}
