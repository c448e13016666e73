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
// group) pairs, so K and V are read once for all heads of the group and all tokens of
// the block.  A unit walks its K/V tiles of 128 slots with an online softmax, O rescaled
// only when a running maximum grows by more than 2^16.
//
// Two forms, chosen per sequence by its rows n G:
//  many  units of 256 rows, two Q tiles of 128 with one MMA issuer each.  S = Q K^T has a
//        row per TMEM lane; P goes to shared memory as the A operand of O += P V.
//  few   n G <= 32 (single tokens, short drafts): transposed, S^T = K Q^T and
//        O^T += V^T P^T with N = 16 or 32, so that the tensor core does no more work than
//        there are rows.  Such units are bound by memory, and padding 4 rows to 128
//        drew the GPU's whole power budget (1000 W at 1.39 GHz instead of 1.97: 64 tokens
//        over 1024..32768 slots took 813 us, where this form takes 652).
//
// Split: the units' K/V tiles form one line per form, and the CTAs (one per SM) are dealt
// out to the two lines by what a tile of each costs; each line is cut into equal parts
// (ragged.cuh).  A part may begin and end inside a unit; such segments leave (O, m, l) in the
// workspace and a second kernel merges them.  So one long sequence of a single token keeps
// every SM busy, and a prompt chunk uses the tensor cores of some SMs while the decode
// beside it streams the cache on the others.
//
// Pipeline (per CTA): a producer warp loads Q by TMA and streams K and V tiles through a
// ring, one box per page (or per part of a page inside a tile); issuer warps drive
// tcgen05.mma with accumulators in TMEM; softmax warps turn S into P; a helper warp clears
// V rows past the last slot that the unit sees (P is zero there, but a cache may hold
// anything, and 0 * NaN would spread).
//
// Measured (Hq 32, Hkv 8, both launches, replayed from a graph):
//   64 single tokens over 1024..32768 slots, 4.25 GB  652 us  6.5 TB/s, what a copy reaches
//   2048 tokens behind 30720 slots, 1.07 TFLOP        1102 us  970 TFLOP/s, 0.60 of a GEMM's burst: the
//     tensor pipe is busy for 52 % of the cycles, the rest is the softmax's exponentials and
//     hand-offs (sustained, the 1000 W limit makes it 1271 us)
//   512 tokens beside 31 sequences of 1..5, 315 MB    114 us  about half from each of the two lines (107
//     on another machine)
//   4 single tokens over 37..1023 slots               14.3 us  latency: plan, one or two tiles, merge
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

constexpr int kBlockRows = 16;             // rows of a block of the few-row form; a unit has one or two
// What one K/V tile costs in each form, for dealing out the CTAs: a tile of the few form is
// 64 KB from memory (1.3 us), one of the many form two tiles' softmax (2.3 to 3.0 us).  Tried on
// one step alone, 512 tokens beside 31 sequences of 1..5 with 32 and 8 heads: 3 : 5 took 9 % longer
// than 4 : 9, 2 : 5 took 3 % longer.  How many SMs stream, and units of a single Q tile, are not
// in it.
constexpr int kCostFew = 4, kCostMany = 9;
// and what a unit's beginning and end cost, in tiles.
constexpr int kExtraFew = 1, kExtraMany = 2;

constexpr int kWarpProducer = 16;
constexpr int kWarpMma = 17;  // and 18 for the second Q tile
constexpr int kWarpHelper = 19;
constexpr int kThreads = 640;
// Register split (setmaxnreg): the launch gives every thread kRegsLaunch registers; the sum
// of each form's shares must stay within the launch allocation, or setmaxnreg.inc would
// wait forever; the host checks the compiled count before the first launch.
constexpr int kRegsLaunch = 96, kRegsHelper = 64, kRegsMany = 104, kRegsFew = 144;
static_assert(4 * 128 * kRegsMany + 128 * kRegsHelper <= kThreads * kRegsLaunch, "register split over budget");
static_assert(2 * 128 * kRegsFew + 3 * 128 * kRegsHelper <= kThreads * kRegsLaunch, "register split over budget");

// Shared memory; the 1024-byte-aligned tiles come first.
struct Many {
  static constexpr int kStages = 3;
  static constexpr int kOffQ = 0, kQHalf = kHalf, kQTile = kTileBytes;  // [2 tiles][2 halves of 64 dims]
  static constexpr int kOffP = 2 * kTileBytes;
  static constexpr int kOffKV = 4 * kTileBytes;
};
struct Few {
  static constexpr int kStages = 6;
  static constexpr int kOffKV = 0;
  static constexpr int kSmall = kBlockRows * 128;  // 64 columns of a block: 2 KB
  static constexpr int kQHalf = kSmall, kQTile = 2 * kSmall;
  static constexpr int kOffQ = 6 * kTileBytes;        // [block][2 halves of 64 dims]
  static constexpr int kOffP = kOffQ + 2 * kQTile;    // [block][2 buffers][2 halves of 64 slots]
  static constexpr int kOffRed = kOffP + 8 * kSmall;  // [block][4 warps][16] floats
  static constexpr int kOffTok = kOffRed + 512;       // [16] token of a row in its block
};
constexpr int kOffX = 7 * kTileBytes;  // row exchange [tile][half][128]: halves differ in one address bit
constexpr int kOffBar = kOffX + 2 * 2 * 128 * 4;
constexpr int kNumBars = 50;
constexpr int kOffTmemPtr = kOffBar + kNumBars * 8;
constexpr int kOffStart = kOffTmemPtr + 16;  // this CTA's place on its line
constexpr int kOffCold = kOffStart + 48;  // [tile] what the many form's softmax needs only between segments
constexpr int kSmemBytes = kOffCold + 2 * 96;
static_assert(Few::kOffTok + 64 <= kOffX, "the few form's buffers");
static_assert(sizeof(Walk) <= 48, "room for the start");
static_assert(kSmemBytes <= 232448, "shared memory over the per-block limit");
static_assert(ragged::kPlanBytes <= kOffX, "the plan's scratch lies in the tiles");

enum : int {
  // [2]: of Q tile t (many) or block t (few)
  B_QFULL = 0,     // [2] Q landed
  B_QEMPTY = 2,    // [2] last QK^T of the segment complete
  B_KVFULL = 4,    // [6] K/V stage landed
  B_KVEMPTY = 10,  // [6] MMAs reading the stage completed (issuers + helper)
  B_SFULL = 16,    // [2] S_t = Q_t K^T complete
  B_SFREE = 18,    // [2] S_t copied to registers
  B_PREADY = 20,   // [2] P_t in shared memory, O_t rescaled
  B_PVDONE = 22,   // [2] O_t += P_t V complete
  B_VZERO = 24,    // [8] rows past the last seen slot cleared (event k in slot k % 8)
  B_DRAIN = 32,    // [2] every MMA of issuer t complete
  // the few form's hand-offs, [block][buffer]
  F_SFULL = 34,
  F_SFREE = 38,
  F_PREADY = 42,
  F_PVDONE = 46,
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
  int tpt, tu;     // query tokens per tile and per unit of the many form
  int few;         // query tokens of a block of the few form, for sequences of up to twice so many
  int box;         // rows of one K/V box: the largest power of two dividing page_size, <= 128
  int part_rows;
  float scale_log2;
};

// Units: blocks of tu query tokens.  Steps: K/V tiles over the slots [0, limit) that some
// row of the unit sees; one at least, so that rows without any slot are written too.
struct Line {
  int tu, causal, from, to;  // sequences with from <= n <= to new tokens
  int extra;
  __device__ __forceinline__ Line(const Params& p, bool many)
      : tu(many ? p.tu : 2 * p.few), causal(p.causal), from(many ? 2 * p.few + 1 : 1), to(many ? 0x7FFFFFFF : 2 * p.few),
        extra(many ? kExtraMany : kExtraFew) {}
  __device__ __forceinline__ bool has(const Seq& s) const { return s.n >= from && s.n <= to; }
  __device__ __forceinline__ int units(const Seq& s) const { return (s.n + tu - 1) / tu; }
  __device__ __forceinline__ bool ends(const Seq& s, int u) const { return (u + 1) * tu >= s.n; }
  __device__ __forceinline__ int limit(const Seq& s, int u) const {
    return causal ? max(0, s.L - s.n + min(s.n, (u + 1) * tu)) : s.L;
  }
  __device__ __forceinline__ int count(const Seq& s, int u) const { return max(1, (limit(s, u) + kBN - 1) / kBN); }
  __device__ __forceinline__ uint32_t before(const Seq& s, int k) const {
    if (!causal) return static_cast<uint32_t>(k) * (count(s, 0) + extra);
    const int n = units(s);
    uint32_t sum = 0;
    const int m = min(k, n - 1);  // the last unit may be shorter
    if (m > 0) {
      const int base = s.L - s.n;
      const int one = base >= kBN ? 0 : min(m, (kBN - base) / tu);  // units whose limit is at most one tile
      sum = one;
      if (m > one) sum += ragged::floor_sum(m - one, kBN, tu, base + (one + 1) * tu + kBN - 1);
    }
    if (k == n) sum += count(s, n - 1);
    return sum + k * extra;
  }
};

// A segment: a CTA's part of a unit.  Its rows lie in Q tiles (many) or blocks (few) t = 0, 1.
struct Seg : Part {
  int tok0, n_tok, base, limit;
  int tiles;   // bit t: tile t has rows
  int second;  // first token (of the unit) of tile 1 where both have rows
  // the unit's last slots lie in this segment and do not fill their tile
  __device__ __forceinline__ bool tail() const { return k1 == count && limit < count * kBN; }
  __device__ __forceinline__ bool has(int t) const { return (tiles >> t) & 1; }
  __device__ __forceinline__ int from(int t) const { return t == 1 && tiles == 3 ? second : 0; }
};

// Units of one block go to the two blocks in turn, so that one's end overlaps the next
// one's beginning.
__device__ __forceinline__ bool next_seg(const Params& p, Walk& w, Seg& x) {
  const bool many = w.line != 0;
  const Line line(p, many);
  if (!ragged::next_part(p.batch, line, w, x)) return false;
  x.tok0 = x.u * line.tu;
  x.n_tok = min(line.tu, x.s.n - x.tok0);
  x.base = x.s.L - x.s.n;
  x.limit = line.limit(x.s, x.u);
  x.second = many ? p.tpt : p.few;
  if (x.n_tok > x.second) {
    x.tiles = 3;
  } else if (many) {
    x.tiles = 1;
  } else {
    x.tiles = 1 << w.turn;
    w.turn ^= 1;
  }
  return true;
}

// ------------------------------------------------------------------ exponentials
// The softmax loop of the many form holds 64 scores a thread in the 104 registers that 512
// of them get, so its shared-memory operands are one 32-bit base each with the rest in the
// instruction.
template <int kOff>
__device__ __forceinline__ bool mbar_try_at(uint32_t base, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1 + %3], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(base), "r"(parity), "n"(kOff)
      : "memory");
  return ok != 0;
}
template <int kOff>
__device__ __forceinline__ bool mbar_wait_at(uint32_t base, uint32_t parity, int site) {
  if (mbar_try_at<kOff>(base, parity)) return true;
  return mbar_wait(base + kOff, parity, site);
}
template <int kOff>
__device__ __forceinline__ void mbar_arrive_at(uint32_t base) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0 + %1];" ::"r"(base), "n"(kOff) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t addr, float x) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}
__device__ __forceinline__ float ld_shared(uint32_t addr) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}

// One 32-column chunk of S -> p = 2^(s*scale_log2 - m) as bf16, stored straight into the
// K-major SW128 P tile: 16-byte chunk c of the row lies at row ^ 16 c (the swizzle flips address bits
// 4-6 by the row, which `row` holds already).  bf16 is the tensor core's operand type; outputs'
// error against 64 bits is 0.0023 of their norm, 0.0017 being the bf16 output's own.  acc sums
// the rounded p that P V multiplies, so that O / l is a mean whose weights add up to one; accf
// sums them unrounded, for the log-sum-exp.
template <bool kEmulate, bool kLse>
__device__ __forceinline__ void exp_chunk_store(const uint32_t (&s)[32], uint32_t row, int c0, float2 sc2, float2 nm2,
                                                float2& acc, float2& accf) {
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
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row ^ (16u * (c0 + c))), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3])
                 : "memory");
  }
}

// ------------------------------------------------------------------ shared roles
// Producer warp (all lanes): per segment K0, its Q tile(s), K1 V0 K2 V1 ...; K and V through the
// ring of C::kStages tiles.
template <class C>
__device__ __forceinline__ void produce(const Params& p, int q_tokens, const CUtensorMap* tmQ, const CUtensorMap* tmK,
                                        const CUtensorMap* tmV, uint32_t sbase, Walk walk, int lane) {
  constexpr int kStages = C::kStages;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  bool ok = true;
  uint32_t L = 0;               // K/V loads issued by this CTA (ring position)
  uint32_t n_q[2] = {0, 0};     // Q tiles loaded
  const Boxes boxes(p.box, lane);
  Seg s;
  while (ok && next_seg(p, walk, s)) {
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
        tma_load_3d(sbase + C::kOffKV + st * kTileBytes + boxes.offset, is_v ? tmV : tmK, bar(B_KVFULL + st),
                    boxes.half * 64, row, 0);
      ++L;
      if (li > 0) continue;
      // The first K tile is on its way.  A Q tile is reused once the last QK^T of its
      // previous segment is done.
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!s.has(t)) continue;
        if (ok && n_q[t] > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar(B_QEMPTY + t), (n_q[t] - 1) & 1, SITE_PRODUCER));
        if (!ok) break;
        ++n_q[t];
        if (lane == 0) {
          const uint32_t dst = sbase + C::kOffQ + t * C::kQTile;
          mbar_expect_tx(bar(B_QFULL + t), 2 * 128 * p.G * q_tokens);
          for (int e = 0; e < 2; ++e)
            tma_load_4d(dst + e * C::kQHalf, tmQ, bar(B_QFULL + t), 64 * e, s.h * p.G, s.s.a + s.tok0 + s.from(t), 0);
        }
      }
    }
  }
  // Drain: every load this warp issued must land before the CTA may exit.
  for (uint32_t i = L > static_cast<uint32_t>(kStages) ? L - kStages : 0u; i < L; ++i)
    mbar_wait_drain(bar(B_KVFULL + static_cast<int>(i % kStages)), (i / kStages) & 1u, SITE_DRAIN);
#pragma unroll
  for (int t = 0; t < 2; ++t)
    if (n_q[t] > 0) mbar_wait_drain(bar(B_QFULL + t), (n_q[t] - 1) & 1, SITE_DRAIN);
  __syncwarp();
}

// Helper warp: a reader of the ring like the issuers, in step with it, that clears the rows
// of a unit's last V tile past its last slot.
template <class C>
__device__ __forceinline__ void clear_tails(const Params& p, uint8_t* smem, uint32_t sbase, Walk walk, int lane) {
  constexpr int kStages = C::kStages;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  bool ok = true;
  uint32_t L = 0, Z = 0;
  Seg s;
  while (ok && next_seg(p, walk, s)) {
    const int n = s.k1 - s.k0;
    for (int li = 0; ok && li < 2 * n; ++li) {
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
        mbar_arrive(bar(B_VZERO + Z % 8));
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(bar(B_KVEMPTY + st));
    }
    if (s.tail()) ++Z;
    L += 2 * n;
  }
}

// ------------------------------------------------------------------ many rows
// MMA issuer of Q tile tq (one thread).  One per tile: a single thread starts a 128x128x16
// MMA only every ~85 cycles, a third slower than the tensor core runs it.
__device__ __forceinline__ void issue_many(const Params& p, uint32_t sbase, uint32_t tmem, Walk walk, int tq) {
  using C = Many;
  constexpr int kStages = C::kStages;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  constexpr uint32_t kIdQK = idesc_bf16_f32(128, kBN, false);
  constexpr uint32_t kIdPV = idesc_bf16_f32(128, kD, true);
  constexpr uint32_t kHi = sdesc_hi_sw128(1024);
  const uint32_t q_lo = sdesc_lo(sbase + C::kOffQ + tq * kTileBytes, 16);
  const uint32_t p_lo = sdesc_lo(sbase + C::kOffP + tq * kTileBytes, 16);
  const uint32_t kv_lo = sdesc_lo(sbase + C::kOffKV, 16);
  const uint32_t v_lo = sdesc_lo(sbase + C::kOffKV, kHalf);
  constexpr uint32_t kTile16 = kTileBytes / 16;
  const uint32_t dS = tmem + 128 * tq, dO = tmem + 256 + 128 * tq;
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
  auto wait_kv = [&](uint32_t ii) -> bool {
    return mbar_wait_spin(bar(B_KVFULL + ii % kStages), (ii / kStages) & 1u, SITE_MMA);
  };
  Seg s;
  while (ok && next_seg(p, walk, s)) {
    const int n = s.k1 - s.k0;
    if (!s.has(tq)) {
      // no rows in this tile: pass the stages on, in step with the ring
      for (int li = 0; ok && li < 2 * n; ++li) {
        ok = wait_kv(L + li);
        if (ok) mbar_arrive(bar(B_KVEMPTY + (L + li) % kStages));
      }
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
        if (n == 1) umma_commit(bar(B_QEMPTY + tq));
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
          if (j + 1 == n - 1) umma_commit(bar(B_QEMPTY + tq));
        }
        ok = wait_kv(iv) && mbar_wait_spin(bar(B_PREADY + tq), g & 1u, SITE_MMA);
        if (ok && j == n - 1 && s.tail()) ok = mbar_wait_spin(bar(B_VZERO + Z % 8), (Z / 8) & 1u, SITE_MMA);
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

// The many form's softmax threads hold two rows of 32 scores each, so what they need only
// between segments lies in shared memory: one warp per Q tile walks the line for its
// eight and writes the segment here.
struct Shared {
  Walk walk;
  int n, k0, whole;               // tiles of the segment (0: no more), its first, whether it is the unit
  int a, h, tok0, n_tok, base, L;
};
static_assert(sizeof(Shared) <= 96, "room for it");

// Softmax warps of the many form: four warpgroups, two per Q tile.
template <bool kLse>
__device__ __forceinline__ void softmax_many(const Params& p, uint8_t* smem, uint32_t sbase, uint32_t tmem, Walk walk,
                                             int warp) {
  using C = Many;
  const int g = warp >> 2;
  const int t = g >> 1;             // Q tile
  const int h = g & 1;              // slots [64h, 64h+64) of each K tile; O dims [64h, 64h+64)
  const int r = threadIdx.x & 127;  // row in tile == TMEM lane
  const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = tmem + lane_off + 128 * t + 64 * h;
  constexpr uint32_t kToO = 256;  // from S_t's columns to O_t's
  // row r of P_t's half h; its 16-byte chunks lie at prow ^ 16 c
  const uint32_t prow = sbase + C::kOffP + t * kTileBytes + h * kHalf + r * 128 + ((r & 7) << 4);
  const uint32_t hot = sbase + kOffBar + 8 * t;                     // this tile's barriers
  const uint32_t own = sbase + kOffX + 1024 * t + 512 * h + 4 * r;  // exchange; the other half's at own ^ 512
  const int bar_x = 1 + t;     // named barrier: both halves of tile t (256 threads)
  const int bar_free = 3 + t;  // named barrier: exchange slots may be rewritten
  constexpr int kNoToken = 0x3FFFFFFF;
  volatile Shared* seg = reinterpret_cast<volatile Shared*>(smem + kOffCold + 96 * t);
  if (h == 0 && (warp & 3) == 0 && (threadIdx.x & 31) == 0) const_cast<Shared*>(seg)->walk = walk;
  bool ok = true;
  uint32_t phase = 0;  // parity of this tile's iterations
  // Every warp of the tile runs every iteration of every segment and meets every named
  // barrier, even after a bounded wait failed (ok == false only skips the work), so
  // the two halves of a tile can never wait on each other forever.
  for (;;) {
    named_bar_sync(bar_free, 256);  // the previous segment has been read
    if (h == 0 && (warp & 3) == 0) {
      __syncwarp();
      Walk w = const_cast<Shared*>(seg)->walk;
      Seg s;
      bool more;
      do more = next_seg(p, w, s);
      while (more && !s.has(t));
      __syncwarp();
      if ((threadIdx.x & 31) == 0) {
        Shared& x = *const_cast<Shared*>(seg);
        x.walk = w;
        x.n = more ? s.k1 - s.k0 : 0;
        x.k0 = s.k0, x.whole = s.whole();
        x.a = s.s.a, x.h = s.h, x.tok0 = s.tok0, x.n_tok = s.n_tok, x.base = s.base, x.L = s.s.L;
      }
    }
    named_bar_sync(bar_x, 256);
    const int n = seg->n;
    if (n == 0) break;
    int rel;  // the last column of this half of the next tile that this row sees
    bool mine;
    {
      // A row without a token computes what nobody reads, unmasked, so that its warp takes
      // the masked path only where a real row needs it.
      const int my_tok = r < p.tpt * p.G ? t * p.tpt + r / p.G : kNoToken;  // token in the unit
      mine = my_tok < seg->n_tok;
      rel = mine ? (p.causal ? seg->base + seg->tok0 + my_tok : seg->L - 1) - seg->k0 * kBN - 64 * h : kNoToken;
    }
    // warps without any token's row only keep the hand-offs going
    const bool work = __any_sync(0xffffffffu, mine);
    float m_run = -INFINITY, l_run = 0.0f, lf_run = 0.0f;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait_at<8 * B_SFULL>(hot, phase, SITE_SOFTMAX));
      uint32_t s0[32], s1[32];
      float mx0 = -INFINITY, mx1 = -INFINITY;
      if (ok && work) {
        tc_fence_after();
        tmem_ld32(tS + 0, s0);
        tmem_ld32(tS + 32, s1);
        tmem_wait_ld_dep(s0);
        reg_dep(s1);
        tc_fence_before();
      }
      if (ok) mbar_arrive_at<8 * B_SFREE>(hot);  // S_t may now be overwritten by the next QK^T
      if (ok && work) {
        if (rel < 63) {  // columns of this half > rel are masked
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
      mx0 = fmaxf(mx0, mx1);
      // row max over both halves
      named_bar_sync(bar_free, 256);  // everyone has read the previous exchange's slots
      st_shared(own, mx0);
      named_bar_sync(bar_x, 256);
      const float m_new = fmaxf(m_run, fmaxf(mx0, ld_shared(own ^ 512u)) * p.scale_log2);
      const bool need = m_new > m_run + kRescaleLog2;
      const float alpha = need ? ex2_approx(m_run - m_new) : 1.0f;
      m_run = need ? m_new : m_run;
      // P_t's buffer (and O_t) are free once the previous PV finished
      if (ok && j > 0) ok = __all_sync(0xffffffffu, mbar_wait_at<8 * B_PVDONE>(hot, phase ^ 1u, SITE_SOFTMAX));
      l_run *= alpha;
      if (kLse) lf_run *= alpha;
      if (ok && work) {
        const float moff = (m_run == -INFINITY) ? 0.0f : -m_run;
        const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), nm2 = make_float2(moff, moff);
        float2 sum = make_float2(0.f, 0.f), sumf = make_float2(0.f, 0.f);
        uint32_t row = prow;
        asm volatile("" : "+r"(row));  // keeps the chunks' addresses from living across the loop
        // Chunks with no masked entry may evaluate part of the exponentials on the FMA pipe.
        // Its cubic is good to 7.5e-5, enough for a weight that is rounded to bf16 but not
        // for the log-sum-exp (where a quintic measured no faster than none).  So the output's
        // last bits depend on whether the log-sum-exp is wanted.
        if (rel >= 63) {
          exp_chunk_store<!kLse, kLse>(s0, row, 0, sc2, nm2, sum, sumf);
          exp_chunk_store<!kLse, kLse>(s1, row, 4, sc2, nm2, sum, sumf);
        } else {
          exp_chunk_store<false, kLse>(s0, row, 0, sc2, nm2, sum, sumf);
          exp_chunk_store<false, kLse>(s1, row, 4, sc2, nm2, sum, sumf);
        }
        l_run += sum.x + sum.y;
        if (kLse) lf_run += sumf.x + sumf.y;
        fence_proxy_async_smem();
        if (j > 0 && __any_sync(0xffffffffu, need)) {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t o[32];
            tmem_ld32(tS + kToO + 32 * c, o);
            tmem_wait_ld_dep(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st32(tS + kToO + 32 * c, o);
          }
          tmem_wait_st();
        }
        tc_fence_before();
      }
      if (ok) mbar_arrive_at<8 * B_PREADY>(hot);
      phase ^= 1u;
      if (mine) rel -= kBN;
    }

    // ---- epilogue
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait_at<8 * B_PVDONE>(hot, phase ^ 1u, SITE_EPILOGUE));
    named_bar_sync(bar_free, 256);
    st_shared(own, l_run);
    named_bar_sync(bar_x, 256);
    const float l_tot = l_run + ld_shared(own ^ 512u);
    float lf_tot = 0.0f;
    if (kLse) {
      named_bar_sync(bar_free, 256);
      st_shared(own, lf_run);
      named_bar_sync(bar_x, 256);
      lf_tot = lf_run + ld_shared(own ^ 512u);
    }
    if (ok && work) {
      tc_fence_after();
      if (seg->whole) {
        const float inv_l = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
        const long long tok = seg->a + seg->tok0 + t * p.tpt + r / p.G;
        const int head = seg->h * p.G + r % p.G;
        uint16_t* dst = p.o + tok * p.o_t + head * p.o_h + 64 * h;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t o[32];
          tmem_ld32(tS + kToO + 32 * c, o);
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
        const int slot = 2 * blockIdx.x + (seg->k0 == 0 ? 1 : 0);
        const int row = t * 128 + r;
        float4* dst = p.part_o + (static_cast<size_t>(slot) * 32 + 16 * h) * p.part_rows + row;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t o[32];
          tmem_ld32(tS + kToO + 32 * c, o);
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
  }
}

// ------------------------------------------------------------------ few rows
// Two blocks of 16 rows, each with its issuer, its softmax warpgroup, its Q, its P and S^T
// double buffers and its O^T; both read the same ring.  TMEM: S^T of block t, buffer b at
// column 32 t + 16 b, O^T of block t at 64 + 16 t.
__device__ __forceinline__ void issue_few(const Params& p, uint32_t sbase, uint32_t tmem, Walk walk, int tq) {
  using C = Few;
  constexpr int kStages = C::kStages;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  constexpr uint32_t kHi = sdesc_hi_sw128(1024);
  constexpr uint32_t kIdQK = idesc_bf16_f32(128, kBlockRows, false);
  constexpr uint32_t kIdPV = idesc_bf16_f32(128, kBlockRows, false) | (1u << 15);  // A (V^T) MN-major
  const uint32_t kv_lo = sdesc_lo(sbase + C::kOffKV, 16);
  const uint32_t vt_lo = sdesc_lo(sbase + C::kOffKV, kHalf);
  const uint32_t q_lo = sdesc_lo(sbase + C::kOffQ + tq * C::kQTile, 16);
  const uint32_t p_lo = sdesc_lo(sbase + C::kOffP + tq * 4 * C::kSmall, 16);
  const uint32_t dS = tmem + 32 * tq, dO = tmem + 64 + 16 * tq;
  constexpr uint32_t kTile16 = kTileBytes / 16;
  auto issue_qk = [&](int st, int bb) {  // S^T = K Q^T
    const uint32_t a0 = kv_lo + st * kTile16;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      umma_ss_lohi(dS + 16u * bb, a0 + ((kk >> 2) * kHalf + (kk & 3) * 32) / 16,
                   q_lo + ((kk >> 2) * C::kSmall + (kk & 3) * 32) / 16, kHi, kIdQK, kk > 0 ? 1u : 0u);
  };
  auto issue_pv = [&](int st, int bb, uint32_t acc) {  // O^T (+)= V^T P^T
    const uint32_t a0 = vt_lo + st * kTile16;
    const uint32_t b0 = p_lo + bb * (2 * C::kSmall / 16);
    umma_ss_lohi(dO, a0, b0, kHi, kIdPV, acc);
#pragma unroll
    for (int kk = 1; kk < 8; ++kk)
      umma_ss_lohi(dO, a0 + kk * (2048 / 16), b0 + ((kk >> 2) * C::kSmall + (kk & 3) * 32) / 16, kHi, kIdPV, 1u);
  };
  bool ok = true;
  uint32_t L = 0, Gb = 0, Z = 0, uc = 0;  // ring position, this block's iterations, clearing events, segments
  auto wait_kv = [&](uint32_t ii) -> bool {
    return mbar_wait_spin(bar(B_KVFULL + ii % kStages), (ii / kStages) & 1u, SITE_MMA);
  };
  auto qk = [&](uint32_t ik, uint32_t g, bool last) -> bool {
    const int hb = 2 * tq + (g & 1);
    if (!wait_kv(ik)) return false;
    if (g >= 2 && !mbar_wait_spin(bar(F_SFREE + hb), ((g >> 1) - 1) & 1u, SITE_MMA)) return false;
    tc_fence_after();
    issue_qk(static_cast<int>(ik % kStages), static_cast<int>(g & 1));
    umma_commit(bar(F_SFULL + hb));
    umma_commit(bar(B_KVEMPTY + ik % kStages));
    if (last) umma_commit(bar(B_QEMPTY + tq));
    return true;
  };
  Seg s;
  while (ok && next_seg(p, walk, s)) {
    const int n = s.k1 - s.k0;
    if (!s.has(tq)) {
      for (int li = 0; ok && li < 2 * n; ++li) {  // pass the stages on, in step with the ring
        ok = wait_kv(L + li);
        if (ok) mbar_arrive(bar(B_KVEMPTY + (L + li) % kStages));
      }
    } else {
      ok = mbar_wait_spin(bar(B_QFULL + tq), uc & 1u, SITE_MMA) && qk(L + load_idx_k(0), Gb, n == 1);
      for (int j = 0; ok && j < n; ++j) {
        const uint32_t g = Gb + j, iv = L + load_idx_v(j, n);
        const int hb = 2 * tq + (g & 1);
        if (j + 1 < n) ok = qk(L + load_idx_k(j + 1), g + 1, j + 1 == n - 1);
        ok = ok && wait_kv(iv) && mbar_wait_spin(bar(F_PREADY + hb), (g >> 1) & 1u, SITE_MMA);
        if (ok && j == n - 1 && s.tail()) ok = mbar_wait_spin(bar(B_VZERO + Z % 8), (Z / 8) & 1u, SITE_MMA);
        if (!ok) break;
        tc_fence_after();
        issue_pv(static_cast<int>(iv % kStages), static_cast<int>(g & 1), j > 0 ? 1u : 0u);
        umma_commit(bar(F_PVDONE + hb));
        umma_commit(bar(B_KVEMPTY + iv % kStages));
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

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  tmem_wait_ld_dep16(r);
}

// Whether `v` holds for any of the barrier's threads.
__device__ __forceinline__ bool named_bar_any(int id, int nthreads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, %3, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "r"(id), "r"(nthreads)
      : "memory");
  return r != 0;
}

// One segment by block wg's softmax warpgroup: thread i holds slot i of each S^T tile, then
// dim i of O^T.  The maximum of a row lies across the threads, so it is not taken per
// tile: a tile only asks whether any score passes its row's running maximum by more than
// 2^16 (one barrier vote), which after the first tile hardly ever happens.
template <bool kLse>
__device__ __forceinline__ void softmax_few(const Params& p, const Seg& s, uint8_t* smem, uint32_t sbase, uint32_t tmem,
                                            uint32_t& Gb, bool& ok) {
  using C = Few;
  constexpr int N = kBlockRows;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };
  const int i = threadIdx.x & 127, wq = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int wg = threadIdx.x >> 7;
  const uint32_t t_lane = tmem + (static_cast<uint32_t>(wq * 32) << 16);
  const uint32_t tS = t_lane + 32 * wg, tO = t_lane + 64 + 16 * wg;
  const int bar_vote = 1 + wg, bar_red = 3 + wg;
  float* red = reinterpret_cast<float*>(smem + C::kOffRed) + 64 * wg;  // [4 warps][16]
  const int* tok = reinterpret_cast<const int*>(smem + C::kOffTok);
  const int n = s.k1 - s.k0;
  const int first_tok = s.from(wg);
  const float sl2 = p.scale_log2;
  float m[N], l[N], lf[kLse ? N : 1];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    m[c] = -INFINITY;
    l[c] = 0.0f;
    if (kLse) lf[c] = 0.0f;
  }
  // x[c] of all 128 threads combined: across a warp by halves (each step exchanges half of
  // the columns left, so lanes 2c and 2c + 1 end with column c: 16 shuffles, not 80), across
  // the warps through `red`
  auto across = [&](float (&x)[N], bool take_max) {
    float y[N];
#pragma unroll
    for (int c = 0; c < N; ++c) y[c] = x[c];
#pragma unroll
    for (int o = N; o >= 2; o /= 2) {
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int c = 0; c < o / 2; ++c) {
        const float give = up ? y[c] : y[c + o / 2], keep = up ? y[c + o / 2] : y[c];
        const float got = __shfl_xor_sync(0xffffffffu, give, o);
        y[c] = take_max ? fmaxf(keep, got) : keep + got;
      }
    }
    const float z = __shfl_xor_sync(0xffffffffu, y[0], 1);
    if ((lane & 1) == 0) red[wq * N + (lane >> 1)] = take_max ? fmaxf(y[0], z) : y[0] + z;
    named_bar_sync(bar_red, 128);
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      float4 v[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) v[w] = *reinterpret_cast<const float4*>(red + w * N + c);
      x[c] = take_max ? fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x)) : (v[0].x + v[1].x) + (v[2].x + v[3].x);
      x[c + 1] = take_max ? fmaxf(fmaxf(v[0].y, v[1].y), fmaxf(v[2].y, v[3].y)) : (v[0].y + v[1].y) + (v[2].y + v[3].y);
      x[c + 2] = take_max ? fmaxf(fmaxf(v[0].z, v[1].z), fmaxf(v[2].z, v[3].z)) : (v[0].z + v[1].z) + (v[2].z + v[3].z);
      x[c + 3] = take_max ? fmaxf(fmaxf(v[0].w, v[1].w), fmaxf(v[2].w, v[3].w)) : (v[0].w + v[1].w) + (v[2].w + v[3].w);
    }
  };
  for (int j = 0; j < n; ++j) {
    const uint32_t g = Gb + j;
    const int bb = static_cast<int>(g & 1), hb = 2 * wg + bb;
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(F_SFULL + hb), (g >> 1) & 1u, SITE_SOFTMAX));
    uint32_t sv[N];
    if (ok) {
      tc_fence_after();
      tmem_ld16(tS + 16 * bb, sv);
      tc_fence_before();
      mbar_arrive(bar(F_SFREE + hb));
    } else {
#pragma unroll
      for (int c = 0; c < N; ++c) sv[c] = 0xFF800000u;
    }
    const int slot0 = (s.k0 + j) * kBN, key = slot0 + i;
    if (slot0 + kBN - 1 > (p.causal ? s.base + first_tok : s.s.L - 1)) {  // some row does not see all of the tile
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (key > (p.causal ? min(s.base + first_tok + tok[c], s.s.L - 1) : s.s.L - 1)) sv[c] = 0xFF800000u;
    }
    float big = -INFINITY;  // -m is +inf as long as the row has seen nothing: its first score votes
#pragma unroll
    for (int c = 0; c < N; ++c) big = fmaxf(big, fmaf(__uint_as_float(sv[c]), sl2, -m[c]));
    if (named_bar_any(bar_vote, 128, big > kRescaleLog2)) {
      float x[N];
#pragma unroll
      for (int c = 0; c < N; ++c) x[c] = __uint_as_float(sv[c]);
      across(x, true);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const float m_new = fmaxf(m[c], x[c] * sl2);
        const bool need = m_new > m[c] + kRescaleLog2;
        x[c] = need ? ex2_approx(m[c] - m_new) : 1.0f;
        m[c] = need ? m_new : m[c];
        l[c] *= x[c];
        if (kLse) lf[c] *= x[c];
      }
      if (j > 0) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(F_PVDONE + (hb ^ 1)), ((g - 1) >> 1) & 1u, SITE_SOFTMAX));
        if (ok) {
          uint32_t o[N];
          tc_fence_after();
          tmem_ld16(tO, o);
#pragma unroll
          for (int c = 0; c < N; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * x[c]);
          tmem_st16(tO, o);
          tmem_wait_st();
        }
      }
    }
    // P's buffer is free once the PV of two tiles ago finished
    if (ok && j >= 2) ok = __all_sync(0xffffffffu, mbar_wait(bar(F_PVDONE + hb), ((g - 2) >> 1) & 1u, SITE_SOFTMAX));
    if (ok) {
      uint8_t* dst = smem + C::kOffP + hb * 2 * C::kSmall + (i >> 6) * C::kSmall + (i & 7) * 2;
      const int chunk = (i & 63) >> 3;
#pragma unroll
      for (int c = 0; c < N; c += 2) {
        const float e0 = ex2_approx(fmaf(__uint_as_float(sv[c]), sl2, m[c] == -INFINITY ? 0.0f : -m[c]));
        const float e1 = ex2_approx(fmaf(__uint_as_float(sv[c + 1]), sl2, m[c + 1] == -INFINITY ? 0.0f : -m[c + 1]));
        if (kLse) {
          lf[c] += e0;
          lf[c + 1] += e1;
        }
        const uint32_t w = pack_bf16x2(e0, e1);
        l[c] += bf16_lo(w);
        l[c + 1] += bf16_hi(w);
        *reinterpret_cast<uint16_t*>(dst + c * 128 + ((chunk ^ (c & 7)) << 4)) = static_cast<uint16_t>(w);
        *reinterpret_cast<uint16_t*>(dst + (c + 1) * 128 + ((chunk ^ ((c + 1) & 7)) << 4)) = static_cast<uint16_t>(w >> 16);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(bar(F_PREADY + hb));
    }
  }
  Gb += n;

  // ---- epilogue.  The last PV needed every thread's P, so `red` has been read.
  const uint32_t last = Gb - 1;
  if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(F_PVDONE + 2 * wg + (last & 1)), (last >> 1) & 1u, SITE_EPILOGUE));
  float my_l = 0.0f, my_lf = 0.0f;  // of row i, where this thread is the one that writes it
  auto mine = [&]() { return i < N ? (red[i] + red[N + i]) + (red[2 * N + i] + red[3 * N + i]) : 0.0f; };
  across(l, false);
  my_l = mine();
  if constexpr (kLse) {
    named_bar_sync(bar_vote, 128);
    across(lf, false);
    my_lf = mine();
  }
  if (!ok) return;
  uint32_t o[N];
  tc_fence_after();
  tmem_ld16(tO, o);
  tc_fence_before();  // O^T may be overwritten by the block's next segment
  const int rows = min(p.few, s.n_tok - first_tok) * p.G;
  float my_m = m[0];
#pragma unroll
  for (int c = 1; c < N; ++c) my_m = i == c ? m[c] : my_m;
  if (s.whole()) {
    const int tok0 = s.s.a + s.tok0 + first_tok;
    uint16_t* dst = p.o + static_cast<long long>(tok0) * p.o_t + static_cast<long long>(s.h) * p.G * p.o_h + i;
    const long long wrap = p.o_t - (p.G - 1) * p.o_h;  // from a token's last head to the next token's first
    int hd = 0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (c < rows)
        *dst = static_cast<uint16_t>(pack_bf16x2(l[c] > 0.0f ? __uint_as_float(o[c]) * __fdividef(1.0f, l[c]) : 0.0f, 0.0f));
      const bool end = ++hd == p.G;
      dst += end ? wrap : p.o_h;
      if (end) hd = 0;
    }
    if (kLse && i < rows)
      p.lse[static_cast<size_t>(tok0 + i / p.G) * p.Hq + s.h * p.G + i % p.G] =
          my_lf > 0.0f ? (my_m + log2f(my_lf)) * kLn2 : -INFINITY;
  } else {
    const int slot = 2 * blockIdx.x + (s.k0 == 0 ? 1 : 0), row0 = first_tok * p.G;
    float* dst =
        reinterpret_cast<float*>(p.part_o + (static_cast<size_t>(slot) * 32 + (i >> 2)) * p.part_rows + row0) + (i & 3);
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < rows) dst[4 * c] = __uint_as_float(o[c]);
    if (i < rows) {
      float* ml = p.part_ml + static_cast<size_t>(slot) * 3 * p.part_rows + row0 + i;
      ml[0] = my_m;
      ml[p.part_rows] = my_l;
      ml[2 * p.part_rows] = my_lf;
    }
  }
}

template <bool kLse>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQfew,
                  const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // uniform across the CTA: leave before any barrier
    if (threadIdx.x == 0) record_error(SITE_SMEM_ALIGN);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  auto bar = [&](int i) -> uint32_t { return sbase + kOffBar + 8 * i; };

  if (warp == kWarpMma) {
    tmem_alloc(sbase + kOffTmemPtr, 512);
    tmem_relinquish();
  }
  if (warp == kWarpHelper) {  // a barrier a lane
    static_assert(kNumBars <= 64, "two a lane");
    for (int i = lane; i < kNumBars; i += 32) {
      int count = 1;
      if (i >= B_KVEMPTY && i < B_SFULL) count = 3;    // issuers and helper
      if (i >= B_SFREE && i < B_PVDONE) count = 256;   // softmax threads of a hand-off
      if (i >= B_VZERO && i < B_DRAIN) count = 32;
      if (i >= F_SFREE && i < F_PVDONE) count = 128;
      mbar_init(bar(i), count);
    }
    fence_mbar_init();
  }
  if (warp == kWarpProducer && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmQfew);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  {
    const Line lines[2] = {Line(p, false), Line(p, true)};
    const int cost[2] = {kCostFew, kCostMany};
    ragged::plan<kThreads>(p.batch, lines, cost, reinterpret_cast<uint32_t*>(smem),
                           reinterpret_cast<Walk*>(smem + kOffStart), p.desc, SITE_Q_START, SITE_LENGTH);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kOffTmemPtr);
  const Walk walk = *reinterpret_cast<const Walk*>(smem + kOffStart);
  const bool many = walk.line != 0;
  if (!many) {
    // Q rows that no box fills stay zero; the token of each row
    for (int i = threadIdx.x; i < 2 * Few::kQTile / 16; i += kThreads)
      reinterpret_cast<uint4*>(smem + Few::kOffQ)[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < kBlockRows) reinterpret_cast<int*>(smem + Few::kOffTok)[threadIdx.x] = threadIdx.x / p.G;
  }
  // Generic writes (the plan's scratch, zeros) lie where TMA will write.
  fence_proxy_async_smem();
  __syncthreads();

  if (warp >= kWarpProducer) {
    regs_dec<kRegsHelper>();
    if (warp == kWarpProducer) {
      if (many)
        produce<Many>(p, p.tpt, &tmQ, &tmK, &tmV, sbase, walk, lane);
      else
        produce<Few>(p, p.few, &tmQfew, &tmK, &tmV, sbase, walk, lane);
    } else if (warp == kWarpHelper) {
      if (many)
        clear_tails<Many>(p, smem, sbase, walk, lane);
      else
        clear_tails<Few>(p, smem, sbase, walk, lane);
    } else {
      if (lane == 0) {
        if (many)
          issue_many(p, sbase, tmem, walk, warp - kWarpMma);
        else
          issue_few(p, sbase, tmem, walk, warp - kWarpMma);
      }
      __syncwarp();
    }
  } else if (many) {
    regs_inc<kRegsMany>();
    softmax_many<kLse>(p, smem, sbase, tmem, walk, warp);
  } else if (warp < 8) {
    regs_inc<kRegsFew>();
    Walk w = walk;
    Seg s;
    bool ok = true;
    uint32_t Gb = 0;
    while (next_seg(p, w, s))
      if (s.has(threadIdx.x >> 7)) softmax_few<kLse>(p, s, smem, sbase, tmem, Gb, ok);
  } else {
    regs_dec<kRegsHelper>();
  }

  // ---- teardown: everyone done with TMEM and shared memory
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merge a split unit's segments: block (c, y) takes the unit that CTA c began, if any.
// O = sum_i O_i 2^(m_i - M) / sum_i l_i 2^(m_i - M), segments in order.  A thread holds
// eight dims of one row: 32 lanes read 32 rows' 16 bytes side by side.
constexpr int kMergeThreads = 128;
constexpr int kBatch = 4;
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const Params p) {
  cudaGridDependencySynchronize();
  const int c0 = blockIdx.x;
  const Desc d = p.desc[c0];
  if (!d.valid) return;
  const Seq& s = d.s;
  const int tu = s.n <= 2 * p.few ? 2 * p.few : p.tu;
  const int n_tok = min(tu, s.n - d.u * tu);
  const int rows_tile = p.tpt * p.G;
  const int rows = n_tok > p.tpt ? 128 + (n_tok - p.tpt) * p.G : n_tok * p.G;
  const int lane = threadIdx.x & 31;
  const int items = ((rows + 31) / 32) * 16;  // (32 rows, 8 dims) per warp
  for (int it = blockIdx.y * (kMergeThreads / 32) + (threadIdx.x >> 5); it < items;
       it += gridDim.y * (kMergeThreads / 32)) {
    const int row = (it >> 4) * 32 + lane, d8 = it & 15;
    const int t = row >> 7, r = row & 127;
    if (row >= rows || r >= rows_tile) continue;
    float M = -INFINITY, l = 0.0f, lf = 0.0f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    // kBatch segments at a time, so that their loads' latencies overlap
    for (int c = c0; c <= d.last; c += kBatch) {
      float m[kBatch], li[kBatch], lfi[kBatch];
      float4 a[kBatch], b[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        m[i] = -INFINITY, li[i] = lfi[i] = 0.0f;
        a[i] = b[i] = make_float4(0, 0, 0, 0);
        if (c + i <= d.last) {
          const size_t slot = 2 * static_cast<size_t>(c + i) + (c + i == c0 ? 1 : 0);
          const float* ml = p.part_ml + slot * 3 * p.part_rows + row;
          const float4* o = p.part_o + (slot * 32 + 2 * d8) * p.part_rows + row;
          m[i] = ml[0];
          li[i] = ml[p.part_rows];
          if (p.lse) lfi[i] = ml[2 * p.part_rows];
          a[i] = o[0];
          b[i] = o[p.part_rows];
        }
      }
      float top = M;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) top = fmaxf(top, m[i]);
      const float keep = M == -INFINITY ? 0.0f : ex2_approx(M - top);
      l *= keep;
      lf *= keep;
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] *= keep;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float w = m[i] == -INFINITY ? 0.0f : ex2_approx(m[i] - top);
        l += li[i] * w;
        lf += lfi[i] * w;
        acc[0] += a[i].x * w, acc[1] += a[i].y * w, acc[2] += a[i].z * w, acc[3] += a[i].w * w;
        acc[4] += b[i].x * w, acc[5] += b[i].y * w, acc[6] += b[i].z * w, acc[7] += b[i].w * w;
      }
      M = top;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const long long tok = s.a + d.u * tu + t * p.tpt + r / p.G;
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

template <bool kLse>
int launch(const CUtensorMap& q, const CUtensorMap& q_few, const CUtensorMap& k, const CUtensorMap& v, const Params& p,
           int grid, cudaStream_t stream) {
  auto* kernel = attend_kernel<kLse>;
  static std::atomic<uint64_t> attr_done{0};
  int rc;
  if ((rc = ensure_smem_attr(kernel, kSmemBytes, attr_done)) != GQA_OK) return rc;
  static std::atomic<int> regs_ok{0};  // the register split assumes the compiled count
  if (regs_ok.load(std::memory_order_acquire) == 0) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess) return GQA_ERR_CUDA;
    regs_ok.store(fa.numRegs == kRegsLaunch ? 1 : -1, std::memory_order_release);
  }
  if (regs_ok.load(std::memory_order_acquire) < 0) return GQA_ERR_UNSUPPORTED;
  kernel<<<grid, kThreads, kSmemBytes, stream>>>(q, q_few, k, v, p);
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
  if (G > 128 || B > kMaxB || capacity > (1LL << 30) || pool_rows > 0x7FFFFFFFLL) return GQA_ERR_UNSUPPORTED;
  // K/V tiles over all units: counted in 32 bits
  const long long units = (static_cast<long long>(T) + 2 * (128 / G) - 1) / (2 * (128 / G)) + std::min(B, T);
  if (static_cast<double>(units) * Hkv * (capacity / kBN + 1 + kExtraMany) >= 2147483648.0) return GQA_ERR_UNSUPPORTED;
  // a TMA dimension needs a stride: heads or tokens that share one row are the caller's to expand
  if ((T > 1 && q_token_stride == 0) || (Hq > 1 && q_head_stride == 0)) return GQA_ERR_UNSUPPORTED;
  const Layout w = layout_of(T, G);
  if (!workspace || workspace_bytes < w.bytes) return GQA_ERR_WORKSPACE;

  Params p;
  p.batch = {block_table, q_start, lens, B, T, Hkv, static_cast<int>(capacity), max_pages_per_seq, page_size, num_pages,
             ragged::whole_log2(page_size)};
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
  p.tu = 2 * p.tpt;
  p.few = kBlockRows / G;

  CUtensorMap tmQ, tmQfew, tmK, tmV;
  int rc;
  const long long ht = Hq > 1 ? q_head_stride : kD, tt = T > 1 ? q_token_stride : static_cast<long long>(Hq) * kD;
  const long long qd[4] = {kD, Hq, T, 1}, qs[3] = {ht * 2, tt * 2, tt * 2};
  const int qb[4] = {64, G, p.tpt, 1}, qf[4] = {64, G, std::max(p.few, 1), 1};
  if ((rc = make_tmap_4d(&tmQ, q, 2, qd, qs, qb)) != GQA_OK) return rc;
  if ((rc = make_tmap_4d(&tmQfew, q, 2, qd, qs, qf)) != GQA_OK) return rc;
  if ((rc = make_tmap_3d_bf16(&tmK, kpages, kD, pool_rows, 1, 64, p.box, 1)) != GQA_OK) return rc;
  if ((rc = make_tmap_3d_bf16(&tmV, vpages, kD, pool_rows, 1, 64, p.box, 1)) != GQA_OK) return rc;

  int dev = 0, sms = kMaxCtas;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int grid = std::min(sms, kMaxCtas);
  rc = lse ? launch<true>(tmQ, tmQfew, tmK, tmV, p, grid, stream) : launch<false>(tmQ, tmQfew, tmK, tmV, p, grid, stream);
  if (rc != GQA_OK) return rc;
  // The merge starts while the first kernel drains and waits for it on the device.
  const int longest = max_q_len > 0 ? std::min(max_q_len, T) : T;  // a grid for so many rows; any number is merged
  const int rows = static_cast<int>(std::min(256LL, (static_cast<long long>(longest) * G + 31) / 32 * 32));
  return launch_after(merge_kernel, dim3(grid, std::max(1, rows / 32 * 16 / (kMergeThreads / 32))), kMergeThreads, stream,
                      p);
}
