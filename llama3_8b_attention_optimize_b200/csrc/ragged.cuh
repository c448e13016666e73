// ragged.cuh -- how the kernels over a ragged batch and a paged cache split their work.
//
// Every (sequence, kv head) has units, and a unit has steps (for attention: blocks of
// query tokens and K/V tiles; for the weight sums: blocks of slots and query tiles).  All steps of
// all units form one line, sequence by sequence, head by head, unit by unit; CTA c of N takes
// an equal part of its W steps.  A unit that lies across a cut is
// finished by a merge kernel from the parts that its CTAs leave: the first part in slot
// 2c + 1 of the CTA where the unit begins, the others in slot 2c of theirs.  So the SMs
// finish together whatever the lengths, nothing is planned on the host, and two
// slots a CTA are enough.
//
// A Line gives, for a sequence: has(s), whether it has units; units(s); count(s, u) steps of
// unit u; ends(s, u), whether u is the last; and before(s, k), the steps of the first k units in
// closed form, with line.extra steps for each unit: what beginning and ending one costs.  They lie
// in front of the unit's own and hold no work.  All steps together are fewer than 2^31 (the host's
// bound).  There may be two lines with a step cost each:
// the CTAs are dealt out in proportion to what the lines cost, and a sequence has units in
// one of them.
#pragma once

#include <cstdint>

#include "common.cuh"

namespace gqa {
namespace ragged {

constexpr int kMaxCtas = 148;  // workspace slots are sized for so many
constexpr int kMaxB = 8192;    // sequences (prefix of their steps in shared memory)

struct Batch {
  const int32_t *table, *q_start, *lens;
  int B, T, Hkv, capacity, max_pages, page_size, num_pages;
  int page_shift;  // log2(page_size) where that is whole, else -1
  __device__ __forceinline__ int page_of(int slot) const { return page_shift >= 0 ? slot >> page_shift : slot / page_size; }
};

struct Seq {
  int a, n, L;  // first token, tokens, slots
};

// Sequence b with what the device holds brought into range (the plan reports it).
__device__ __forceinline__ Seq seq_of(const Batch& p, int b) {
  Seq s;
  s.a = __ldg(p.q_start + b);
  const int z = __ldg(p.q_start + b + 1);
  s.n = (s.a < 0 || z < s.a || z > p.T) ? 0 : z - s.a;
  s.L = min(max(__ldg(p.lens + b), 0), p.capacity);
  return s;
}

// sum_{i < n} floor((a i + b) / m), by Euclid's steps on (a, m) (the reciprocity of floor sums:
// Graham, Knuth, Patashnik, Concrete Mathematics, 3.5).  The caller knows that the
// sum is below 2^31; what wraps on the way is multiplied by zero.
__device__ __forceinline__ uint32_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  uint32_t sum = 0;
#pragma unroll 1
  while (n > 0) {
    const uint32_t qa = a / m, qb = b / m;
    sum += qa * (n * (n - 1) / 2) + qb * n;
    a -= qa * m;
    b -= qb * m;
    const uint32_t top = a * n + b;
    if (top < m) break;
    n = top / m;  // count lattice points the other way round
    b = top - n * m;
    const uint32_t x = m;
    m = a;
    a = x;
  }
  return sum;
}

struct Walk {
  int b, h, u, k, left;  // place on the line, and the steps left to this CTA
  int line;
  int turn;              // for the kernel's own use
  Seq s;                 // sequence b
};

struct Part {
  Seq s;
  int b, h, u, k0, k1, count;  // steps [k0, k1) of the unit's count
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == count; }
};

// The CTA's next part of a unit; false when its steps are done.
template <class Line>
__device__ __forceinline__ bool next_part(const Batch& p, const Line& line, Walk& w, Part& x) {
  for (;;) {
    if (w.left <= 0) return false;
    x.s = w.s;
    x.b = w.b;
    x.h = w.h;
    x.u = w.u;
    x.count = line.count(x.s, w.u);
    const int end = min(x.count + line.extra, w.k + w.left);
    w.left -= end - w.k;
    x.k0 = max(0, w.k - line.extra);
    x.k1 = end - line.extra;
    w.k = 0;
    if (line.ends(x.s, w.u++)) {
      w.u = 0;
      if (++w.h == p.Hkv) {
        w.h = 0;
        do {  // the next sequence of this line, read once
          if (++w.b >= p.B) {
            w.left = 0;
            break;
          }
          w.s = seq_of(p, w.b);
        } while (!line.has(w.s));
      }
    }
    if (x.k1 > x.k0) return true;  // else the cut lies in the extra steps: all work is the next CTA's
  }
}

struct Desc {  // a unit split over CTAs c .. last, written by CTA c (valid = 0: none)
  int valid, b, h, u, last;
  Seq s;
};
static_assert(sizeof(Desc) == 32, "two 16-byte loads");

// By the whole block: this CTA's place on its line (`start`, shared) and the unit that it
// begins but does not finish (desc[blockIdx.x]).  `scratch`: shared, kPlanBytes.  Ends
// before a barrier that the caller gives.
constexpr int kPlanBytes = (2 * kMaxB + 64) * 4;
template <int kThreads, int kLines, class Line>
__device__ __forceinline__ void plan(const Batch& p, const Line (&lines)[kLines], const int (&cost)[kLines],
                                     uint32_t* scratch, Walk* start, Desc* desc, int site_q_start, int site_length) {
  static_assert(kLines == 1 || kLines == 2, "one line or two");
  constexpr int kWarps = kThreads / 32;
  static_assert(kWarps <= 32 && kLines * kWarps <= 64, "room for the warps' sums");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* wsum = scratch + 2 * kMaxB;  // [kLines][warps]
  // warps 0 and 1 need the totals; the others work only where there are sequences for them
  const int warps = max(2, min(kWarps, (p.B + 31) / 32));
  // ---- steps in front of each sequence, per line: scratch[i * kMaxB + b]
  uint32_t total[kLines] = {};
  // A q_start out of order leaves no work at all: its sequences could share tokens, and so
  // have more steps than the host has counted.
  int disordered = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    uint32_t mine[kLines] = {}, scan[kLines] = {};
    if (warp < warps) {
      Seq s = {0, 0, 0};
      if (b < p.B) {
        s = seq_of(p, b);
        const int z = __ldg(p.q_start + b + 1);
        if (s.a < 0 || z < s.a || z > p.T) {
          disordered = 1;
          if (blockIdx.x == 0) record_input_error(site_q_start);
        }
        if (blockIdx.x == 0) {
          const int L = __ldg(p.lens + b);
          if (L < 0 || L > p.capacity) record_input_error(site_length);
        }
      }
#pragma unroll
      for (int i = 0; i < kLines; ++i) {
        mine[i] = b < p.B && lines[i].has(s) ? lines[i].before(s, lines[i].units(s)) * p.Hkv : 0u;
        scan[i] = mine[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_up_sync(0xffffffffu, scan[i], o);
          if (lane >= o) scan[i] += x;
        }
        if (lane == 31) wsum[i * kWarps + warp] = scan[i];
      }
    }
    disordered = __syncthreads_or(disordered);
    if (warp < warps) {
#pragma unroll
      for (int i = 0; i < kLines; ++i) {
        const uint32_t x = lane < warps ? wsum[i * kWarps + lane] : 0u;
        const uint32_t front = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0u);
        if (b < p.B) scratch[i * kMaxB + b] = total[i] + front + scan[i] - mine[i];
        total[i] += __reduce_add_sync(0xffffffffu, x);
      }
    }
    __syncthreads();
  }
  if (warp >= 2) return;
  if (disordered)
    for (uint32_t& x : total) x = 0;
  // ---- this CTA's line, its first CTA and number of CTAs
  const int n = static_cast<int>(gridDim.x);
  int on = 0, c0 = 0, nc = n;
  if constexpr (kLines == 2) {
    if (total[1] > 0) {
      const float w0 = static_cast<float>(total[0]) * cost[0], w1 = static_cast<float>(total[1]) * cost[1];
      const int n0 = total[0] == 0 ? 0 : min(max(static_cast<int>(n * (w0 / (w0 + w1)) + 0.5f), 1), n - 1);
      on = static_cast<int>(blockIdx.x) < n0 ? 0 : 1;
      c0 = on ? n0 : 0;
      nc = on ? n - n0 : n0;
    }
  }
  const Line line = lines[on];
  const uint32_t* prefix = scratch + on * kMaxB;
  const uint32_t W = kLines == 2 && on ? total[kLines - 1] : total[0];
  const uint32_t ctas = min(static_cast<uint32_t>(nc), W);
  const uint32_t c = blockIdx.x - c0;
  // parts: W / ctas steps, the first W % ctas of them one more
  const uint32_t q = ctas > 0 ? W / ctas : 0u, more = W - q * ctas;
  auto begin = [&](uint32_t i) -> uint32_t { return i * q + min(i, more); };
  // Warp 0 finds where the part begins, warp 1 the unit that its end cuts, both by 32-way
  // searches.
  const uint32_t x = begin(warp == 0 ? c : c + 1);
  const bool wanted = warp == 0 ? c < ctas : c + 1 < ctas;
  Walk w = {0, 0, 0, 0, 0, on, 0, {0, 0, 0}};
  if (wanted) {
    int lo = 0, hi = p.B;  // the last b with prefix[b] <= x
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const int below = __popc(__ballot_sync(0xffffffffu, at < hi && prefix[at] <= x));
      lo += (below - 1) * step;
      hi = min(hi, lo + step);
    }
    const Seq s = seq_of(p, lo);
    w.s = s;
    const int units = line.units(s);
    const uint32_t head = line.before(s, units), rem = x - prefix[lo];
    w.b = lo;
    w.h = static_cast<int>(rem / head);
    const uint32_t r = rem - w.h * head;
    int u0 = 0, u1 = units;  // the last unit with before(u) <= r
    while (u1 - u0 > 1) {
      const int step = (u1 - u0 + 31) / 32, at = u0 + lane * step;
      const int below = __popc(__ballot_sync(0xffffffffu, at < u1 && line.before(s, at) <= r));
      u0 += (below - 1) * step;
      u1 = min(u1, u0 + step);
    }
    w.u = u0;
    w.k = static_cast<int>(r - line.before(s, u0));
  }
  if (lane != 0) return;
  if (warp == 0) {
    if (wanted) w.left = static_cast<int>(begin(c + 1) - x);
    *start = w;
  } else {
    Desc d = {0, 0, 0, 0, 0, {0, 0, 0}};
    // cut behind a step with work, the first of which is this CTA's
    if (wanted && w.k > line.extra && x - w.k + line.extra >= begin(c)) {
      d.valid = 1;
      d.b = w.b;
      d.h = w.h;
      d.u = w.u;
      d.s = w.s;
      const uint32_t last = x - w.k + line.extra + line.count(w.s, w.u) - 1;  // the unit's last step, and its CTA
      d.last = c0 + static_cast<int>(last < more * (q + 1) ? last / (q + 1) : more + (last - more * (q + 1)) / q);
    }
    desc[blockIdx.x] = d;
  }
}

// One lane's share of a 128-slot tile's load: box i of the tile (box rows of one page) and
// half e of its 64-column blocks, lane = 2 i + e.
struct Boxes {
  int box, slot, half;  // rows of a box, this lane's first slot in the tile, its half
  bool loads;
  uint32_t offset;      // in the tile's shared memory
  __device__ __forceinline__ Boxes(int box_, int lane) {
    box = box_;
    slot = (lane >> 1) * box;
    half = lane & 1;
    loads = (lane >> 1) < 128 / box;
    offset = half * (128 * 64 * 2) + slot * 128;
  }
  // The page of this lane's box of the tile at slot0 (-1: it begins at `limit` or above).
  __device__ __forceinline__ int page(const Batch& p, const int32_t* table, int slot0, int limit) const {
    const int at = slot0 + slot;
    return loads && at < limit ? __ldg(table + p.page_of(at)) : -1;
  }
  // Its first row of the pool, -1 for none; a page outside the pool is reported and
  // replaced by page 0, to keep the pipeline flowing.
  __device__ __forceinline__ int row(const Batch& p, int page, int h, int slot0, int limit, int site) const {
    const int at = slot0 + slot;
    if (!loads || at >= limit) return -1;
    if (page < 0 || page >= p.num_pages) {
      record_input_error(site);
      page = 0;
    }
    return (page * p.Hkv + h) * p.page_size + at - p.page_of(at) * p.page_size;
  }
};

// log2 of a power of two, else -1.
inline int whole_log2(int x) {
  if (x <= 0 || (x & (x - 1))) return -1;
  int n = 0;
  while (x >>= 1) ++n;
  return n;
}

}  // namespace ragged
}  // namespace gqa
