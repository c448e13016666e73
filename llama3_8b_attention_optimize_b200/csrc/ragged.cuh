// ragged.cuh -- how the kernels over a ragged batch and a paged cache split their work.
//
// Every (sequence, kv head) has units, and a unit has steps (for attention: blocks of
// query tokens and K/V tiles; for the weight sums: blocks of slots and query tiles).  All steps of
// all units form one line, sequence by sequence, head by head, unit by unit; CTA c of N takes
// the steps [c W / N, (c + 1) W / N) of its W.  A unit that lies across a cut is
// finished by a merge kernel from the parts that its CTAs leave: the first part in slot
// 2c + 1 of the CTA where the unit begins, the others in slot 2c of theirs.  So the SMs
// finish together whatever the lengths, nothing is planned on the host, and two
// slots a CTA are enough.
//
// A Line gives, for a sequence: units(s), count(s, u) steps of unit u, and before(s, k), the
// steps of the first k units in closed form.
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

// sum_{i < n} floor((a i + b) / m), by Euclid's steps on (a, m); a, b >= 0, m > 0.
__device__ __forceinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
  long long sum = 0;
  while (n > 0) {
    sum += (a / m) * (n * (n - 1) / 2) + (b / m) * n;
    a %= m;
    b %= m;
    const long long top = a * n + b;
    if (top < m) break;
    n = top / m;  // count lattice points the other way round
    b = top % m;
    const long long x = m;
    m = a;
    a = x;
  }
  return sum;
}

struct Walk {
  int b, h, u, k, left;  // place on the line, and the steps left to this CTA
};

struct Part {
  Seq s;
  int b, h, u, k0, k1, count;  // steps [k0, k1) of the unit's count
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == count; }
};

// The CTA's next part of a unit; false when its steps are done.
template <class Line>
__device__ __forceinline__ bool next_part(const Batch& p, const Line& line, Walk& w, Part& x) {
  if (w.left <= 0 || w.b >= p.B) return false;
  x.s = seq_of(p, w.b);
  while (line.units(x.s) == 0) {
    if (++w.b >= p.B) return false;
    x.s = seq_of(p, w.b);
  }
  x.b = w.b;
  x.h = w.h;
  x.u = w.u;
  x.count = line.count(x.s, w.u);
  x.k0 = w.k;
  x.k1 = min(x.count, w.k + w.left);
  w.left -= x.k1 - x.k0;
  w.k = 0;
  if (++w.u >= line.units(x.s)) {
    w.u = 0;
    if (++w.h == p.Hkv) {
      w.h = 0;
      ++w.b;
    }
  }
  return true;
}

struct Desc {  // a unit split over CTAs c .. last, written by CTA c (valid = 0: none)
  int valid, b, h, u, last, pad[3];
};

// By the whole block: this CTA's place on the line (`start`, shared) and the unit that it
// begins but does not finish (desc[blockIdx.x]).  `scratch`: shared, 8 (kMaxB + 64) bytes.
// Ends before a barrier that the caller gives.
template <int kThreads, class Line>
__device__ __forceinline__ void plan(const Batch& p, const Line& line, long long* scratch, Walk* start, Desc* desc,
                                     int site_q_start, int site_length) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long* prefix = scratch;          // [B] steps in front of each sequence
  long long* wsum = scratch + kMaxB;    // [warps]
  long long carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    long long mine = 0;
    if (b < p.B) {
      const Seq s = seq_of(p, b);
      const int units = line.units(s);
      if (units > 0) mine = line.before(s, units) * p.Hkv;
      if (blockIdx.x == 0) {
        const int z = __ldg(p.q_start + b + 1), L = __ldg(p.lens + b);
        if (s.a < 0 || z < s.a || z > p.T) record_input_error(site_q_start);
        if (L < 0 || L > p.capacity) record_input_error(site_length);
      }
    }
    long long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += x;
    }
    if (lane == 31) wsum[warp] = scan;
    __syncthreads();
    long long before = carry, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += wsum[w];
      all += wsum[w];
    }
    if (b < p.B) prefix[b] = before + scan - mine;
    carry += all;
    __syncthreads();
  }
  const long long W = carry;
  const long long ctas = min(static_cast<long long>(gridDim.x), W);
  const long long c = blockIdx.x;
  auto locate = [&](long long x) -> Walk {  // the unit and step at place x < W of the line
    int lo = 0, hi = p.B;                   // the last b with prefix[b] <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid;
      else hi = mid;
    }
    const Seq s = seq_of(p, lo);
    const int units = line.units(s);
    const long long head = line.before(s, units);
    const long long rem = x - prefix[lo];
    Walk w;
    w.b = lo;
    w.h = static_cast<int>(rem / head);
    const long long r = rem - w.h * head;
    int u0 = 0, u1 = units;  // the last unit with before(u) <= r
    while (u1 - u0 > 1) {
      const int mid = (u0 + u1) >> 1;
      if (line.before(s, mid) <= r) u0 = mid;
      else u1 = mid;
    }
    w.u = u0;
    w.k = static_cast<int>(r - line.before(s, u0));
    w.left = 0;
    return w;
  };
  if (threadIdx.x == 0) {
    Walk w = {0, 0, 0, 0, 0};
    if (c < ctas) {
      const long long r0 = c * W / ctas, r1 = (c + 1) * W / ctas;
      w = locate(r0);
      w.left = static_cast<int>(r1 - r0);
    }
    *start = w;
  }
  if (threadIdx.x == 32) {
    Desc d = {0, 0, 0, 0, 0, {0, 0, 0}};
    if (c + 1 < ctas) {
      const long long r0 = c * W / ctas, r1 = (c + 1) * W / ctas;
      const Walk w = locate(r1);
      if (w.k > 0 && r1 - w.k >= r0) {
        d.valid = 1;
        d.b = w.b;
        d.h = w.h;
        d.u = w.u;
        const long long end = r1 - w.k + line.count(seq_of(p, w.b), w.u);
        d.last = static_cast<int>((end * ctas - 1) / W);  // the CTA of step end - 1
      }
    }
    desc[c] = d;
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
    return loads && at < limit ? __ldg(table + at / p.page_size) : -1;
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
    return (page * p.Hkv + h) * p.page_size + at % p.page_size;
  }
};

}  // namespace ragged
}  // namespace gqa
