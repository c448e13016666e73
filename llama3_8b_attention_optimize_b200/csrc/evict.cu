// evict.cu -- cut a paged K/V cache to a budget of slots per sequence and kv head.
//
// Of the n = lens[b] slots of (b, h), left = min(n, budget) are kept: first those whose
// token position is below `sink` or among the last `recent` before next_pos[b], then
// those with the largest accumulated weight; equal ones go by the lower slot.  The i-th
// slot below `left` that is not kept takes the i-th kept slot at `left` or above, in
// ascending order: rows that can stay do, and no row is both read and written, so all
// rows move at once and in place.
//
// Kernel 1, one block per (b, h): order-preserving 32-bit keys of the weights in shared
// memory, the budget-th largest by three histogram passes (11, 11 and 10 bits), then the
// lists of holes and movers by ballots (each warp owns a contiguous run of slots, so three
// block barriers order everything).  Bound by latencies: loads are issued eight at a time.
// Kernel 2 moves the rows, bound by memory: 16 rows a warp step, their slots turned into
// addresses by one lane each, K by lanes 0-15 and V by 16-31, 16 bytes a lane.
//
// Measured (8 kv heads, both launches, replayed from a graph): 16 sequences of 20000..32768
// slots cut to 16384, 806 MB in 165 us, 4.9 TB/s (the selection about 32 us of it; the moved
// weights and positions copied by kernel 2 instead: 3 % longer); 4 of 1100..2048 cut to 1024,
// 13.2 us, latency; one slot a sequence, as a cache at its budget is cut: 16 of 16385 25 us, 64 of
// 4097 43 us: the selection, and a launch for a row a head.
#include <algorithm>

#include "common.cuh"
#include "gqa_internal.h"
#include "ragged.cuh"

namespace gqa {
namespace evict {

constexpr int kD = 128;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMoveWarps = 8;
constexpr int kRowsPerWarp = 16;           // of a step, in two batches
constexpr int kBins = 2048;
static_assert(2 * kThreads == kBins, "two bins a thread");
constexpr int kUnroll = 8;                  // loads in flight a thread
constexpr int kCachedKeys = 48 * 1024;      // keys of up to so many slots stay in shared memory
constexpr int kMaxCapacity = 1 << 20;       // slots of a sequence (kept bits in shared memory)

enum : int {
  SITE_LENGTH = 0x610,    // lens[b] outside [0, capacity]
  SITE_BAD_PAGE = 0x611,  // block-table entry outside [0, num_pages)
};

struct Params {
  uint16_t *kp, *vp;
  const int32_t *table, *lens, *next_pos, *slot_pos;
  const float* acc;
  float* acc_out;
  int32_t *pos_out, *lens_out;
  int32_t *src, *dst, *count;  // workspace: [B * Hkv][rows] twice, [B * Hkv]; none where rows is 0
  int Hkv, capacity, max_pages, page_size, num_pages, budget, recent, sink, cached, page_shift;
  int rows;  // rows of one (b, h) that can move at most
};

// Order-preserving key: larger weight, larger key; NaN below every number, -0 equals +0,
// a held slot above all.
__device__ __forceinline__ uint32_t key_of(float w, bool held) {
  if (held) return 0xFFFFFFFFu;
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kThreads, 1) select_kernel(const Params p) {
  extern __shared__ uint32_t smem[];
  __shared__ int hist[kBins];
  __shared__ int counts[2][kWarps];
  __shared__ int chosen[3];
  const int bh = blockIdx.x, b = bh / p.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int n = __ldg(p.lens + b);
  if (n < 0 || n > p.capacity) {
    if (tid == 0) record_input_error(SITE_LENGTH);
    n = min(max(n, 0), p.capacity);
  }
  const int left = min(n, p.budget);
  const size_t base = static_cast<size_t>(bh) * p.capacity;
  const float* acc = p.acc + base;
  const int32_t* pos = p.slot_pos + base;
  float* acc_out = p.acc_out + base;
  int32_t* pos_out = p.pos_out + base;
  if (bh % p.Hkv == 0 && tid == 0 && p.lens_out != p.lens) p.lens_out[b] = left;
  if (n <= p.budget) {
    if (tid == 0 && p.rows > 0) p.count[bh] = 0;
    if (acc_out != acc)
      for (int i = tid; i < n; i += kThreads) acc_out[i] = acc[i];
    if (pos_out != pos)
      for (int i = tid; i < n; i += kThreads) pos_out[i] = pos[i];
    return;
  }
  uint32_t* bits = smem;                           // kept slots, [ceil(capacity / 32)]
  uint32_t* keys = smem + (p.capacity + 31) / 32;  // [capacity] when cached
  const long long recent_from = static_cast<long long>(__ldg(p.next_pos + b)) - p.recent;
  auto make_key = [&](float w, int q) { return key_of(w, q < p.sink || q >= recent_from); };
  if (p.cached) {
    for (int i0 = tid; i0 < n; i0 += kUnroll * kThreads) {
      float w[kUnroll];
      int q[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int i = i0 + k * kThreads;
        w[k] = i < n ? acc[i] : 0.0f;
        q[k] = i < n ? pos[i] : 0;
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (i0 + k * kThreads < n) keys[i0 + k * kThreads] = make_key(w[k], q[k]);
    }
  }
  auto key_at = [&](int i) { return p.cached ? keys[i] : make_key(acc[i], pos[i]); };

  // ---- the budget-th largest key, and how many of its equals are kept
  uint32_t prefix = 0, mask = 0;
  int need = p.budget;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t k = key_at(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1);
    }
    __syncthreads();
    // thread t holds bins 2047 - 2t and 2046 - 2t, largest first: a scan over the block
    const int a = hist[kBins - 1 - 2 * tid], c = hist[kBins - 2 - 2 * tid];
    int above = a + c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, above, o);
      if (lane >= o) above += x;
    }
    if (lane == 31) counts[0][warp] = above;
    __syncthreads();
    above += __reduce_add_sync(0xffffffffu, lane < warp ? counts[0][lane] : 0) - a - c;
    if (above < need && above + a + c >= need) {
      const bool first = above + a >= need;
      chosen[0] = kBins - 1 - 2 * tid - (first ? 0 : 1);
      chosen[1] = need - above - (first ? 0 : a);
      chosen[2] = first ? a : c;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(chosen[0]) << shift;
    mask |= digits << shift;
    need = chosen[1];
  }

  // ---- kept bits: keys above the threshold, and the first `need` equal to it.  A word of
  // 32 slots at a time; of the word at i0, `low` marks the slots below `left`.
  const int run = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;  // slots of one warp
  const int r0 = min(n, warp * run), r1 = min(n, r0 + run);
  auto low = [&](int i0) -> uint32_t { return left - i0 >= 32 ? 0xFFFFFFFFu : left > i0 ? (1u << (left - i0)) - 1 : 0u; };
  int holes = 0, movers = 0;
  auto note = [&](int i0, uint32_t kept) {
    if (lane == 0) bits[i0 >> 5] = kept;
    holes += __popc(~kept & low(i0));
    movers += __popc(kept & ~low(i0));
  };
  if (need == chosen[2]) {  // all that equal the threshold: no order among them
#pragma unroll 4
    for (int i0 = r0; i0 < r1; i0 += 32)
      note(i0, __ballot_sync(0xffffffffu, i0 + lane < r1 && key_at(i0 + lane) >= prefix));
  } else {
    int ties = 0;
    for (int i0 = r0; i0 < r1; i0 += 32)
      ties += __popc(__ballot_sync(0xffffffffu, i0 + lane < r1 && key_at(i0 + lane) == prefix));
    if (lane == 0) counts[0][warp] = ties;
    __syncthreads();
    int rank = 0;
    for (int w = 0; w < warp; ++w) rank += counts[0][w];
    for (int i0 = r0; i0 < r1; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t k = i < r1 ? key_at(i) : 0u;
      const uint32_t tied = __ballot_sync(0xffffffffu, i < r1 && k == prefix);
      const bool keep = i < r1 && (k > prefix || (k == prefix && rank + __popc(tied & ((1u << lane) - 1)) < need));
      rank += __popc(tied);
      note(i0, __ballot_sync(0xffffffffu, keep));
    }
  }
  __syncthreads();  // counts[0] has been read
  if (lane == 0) {
    counts[0][warp] = holes;
    counts[1][warp] = movers;
  }
  __syncthreads();
  int hole = 0, mover = 0;
  for (int w = 0; w < warp; ++w) {
    hole += counts[0][w];
    mover += counts[1][w];
  }
  int32_t* src = p.src + static_cast<size_t>(bh) * p.rows;
  int32_t* dst = p.dst + static_cast<size_t>(bh) * p.rows;
  const uint32_t below = (1u << lane) - 1;
  for (int i0 = r0; i0 < r1; i0 += 32) {
    const uint32_t kept = bits[i0 >> 5], is_hole = ~kept & low(i0), is_mover = kept & ~low(i0);
    if ((is_hole >> lane) & 1u) dst[hole + __popc(is_hole & below)] = i0 + lane;
    if ((is_mover >> lane) & 1u) src[mover + __popc(is_mover & below)] = i0 + lane;
    hole += __popc(is_hole);
    mover += __popc(is_mover);
  }
  int total = 0;
  for (int w = 0; w < kWarps; ++w) total += counts[0][w];
  if (tid == 0) p.count[bh] = total;
  // what stays keeps its place
  if (acc_out != acc || pos_out != pos) {
    for (int i0 = tid; i0 < left; i0 += kUnroll * kThreads) {
      float w[kUnroll];
      int q[kUnroll];
      bool keep[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int i = i0 + k * kThreads;
        keep[k] = i < left && ((bits[i >> 5] >> (i & 31)) & 1u);
        w[k] = keep[k] ? acc[i] : 0.0f;
        q[k] = keep[k] ? pos[i] : 0;
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int i = i0 + k * kThreads;
        if (keep[k] && acc_out != acc) acc_out[i] = w[k];
        if (keep[k] && pos_out != pos) pos_out[i] = q[k];
      }
    }
  }
  __syncthreads();  // the lists are complete
  for (int i0 = tid; i0 < total; i0 += kUnroll * kThreads) {
    int from[kUnroll], to[kUnroll], q[kUnroll];
    float w[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int i = i0 + k * kThreads;
      from[k] = i < total ? src[i] : -1;
      to[k] = i < total ? dst[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      w[k] = from[k] >= 0 ? acc[from[k]] : 0.0f;
      q[k] = from[k] >= 0 ? pos[from[k]] : 0;
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (from[k] >= 0) {
        acc_out[to[k]] = w[k];
        pos_out[to[k]] = q[k];
      }
  }
}

__global__ void __launch_bounds__(kMoveWarps * 32) move_kernel(const Params p) {
  cudaGridDependencySynchronize();  // launched while the selection drains
  const int bh = blockIdx.y, b = bh / p.Hkv, h = bh % p.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = p.count[bh];
  const int32_t* src = p.src + static_cast<size_t>(bh) * p.rows;
  const int32_t* dst = p.dst + static_cast<size_t>(bh) * p.rows;
  uint16_t* pool = (lane < 16 ? p.kp : p.vp) + (lane & 15) * 8;
  const int32_t* table = p.table + static_cast<long long>(b) * p.max_pages;
  const int32_t* list = lane < 16 ? src : dst;
  for (int i0 = (blockIdx.x * kMoveWarps + warp) * kRowsPerWarp; i0 < count;
       i0 += gridDim.x * kMoveWarps * kRowsPerWarp) {
    // lane j: the pool row that move j reads, lane 16 + j: the one it writes; -1 for none
    long long row = -1;
    if (i0 + (lane & 15) < count) {
      const int slot = list[i0 + (lane & 15)];
      const int lp = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
      const int page = __ldg(table + lp);
      if (page < 0 || page >= p.num_pages)
        record_input_error(SITE_BAD_PAGE);
      else
        row = (static_cast<long long>(page) * p.Hkv + h) * p.page_size + (slot - lp * p.page_size);
    }
    if (__shfl_xor_sync(0xffffffffu, row < 0 ? 1 : 0, 16)) row = -1;  // both ends or none
#pragma unroll
    for (int j0 = 0; j0 < kRowsPerWarp; j0 += 8) {
      uint4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const long long from = __shfl_sync(0xffffffffu, row, j0 + j);
        if (from >= 0) v[j] = *reinterpret_cast<const uint4*>(pool + from * kD);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const long long to = __shfl_sync(0xffffffffu, row, 16 + j0 + j);
        if (to >= 0) *reinterpret_cast<uint4*>(pool + to * kD) = v[j];
      }
    }
  }
}

// After every block has read lens: lens_out may be lens.
__global__ void shorten_kernel(int32_t* lens, int B, int capacity, int budget) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < B) lens[b] = min(min(max(lens[b], 0), capacity), budget);
}

}  // namespace evict

GQA_ERROR_FLAG_ACCESSOR(error_flag_evict)

}  // namespace gqa

extern "C" size_t gqa_kv_evict_workspace_size(int B, int Hkv, int rows) {
  if (B <= 0 || Hkv <= 0 || rows <= 0) return 0;
  return static_cast<size_t>(B) * Hkv * (2 * static_cast<size_t>(rows) + 1) * sizeof(int32_t);
}

extern "C" int gqa_kv_evict_bf16(void* kpages, void* vpages, const int32_t* block_table, int max_pages_per_seq,
                                 int page_size, int num_pages, const int32_t* lens, int32_t* lens_out,
                                 const float* acc, float* acc_out, const int32_t* slot_pos, int32_t* slot_pos_out,
                                 const int32_t* next_pos, void* workspace, size_t workspace_bytes, int B, int Hkv,
                                 int head_dim, int budget, int recent, int sink, gqa_stream_t stream) {
  using namespace gqa;
  using namespace gqa::evict;
  if (!kpages || !vpages || !block_table || !lens || !lens_out || !acc || !acc_out || !slot_pos || !slot_pos_out ||
      !next_pos)
    return GQA_ERR_INVALID_ARGUMENT;
  if (B <= 0 || Hkv <= 0 || max_pages_per_seq <= 0 || page_size <= 0 || num_pages <= 0) return GQA_ERR_INVALID_ARGUMENT;
  if (head_dim != kD) return GQA_ERR_UNSUPPORTED;
  if (budget <= 0 || recent < 0 || sink < 0 || static_cast<long long>(recent) + sink > budget)
    return GQA_ERR_INVALID_ARGUMENT;
  const long long capacity = static_cast<long long>(max_pages_per_seq) * page_size;
  if (capacity > kMaxCapacity || static_cast<long long>(B) * Hkv > 65535) return GQA_ERR_UNSUPPORTED;
  if (!aligned16(kpages) || !aligned16(vpages)) return GQA_ERR_MISALIGNED;
  for (const void* ptr : {static_cast<const void*>(block_table), static_cast<const void*>(lens),
                          static_cast<const void*>(lens_out), static_cast<const void*>(acc),
                          static_cast<const void*>(acc_out), static_cast<const void*>(slot_pos),
                          static_cast<const void*>(slot_pos_out), static_cast<const void*>(next_pos),
                          static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(ptr) % 4) return GQA_ERR_MISALIGNED;
  // kept slots at `budget` or above move into holes below it
  const int rows = static_cast<int>(std::min<long long>(budget, std::max(0LL, capacity - budget)));
  if (rows > 0 && (!workspace || workspace_bytes < gqa_kv_evict_workspace_size(B, Hkv, rows))) return GQA_ERR_WORKSPACE;
  Params p;
  p.kp = static_cast<uint16_t*>(kpages);
  p.vp = static_cast<uint16_t*>(vpages);
  p.table = block_table;
  p.lens = lens;
  p.next_pos = next_pos;
  p.slot_pos = slot_pos;
  p.acc = acc;
  p.acc_out = acc_out;
  p.pos_out = slot_pos_out;
  p.lens_out = lens_out;
  const size_t n_list = static_cast<size_t>(B) * Hkv * rows;
  p.src = static_cast<int32_t*>(workspace);
  p.dst = p.src + n_list;
  p.count = p.dst + n_list;
  p.Hkv = Hkv;
  p.capacity = static_cast<int>(capacity);
  p.max_pages = max_pages_per_seq;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.budget = budget;
  p.rows = rows;
  p.recent = recent;
  p.sink = sink;
  p.cached = capacity <= kCachedKeys ? 1 : 0;
  p.page_shift = ragged::whole_log2(page_size);
  const int smem = static_cast<int>((capacity + 31) / 32 + (p.cached ? capacity : 0)) * 4;
  static std::atomic<uint64_t> attr_done{0};
  int rc;
  if ((rc = ensure_smem_attr(select_kernel, (kCachedKeys + kCachedKeys / 32) * 4, attr_done)) != GQA_OK) return rc;
  select_kernel<<<B * Hkv, kThreads, smem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GQA_ERR_CUDA;
  // no more blocks than fill the GPU a few times
  if (rows > 0) {
    const long long per_block = kMoveWarps * kRowsPerWarp;
    const long long want = (rows + per_block - 1) / per_block;
    const long long cap = std::max<long long>(1, 148 * 16 / (static_cast<long long>(B) * Hkv));
    if ((rc = launch_after(move_kernel, dim3(static_cast<unsigned>(std::min(want, cap)), B * Hkv), kMoveWarps * 32, stream,
                           p)) != GQA_OK)
      return rc;
  }
  if (lens_out == lens) {
    shorten_kernel<<<(B + 255) / 256, 256, 0, stream>>>(lens_out, B, p.capacity, budget);
    if (cudaGetLastError() != cudaSuccess) return GQA_ERR_CUDA;
  }
  return GQA_OK;
}
