// evict.cu -- cut a paged K/V cache to a budget of slots per sequence and kv head.
//
// Of the n = lens[b] slots of (b, h), left = min(n, budget) are kept: first those whose
// token position is below `sink` or among the last `recent` before next_pos[b], then
// those with the largest accumulated weight; equal ones go by the lower slot.  The i-th
// slot below `left` that is not kept takes the i-th kept slot at `left` or above, in
// ascending order: rows that can stay do, and no row is both read and written, so all
// rows move at once and in place.
//
// Kernel 1, one block per (b, h): order-preserving 32-bit keys of the weights, the
// budget-th largest by four 8-bit histogram passes, then the lists of holes and movers
// by ballots (each warp owns a contiguous run of slots, so three block barriers order
// everything).  Kernel 2 moves the rows: 512 bytes (K and V) a warp step.
#include <algorithm>

#include "common.cuh"
#include "gqa_internal.h"

namespace gqa {
namespace evict {

constexpr int kD = 128;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMoveWarps = 8;
constexpr int kRowsPerWarp = 4;
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
  int32_t *src, *dst, *count;  // workspace: [B * Hkv][budget] twice, [B * Hkv]
  int Hkv, capacity, max_pages, page_size, num_pages, budget, recent, sink, cached, max_moves;
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
  __shared__ int hist[256];
  __shared__ int counts[2][kWarps];
  __shared__ int chosen[2];
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
    if (tid == 0) p.count[bh] = 0;
    if (acc_out != acc)
      for (int i = tid; i < n; i += kThreads) acc_out[i] = acc[i];
    if (pos_out != pos)
      for (int i = tid; i < n; i += kThreads) pos_out[i] = pos[i];
    return;
  }
  uint32_t* bits = smem;                              // kept slots, [ceil(capacity / 32)]
  uint32_t* keys = smem + (p.capacity + 31) / 32;     // [capacity] when cached
  const long long recent_from = static_cast<long long>(__ldg(p.next_pos + b)) - p.recent;
  auto make_key = [&](int i) {
    const int q = pos[i];
    return key_of(acc[i], q < p.sink || q >= recent_from);
  };
  if (p.cached) {
    for (int i = tid; i < n; i += kThreads) keys[i] = make_key(i);
  }
  auto key_at = [&](int i) { return p.cached ? keys[i] : make_key(i); };

  // ---- the budget-th largest key, and how many of its equals are kept
  uint32_t prefix = 0, mask = 0;
  int need = p.budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i0 = warp * 32; i0 < n; i0 += kThreads) {
      const int i = i0 + lane;
      const uint32_t k = i < n ? key_at(i) : 0u;
      const bool in = i < n && (k & mask) == prefix;
      // one add per distinct digit of the warp: weights crowd into few exponents
      const uint32_t digit = in ? (k >> shift) & 255u : 256u;
      const uint32_t peers = __match_any_sync(0xffffffffu, digit);
      if (in && lane == __ffs(peers) - 1) atomicAdd(&hist[digit], __popc(peers));
    }
    __syncthreads();
    if (warp == 0) {  // lane l holds digits [255 - 8l - 7, 255 - 8l], largest first
      int mine[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += mine[j] = hist[255 - 8 * lane - j];
      int above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += x;
      }
      above -= sum;
      if (above < need && above + sum >= need) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (above < need && above + mine[j] >= need) {
            chosen[0] = 255 - 8 * lane - j;
            chosen[1] = need - above;
          }
          above += mine[j];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(chosen[0]) << shift;
    mask |= 255u << shift;
    need = chosen[1];
  }

  // ---- kept bits: keys above the threshold, and the first `need` equal to it
  const int run = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;  // slots of one warp
  const int r0 = min(n, warp * run), r1 = min(n, r0 + run);
  int ties = 0;
  for (int i0 = r0; i0 < r1; i0 += 32)
    ties += __popc(__ballot_sync(0xffffffffu, i0 + lane < r1 && key_at(i0 + lane) == prefix));
  if (lane == 0) counts[0][warp] = ties;
  __syncthreads();
  int rank = 0;
  for (int w = 0; w < warp; ++w) rank += counts[0][w];
  int holes = 0, movers = 0;
  for (int i0 = r0; i0 < r1; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t k = i < r1 ? key_at(i) : 0u;
    const uint32_t tied = __ballot_sync(0xffffffffu, i < r1 && k == prefix);
    const bool keep = i < r1 && (k > prefix || (k == prefix && rank + __popc(tied & ((1u << lane) - 1)) < need));
    rank += __popc(tied);
    const uint32_t kept = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) bits[i0 >> 5] = kept;
    holes += __popc(__ballot_sync(0xffffffffu, i < left && !keep && i < r1));
    movers += __popc(__ballot_sync(0xffffffffu, i >= left && keep));
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
  int32_t* src = p.src + static_cast<size_t>(bh) * p.budget;
  int32_t* dst = p.dst + static_cast<size_t>(bh) * p.budget;
  const uint32_t below = (1u << lane) - 1;
  for (int i0 = r0; i0 < r1; i0 += 32) {
    const int i = i0 + lane;
    const bool keep = (bits[i0 >> 5] >> lane) & 1u;
    const uint32_t is_hole = __ballot_sync(0xffffffffu, i < left && !keep);
    const uint32_t is_mover = __ballot_sync(0xffffffffu, i >= left && i < r1 && keep);
    if ((is_hole >> lane) & 1u) dst[hole + __popc(is_hole & below)] = i;
    if ((is_mover >> lane) & 1u) src[mover + __popc(is_mover & below)] = i;
    hole += __popc(is_hole);
    mover += __popc(is_mover);
    if (i < left && keep) {
      if (acc_out != acc) acc_out[i] = acc[i];
      if (pos_out != pos) pos_out[i] = pos[i];
    }
  }
  int total = 0;
  for (int w = 0; w < kWarps; ++w) total += counts[0][w];
  if (tid == 0) p.count[bh] = total;
  __syncthreads();  // the lists are complete
  for (int i = tid; i < total; i += kThreads) {
    const int s = src[i], d = dst[i];
    acc_out[d] = acc[s];
    pos_out[d] = pos[s];
  }
}

__global__ void __launch_bounds__(kMoveWarps * 32) move_kernel(const Params p) {
  const int bh = blockIdx.y, b = bh / p.Hkv, h = bh % p.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = p.count[bh];
  const int32_t* src = p.src + static_cast<size_t>(bh) * p.budget;
  const int32_t* dst = p.dst + static_cast<size_t>(bh) * p.budget;
  uint16_t* pool = lane < 16 ? p.kp : p.vp;
  auto row_of = [&](int slot) -> long long {
    const int page = __ldg(p.table + static_cast<long long>(b) * p.max_pages + slot / p.page_size);
    if (page < 0 || page >= p.num_pages) {
      record_input_error(SITE_BAD_PAGE);
      return -1;
    }
    return ((static_cast<long long>(page) * p.Hkv + h) * p.page_size + slot % p.page_size) * kD + (lane & 15) * 8;
  };
  for (int i0 = (blockIdx.x * kMoveWarps + warp) * kRowsPerWarp; i0 < count;
       i0 += gridDim.x * kMoveWarps * kRowsPerWarp) {
    uint4 v[kRowsPerWarp];
    long long to[kRowsPerWarp];
#pragma unroll
    for (int j = 0; j < kRowsPerWarp; ++j) {
      to[j] = -1;
      if (i0 + j < count) {
        const long long from = row_of(src[i0 + j]);
        to[j] = row_of(dst[i0 + j]);
        if (from < 0) to[j] = -1;
        if (to[j] >= 0) v[j] = *reinterpret_cast<const uint4*>(pool + from);
      }
    }
#pragma unroll
    for (int j = 0; j < kRowsPerWarp; ++j)
      if (to[j] >= 0) *reinterpret_cast<uint4*>(pool + to[j]) = v[j];
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

extern "C" size_t gqa_kv_evict_workspace_size(int B, int Hkv, int budget) {
  if (B <= 0 || Hkv <= 0 || budget <= 0) return 0;
  return static_cast<size_t>(B) * Hkv * (2 * static_cast<size_t>(budget) + 1) * sizeof(int32_t);
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
  if (!workspace || workspace_bytes < gqa_kv_evict_workspace_size(B, Hkv, budget)) return GQA_ERR_WORKSPACE;
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
  const size_t n_list = static_cast<size_t>(B) * Hkv * budget;
  p.src = static_cast<int32_t*>(workspace);
  p.dst = p.src + n_list;
  p.count = p.dst + n_list;
  p.Hkv = Hkv;
  p.capacity = static_cast<int>(capacity);
  p.max_pages = max_pages_per_seq;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.budget = budget;
  p.recent = recent;
  p.sink = sink;
  p.cached = capacity <= kCachedKeys ? 1 : 0;
  const int smem = static_cast<int>((capacity + 31) / 32 + (p.cached ? capacity : 0)) * 4;
  static std::atomic<uint64_t> attr_done{0};
  int rc;
  if ((rc = ensure_smem_attr(select_kernel, (kCachedKeys + kCachedKeys / 32) * 4, attr_done)) != GQA_OK) return rc;
  select_kernel<<<B * Hkv, kThreads, smem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return GQA_ERR_CUDA;
  // as many rows as can move at most, and no more blocks than fill the GPU a few times
  const long long moves = std::min<long long>(budget, capacity - budget);
  if (moves > 0) {
    const long long per_block = kMoveWarps * kRowsPerWarp;
    const long long want = (moves + per_block - 1) / per_block;
    const long long cap = std::max<long long>(1, 148 * 32 / (static_cast<long long>(B) * Hkv));
    move_kernel<<<dim3(static_cast<unsigned>(std::min(want, cap)), B * Hkv), kMoveWarps * 32, 0, stream>>>(p);
    if (cudaGetLastError() != cudaSuccess) return GQA_ERR_CUDA;
  }
  if (lens_out == lens) {
    shorten_kernel<<<(B + 255) / 256, 256, 0, stream>>>(lens_out, B, p.capacity, budget);
    if (cudaGetLastError() != cudaSuccess) return GQA_ERR_CUDA;
  }
  return GQA_OK;
}
