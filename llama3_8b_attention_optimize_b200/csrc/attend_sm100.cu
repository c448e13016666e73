// attend_sm100.cu -- attention of a ragged chunk of new tokens over a paged K/V cache.
//
// Sequence b brings tokens q_start[b] .. q_start[b + 1] - 1 (n of them); lens[b] counts
// its cached slots with those tokens included, so its token i sits in slot lens[b] - n + i.
//   o[t, h, :] = sum_j softmax_j(q[t, h] . K[b, h / G, j] * scale) V[b, h / G, j, :]
// over the slots j it sees (j <= its own slot when causal, else j < lens[b]), and
// lse[t, h] = ln sum_j exp(q[t, h] . K[b, h / G, j] * scale).  A row that sees no slot gives zeros and -inf.
//
// One block per (token, query head): each warp walks every fourth slot with an online softmax,
// a lane holding four of the 128 dims; the four warps' states are merged at the end.
#include "common.cuh"
#include "gqa_internal.h"

namespace gqa {
namespace attend {

constexpr int kD = 128;
constexpr int kWarps = 4;

enum : int {
  SITE_Q_START = 0x620,   // q_start not ascending or outside [0, T]
  SITE_LENGTH = 0x621,    // lens[b] outside [0, capacity]
  SITE_BAD_PAGE = 0x622,  // block-table entry outside [0, num_pages)
};

struct Params {
  const uint16_t *q, *kp, *vp;
  uint16_t* o;
  float* lse;
  const int32_t *table, *q_start, *lens;
  long long q_t, q_h, o_t, o_h;
  int B, T, Hq, Hkv, max_pages, page_size, num_pages, causal;
  float scale;
};

__global__ void __launch_bounds__(kWarps * 32) attend_kernel(const Params p) {
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][kD];
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = h / (p.Hq / p.Hkv);
  int lo = 0, hi = p.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int a = p.q_start[lo], z = p.q_start[lo + 1];
  if (a < 0 || z > p.T || t < a || t >= z) {
    if (threadIdx.x == 0 && (a < 0 || z > p.T || t < a || t < p.q_start[p.B])) record_input_error(SITE_Q_START);
    return;
  }
  const long long capacity = static_cast<long long>(p.max_pages) * p.page_size;
  int len = p.lens[lo];
  if (len < 0 || len > capacity) {
    if (threadIdx.x == 0) record_input_error(SITE_LENGTH);
    len = static_cast<int>(min(max(static_cast<long long>(len), 0ll), capacity));
  }
  const int last = p.causal ? len - z + t : len - 1;
  float q[4];
  {
    const uint2 w = *reinterpret_cast<const uint2*>(p.q + t * p.q_t + h * p.q_h + 4 * lane);
    q[0] = bf16_lo(w.x), q[1] = bf16_hi(w.x), q[2] = bf16_lo(w.y), q[3] = bf16_hi(w.y);
  }
  float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
  for (int j = warp; j <= last; j += kWarps) {
    int page = p.table[static_cast<long long>(lo) * p.max_pages + j / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      record_input_error(SITE_BAD_PAGE);
      page = 0;
    }
    const size_t row = ((static_cast<size_t>(page) * p.Hkv + hk) * p.page_size + j % p.page_size) * kD + 4 * lane;
    const uint2 k = *reinterpret_cast<const uint2*>(p.kp + row), v = *reinterpret_cast<const uint2*>(p.vp + row);
    float s = q[0] * bf16_lo(k.x) + q[1] * bf16_hi(k.x) + q[2] * bf16_lo(k.y) + q[3] * bf16_hi(k.y);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale;
    const float mn = fmaxf(m, s), f = expf(m - mn), e = expf(s - mn);
    m = mn;
    l = l * f + e;
    o[0] = o[0] * f + e * bf16_lo(v.x);
    o[1] = o[1] * f + e * bf16_hi(v.x);
    o[2] = o[2] * f + e * bf16_lo(v.y);
    o[3] = o[3] * f + e * bf16_hi(v.y);
  }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int i = 0; i < 4; ++i) so[warp][4 * lane + i] = o[i];
  __syncthreads();
  float M = -INFINITY, L = 0.0f, x = 0.0f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < kWarps; ++w) {
    const float f = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - M);
    L += sl[w] * f;
    x += so[w][threadIdx.x] * f;
  }
  p.o[t * p.o_t + h * p.o_h + threadIdx.x] = f2bf_bits(L > 0.0f ? x / L : 0.0f);
  if (p.lse && threadIdx.x == 0) p.lse[static_cast<size_t>(t) * p.Hq + h] = L > 0.0f ? M + logf(L) : -INFINITY;
}

}  // namespace attend

GQA_ERROR_FLAG_ACCESSOR(error_flag_attend)

}  // namespace gqa

using namespace gqa;

extern "C" size_t gqa_attend_chunk_workspace_size(int T, int Hq, int Hkv) {
  (void)T, (void)Hq, (void)Hkv;
  return 16;
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
  if (!workspace || workspace_bytes < gqa_attend_chunk_workspace_size(T, Hq, Hkv)) return GQA_ERR_WORKSPACE;
  Params p;
  p.q = static_cast<const uint16_t*>(q);
  p.kp = static_cast<const uint16_t*>(kpages);
  p.vp = static_cast<const uint16_t*>(vpages);
  p.o = static_cast<uint16_t*>(o);
  p.lse = lse;
  p.table = block_table, p.q_start = q_start, p.lens = lens;
  p.q_t = q_token_stride, p.q_h = q_head_stride, p.o_t = o_token_stride, p.o_h = o_head_stride;
  p.B = B, p.T = T, p.Hq = Hq, p.Hkv = Hkv, p.max_pages = max_pages_per_seq, p.page_size = page_size;
  p.num_pages = num_pages, p.causal = (flags & GQA_FLAG_CAUSAL) != 0, p.scale = scale;
  attend_kernel<<<dim3(T, Hq), kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}
