// weights_sm100.cu -- accumulated attention weight of every cached slot.
//
// For the chunk of attend_sm100.cu (same q_start, lens, slots and mask) and its lse,
//   acc_out[b, h, j] = (j < lens[b] - n ? acc[b, h, j] : 0)
//                      + sum over the group's heads and the chunk's tokens that see slot j
//                        of exp(q . K[b, h, j] * scale - lse),
// for j < lens[b]; entries at lens[b] and above are left alone.  Slots that the chunk itself wrote start
// from zero.  Each sum is taken by one thread in token order: no atomics, the same bits on every run.
//
// One thread per slot, K's row in registers, a query row at a time in shared memory.
#include "common.cuh"
#include "gqa_internal.h"

namespace gqa {
namespace weights {

constexpr int kD = 128;

enum : int {
  SITE_Q_START = 0x630,   // q_start not ascending or outside [0, T]
  SITE_LENGTH = 0x631,    // lens[b] outside [0, capacity]
  SITE_BAD_PAGE = 0x632,  // block-table entry outside [0, num_pages)
};

struct Params {
  const uint16_t *q, *kp;
  const float *lse, *acc;
  float* acc_out;
  const int32_t *table, *q_start, *lens;
  long long q_t, q_h;
  int B, T, Hq, Hkv, max_pages, page_size, num_pages, causal;
  float scale;
};

__global__ void __launch_bounds__(128) weights_kernel(const Params p) {
  __shared__ float sq[kD];
  const int hk = blockIdx.y % p.Hkv, b = blockIdx.y / p.Hkv, G = p.Hq / p.Hkv;
  const long long capacity = static_cast<long long>(p.max_pages) * p.page_size;
  int len = p.lens[b], a = p.q_start[b], z = p.q_start[b + 1];
  if (len < 0 || len > capacity) {
    if (threadIdx.x == 0) record_input_error(SITE_LENGTH);
    len = static_cast<int>(min(max(static_cast<long long>(len), 0ll), capacity));
  }
  if (a < 0 || z < a || z > p.T) {
    if (threadIdx.x == 0) record_input_error(SITE_Q_START);
    a = z = 0;
  }
  if (static_cast<int>(blockIdx.x) * 128 >= len) return;  // the whole block
  const int j = blockIdx.x * 128 + threadIdx.x;
  uint32_t k[64];
  if (j < len) {
    int page = p.table[static_cast<long long>(b) * p.max_pages + j / p.page_size];
    if (page < 0 || page >= p.num_pages) {
      record_input_error(SITE_BAD_PAGE);
      page = 0;
    }
    const uint4* row = reinterpret_cast<const uint4*>(
        p.kp + ((static_cast<size_t>(page) * p.Hkv + hk) * p.page_size + j % p.page_size) * kD);
#pragma unroll
    for (int i = 0; i < 16; ++i) *reinterpret_cast<uint4*>(k + 4 * i) = row[i];
  }
  float sum = 0.0f;
  for (int t = a; t < z; ++t) {
    const int last = p.causal ? len - z + t : len - 1;
    for (int h = hk * G; h < (hk + 1) * G; ++h) {
      __syncthreads();
      sq[threadIdx.x] = bf2f_bits(p.q[t * p.q_t + h * p.q_h + threadIdx.x]);
      __syncthreads();
      const float lse = p.lse[static_cast<size_t>(t) * p.Hq + h];
      if (j < len && j <= last && lse != -INFINITY) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          s = fmaf(sq[2 * i], bf16_lo(k[i]), s);
          s = fmaf(sq[2 * i + 1], bf16_hi(k[i]), s);
        }
        sum += expf(fmaf(s, p.scale, -lse));
      }
    }
  }
  if (j < len) {
    const size_t at = static_cast<size_t>(blockIdx.y) * capacity + j;
    p.acc_out[at] = (j < len - (z - a) ? p.acc[at] : 0.0f) + sum;
  }
}

}  // namespace weights

GQA_ERROR_FLAG_ACCESSOR(error_flag_weights)

}  // namespace gqa

using namespace gqa;

extern "C" int gqa_attn_weight_sums_f32(const void* q, long long q_token_stride, long long q_head_stride,
                                        const void* kpages, const int32_t* block_table, int max_pages_per_seq,
                                        int page_size, int num_pages, const int32_t* q_start, const int32_t* lens,
                                        const float* lse, const float* acc, float* acc_out, int B, int T, int Hq,
                                        int Hkv, int head_dim, int max_q_len, float scale, int flags,
                                        gqa_stream_t stream) {
  using namespace weights;
  if (B <= 0 || T < 0 || Hq <= 0 || Hkv <= 0 || max_pages_per_seq <= 0 || page_size <= 0 || num_pages <= 0)
    return GQA_ERR_INVALID_ARGUMENT;
  if (head_dim != kD || Hq % Hkv || page_size % 16) return GQA_ERR_UNSUPPORTED;
  if (!(scale > 0.0f) || !(scale < 1e30f) || (flags & ~GQA_FLAG_CAUSAL) || max_q_len < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (q_token_stride < 0 || q_head_stride < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (!kpages || !block_table || !q_start || !lens || !acc || !acc_out || (T > 0 && (!q || !lse)))
    return GQA_ERR_INVALID_ARGUMENT;
  auto odd = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 4 != 0; };
  if (!aligned16(q) || !aligned16(kpages) || odd(block_table) || odd(q_start) || odd(lens) || odd(lse) || odd(acc) ||
      odd(acc_out))
    return GQA_ERR_MISALIGNED;
  if ((T > 1 && q_token_stride % 8) || (Hq > 1 && q_head_stride % 8)) return GQA_ERR_MISALIGNED;
  const long long capacity = static_cast<long long>(max_pages_per_seq) * page_size;
  Params p;
  p.q = static_cast<const uint16_t*>(q);
  p.kp = static_cast<const uint16_t*>(kpages);
  p.lse = lse, p.acc = acc, p.acc_out = acc_out;
  p.table = block_table, p.q_start = q_start, p.lens = lens;
  p.q_t = q_token_stride, p.q_h = q_head_stride;
  p.B = B, p.T = T, p.Hq = Hq, p.Hkv = Hkv, p.max_pages = max_pages_per_seq, p.page_size = page_size;
  p.num_pages = num_pages, p.causal = (flags & GQA_FLAG_CAUSAL) != 0, p.scale = scale;
  weights_kernel<<<dim3(static_cast<unsigned>((capacity + 127) / 128), B * Hkv), 128, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}
