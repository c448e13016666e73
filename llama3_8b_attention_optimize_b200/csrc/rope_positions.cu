// rope_positions.cu -- rotary positions for ragged batches, and the paged append that
// rotates on the way in.
//
// With theta_{p,i} = p * inv_freq[i] (i < rot/2) and a pair (a, b) of a head's values,
//   a' = (a cos - b sin) * m,  b' = (b cos + a sin) * m,
// where the pair is (x[i], x[i + rot/2]) in the half layout and (x[2i], x[2i + 1]) in the
// interleaved one; values at rot and above pass through.  The tables hold m cos and m sin
// in 32 bits, computed from 64-bit angles: a 32-bit angle at position 131071 is already
// 0.004 rad off, more than the rounding of a bf16 result.  With the inverse flag sin changes its
// sign: for m = 1 that is the inverse rotation, and for any m the gradient, since the
// rotation matrix is orthogonal up to m.
//
// Products and sums are 32-bit, rounded once to the output type.
//
// Both kernels move each value once, 16 bytes a thread, and are bound by memory.  Measured
// (replayed from a graph): 8191 x 40 rows of 128 fp32, half of each rotated, 338 MB in 54 us,
// 6.2 TB/s; as many rows in bf16, all of each rotated, 172 MB in 46 us (half layout) and 38 us
// (interleaved); the append of 8192 tokens with 32 + 2 x 8 heads into pages of 16, 205 MB in
// 39.6 us, 5.2 TB/s; 4 x 32 rows 2.1 us and an append of 64 tokens 3.6 us, latency.
#include <algorithm>

#include "common.cuh"
#include "gqa_internal.h"

namespace gqa {
namespace ropepos {

enum : int {
  SITE_POSITION = 0x604,  // position outside the table
  SITE_Q_START = 0x605,   // q_start not ascending or outside [0, T]
  SITE_SLOT = 0x606,      // slot outside the cache
  SITE_BAD_PAGE = 0x607,  // block-table entry outside [0, num_pages)
};

__global__ void __launch_bounds__(256) table_kernel(const double* inv_freq, float* cos_t, float* sin_t, long long n,
                                                    int half, int pos0, double mscale) {
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  double s, c;
  sincos((static_cast<double>(pos0) + static_cast<double>(i / half)) * inv_freq[i % half], &s, &c);
  cos_t[i] = static_cast<float>(c * mscale);
  sin_t[i] = static_cast<float>(s * mscale);
}

// E values of type T, read and written as one vector (16 bytes) or singly; kept as they
// were read until they are used.
template <typename T, int E>
struct Vec;
template <>
struct Vec<uint16_t, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16_lo(w[i]);
      f[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Vec<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[4]) {
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[4]) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Vec<uint16_t, 1> {
  using Raw = uint16_t;
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[1]) { f[0] = bf2f_bits(v); }
  static __device__ __forceinline__ Raw pack(const float (&f)[1]) { return f2bf_bits(f[0]); }
};
template <>
struct Vec<float, 1> {
  using Raw = float;
  static __device__ __forceinline__ void unpack(const Raw& v, float (&f)[1]) { f[0] = v; }
  static __device__ __forceinline__ Raw pack(const float (&f)[1]) { return f[0]; }
};
template <typename T, int E>
__device__ __forceinline__ typename Vec<T, E>::Raw ld(const T* p) {
  return *reinterpret_cast<const typename Vec<T, E>::Raw*>(p);
}
template <typename T, int E>
__device__ __forceinline__ void st(T* p, const typename Vec<T, E>::Raw& v) {
  *reinterpret_cast<typename Vec<T, E>::Raw*>(p) = v;
}

// A head row is cut into chunks of vectors E values long (16 bytes, or single values where
// sizes or alignment do not allow more): first the rotated ones, then those that pass
// through.  In the half layout a rotated chunk is two vectors, rot/2 apart, with E table
// entries; in the interleaved one it is a vector of E/2 pairs with E/2 entries (two single
// values where E is 1).
struct Shape {
  int half, n_pairs, n_chunks;  // rot/2, rotated chunks, all chunks
};

template <int E, bool IL>
struct Chunk {
  static constexpr bool kTwo = !IL || E == 1;   // two vectors
  static constexpr int kEntries = kTwo ? E : E / 2;
  int a, b, entry;  // vectors' offsets (b < 0: one), first table entry (-1: passes through)
  __device__ __forceinline__ Chunk(const Shape& s, int c) {
    entry = c < s.n_pairs ? c * kEntries : -1;
    if (entry < 0) {
      a = 2 * s.half + (c - s.n_pairs) * E;
      b = -1;
    } else {
      a = IL ? (E == 1 ? 2 * c : c * E) : c * E;
      b = !kTwo ? -1 : IL ? a + 1 : a + s.half;
    }
  }
};

// Table entries [i0, i0 + N) of one row.
template <int N>
__device__ __forceinline__ void ld_table(const float* row, int i0, float (&f)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(row + i0 + i));
      f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const float2 v = __ldg(reinterpret_cast<const float2*>(row + i0));
    f[0] = v.x, f[1] = v.y;
  } else {
    f[0] = __ldg(row + i0);
  }
}

// Rotate a chunk: vectors a and (where there are two) b.
template <typename T, int E, bool IL>
__device__ __forceinline__ void rotate(typename Vec<T, E>::Raw& ra, typename Vec<T, E>::Raw& rb,
                                       const float (&c)[Chunk<E, IL>::kEntries], const float (&s)[Chunk<E, IL>::kEntries]) {
  float u[E], w[E];
  Vec<T, E>::unpack(ra, u);
  if constexpr (Chunk<E, IL>::kTwo) Vec<T, E>::unpack(rb, w);
#pragma unroll
  for (int i = 0; i < Chunk<E, IL>::kEntries; ++i) {
    float& x = Chunk<E, IL>::kTwo ? u[i] : u[(2 * i) % E];
    float& y = Chunk<E, IL>::kTwo ? w[i] : u[(2 * i + 1) % E];
    const float a = x, b = y;
    x = fmaf(a, c[i], -(b * s[i]));
    y = fmaf(b, c[i], a * s[i]);
  }
  ra = Vec<T, E>::pack(u);
  if constexpr (Chunk<E, IL>::kTwo) rb = Vec<T, E>::pack(w);
}

template <typename T>
struct Params {
  const T* x;
  T* y;
  const int32_t* positions;
  const float* cos;
  const float* sin;
  long long x_t, x_h, y_t, y_h;  // strides in elements
  int T_, H, rows;
  float sign;
  Shape s;
};

// Block (chunks, heads, tokens); a thread keeps its chunk's table entries over its heads.
// Bound by memory: the first kAhead heads are on their way before the position is known.
constexpr int kAhead = 4;
template <typename T, int E, bool IL>
__global__ void __launch_bounds__(512) rope_kernel(const Params<T> p) {
  using C = Chunk<E, IL>;
  const long long t = static_cast<long long>(blockIdx.x) * blockDim.z + threadIdx.z;
  if (t >= p.T_) return;
  const C ch(p.s, threadIdx.x);
  const T* x = p.x + t * p.x_t;
  T* y = p.y + t * p.y_t;
  typename Vec<T, E>::Raw u[kAhead], w[kAhead];
  auto load = [&](int h0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int h = h0 + k * blockDim.y;
      if (h < p.H) {
        u[k] = ld<T, E>(x + h * p.x_h + ch.a);
        if (C::kTwo && ch.b >= 0) w[k] = ld<T, E>(x + h * p.x_h + ch.b);
      }
    }
  };
  load(threadIdx.y);
  const int pos = __ldg(p.positions + t);
  if (pos < 0 || pos >= p.rows) {
    if (threadIdx.x == 0 && threadIdx.y == 0) record_input_error(SITE_POSITION);
    return;
  }
  float cs[C::kEntries], sn[C::kEntries];
  if (ch.entry >= 0) {
    ld_table<C::kEntries>(p.cos + static_cast<size_t>(pos) * p.s.half, ch.entry, cs);
    ld_table<C::kEntries>(p.sin + static_cast<size_t>(pos) * p.s.half, ch.entry, sn);
#pragma unroll
    for (int i = 0; i < C::kEntries; ++i) sn[i] *= p.sign;
  }
  for (int h0 = threadIdx.y; h0 < p.H; h0 += kAhead * blockDim.y) {
    if (h0 != static_cast<int>(threadIdx.y)) load(h0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int h = h0 + k * blockDim.y;
      if (h < p.H) {
        if (ch.entry >= 0) rotate<T, E, IL>(u[k], w[k], cs, sn);
        st<T, E>(y + h * p.y_h + ch.a, u[k]);
        if (C::kTwo && ch.b >= 0) st<T, E>(y + h * p.y_h + ch.b, w[k]);
      }
    }
  }
}

// ------------------------------------------------------------------ ragged paged append
constexpr int kD = 128;
constexpr int kMaxTokens = 4;  // tokens of one block

struct ExtendParams {
  const uint16_t *k, *v, *q;
  uint16_t *q_out, *kp, *vp;
  const int32_t *table, *q_start, *lens, *positions;
  const float *cos, *sin;
  int32_t* slot_pos;  // [B][Hkv][capacity] or nullptr
  long long k_t, k_h, v_t, v_h, q_t, q_h, o_t, o_h;
  int B, T, Hq, Hkv, max_pages, page_size, num_pages, rows, tokens;
  Shape s;
};

struct Token {
  long long page_row;  // (page * Hkv) * page_size + row in the page, or -1: nothing is written
  long long pos_at;    // index of (b, head 0, slot) in slot_pos
  int pos;
};

// Block (chunks, rows): rows walk the token's q heads, k heads and v heads.
template <int E, bool IL>
__global__ void __launch_bounds__(512) extend_kernel(const ExtendParams p) {
  __shared__ Token tok[kMaxTokens];
  const int t0 = blockIdx.x * p.tokens;
  const int n_tok = min(p.tokens, p.T - t0);
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  if (tid < n_tok) {
    const int t = t0 + tid;
    Token k;
    k.page_row = -1;
    k.pos_at = 0;
    k.pos = 0;
    int lo = 0, hi = p.B;  // the last b with q_start[b] <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.q_start + mid) <= t) lo = mid;
      else hi = mid;
    }
    const int a = __ldg(p.q_start + lo), z = __ldg(p.q_start + lo + 1);
    if (a >= 0 && z <= p.T && t >= a && t < z) {
      const long long capacity = static_cast<long long>(p.max_pages) * p.page_size;
      const long long slot = static_cast<long long>(__ldg(p.lens + lo)) - z + t;
      const long long pos = p.positions ? __ldg(p.positions + t) : slot;
      if (slot < 0 || slot >= capacity) {
        record_input_error(SITE_SLOT);
      } else if (p.s.half > 0 && (pos < 0 || pos >= p.rows)) {
        record_input_error(SITE_POSITION);
      } else {
        const int at = static_cast<int>(slot);  // lens is 32-bit
        const int page = __ldg(p.table + static_cast<long long>(lo) * p.max_pages + at / p.page_size);
        if (page < 0 || page >= p.num_pages) {
          record_input_error(SITE_BAD_PAGE);
        } else {
          k.page_row = static_cast<long long>(page) * p.Hkv * p.page_size + at % p.page_size;
          k.pos_at = static_cast<long long>(lo) * p.Hkv * capacity + slot;
          k.pos = static_cast<int>(pos);
        }
      }
    } else if (a < 0 || z > p.T || t < a || t < __ldg(p.q_start + p.B)) {
      record_input_error(SITE_Q_START);  // or a token of no sequence in front of q_start[B]
    }
    tok[tid] = k;
  }
  __syncthreads();
  using C = Chunk<E, IL>;
  const C ch(p.s, threadIdx.x);
  const int n_rows = p.Hq + 2 * p.Hkv;
  const long long capacity = static_cast<long long>(p.max_pages) * p.page_size;
  // kAhead rows at a time, their loads on the way together
  for (int w0 = threadIdx.y; w0 < n_tok * n_rows; w0 += kAhead * blockDim.y) {
    typename Vec<uint16_t, E>::Raw u[kAhead], x[kAhead];
    uint16_t* dst[kAhead];
    int pos[kAhead];  // -1: not rotated
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      dst[k] = nullptr;
      pos[k] = -1;
      const int w = w0 + k * blockDim.y;
      if (w >= n_tok * n_rows) continue;
      const int i = w / n_rows, r = w - i * n_rows;
      const Token tk = tok[i];
      if (tk.page_row < 0) continue;
      const long long t = t0 + i;
      const uint16_t* src;
      if (r < p.Hq) {
        src = p.q + t * p.q_t + r * p.q_h;
        dst[k] = p.q_out + t * p.o_t + r * p.o_h;
        pos[k] = tk.pos;
      } else if (r < p.Hq + p.Hkv) {
        const int h = r - p.Hq;
        src = p.k + t * p.k_t + h * p.k_h;
        dst[k] = p.kp + (tk.page_row + static_cast<long long>(h) * p.page_size) * kD;
        pos[k] = tk.pos;
        if (p.slot_pos && threadIdx.x == 0) p.slot_pos[tk.pos_at + h * capacity] = tk.pos;
      } else {
        const int h = r - p.Hq - p.Hkv;
        src = p.v + t * p.v_t + h * p.v_h;
        dst[k] = p.vp + (tk.page_row + static_cast<long long>(h) * p.page_size) * kD;
      }
      u[k] = ld<uint16_t, E>(src + ch.a);
      if (C::kTwo && ch.b >= 0) x[k] = ld<uint16_t, E>(src + ch.b);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (!dst[k]) continue;
      if (pos[k] >= 0 && ch.entry >= 0) {
        float cs[C::kEntries], sn[C::kEntries];
        ld_table<C::kEntries>(p.cos + static_cast<size_t>(pos[k]) * p.s.half, ch.entry, cs);
        ld_table<C::kEntries>(p.sin + static_cast<size_t>(pos[k]) * p.s.half, ch.entry, sn);
        rotate<uint16_t, E, IL>(u[k], x[k], cs, sn);
      }
      st<uint16_t, E>(dst[k] + ch.a, u[k]);
      if (C::kTwo && ch.b >= 0) st<uint16_t, E>(dst[k] + ch.b, x[k]);
    }
  }
}

inline bool vec_ok(const void* ptr, int esize, long long st, long long sh, int heads) {
  return aligned16(ptr) && (st * esize) % 16 == 0 && (heads == 1 || (sh * esize) % 16 == 0);
}

inline Shape shape_of(int head_dim, int rot, int E, bool il) {
  const int pairs = il && E > 1 ? rot / E : rot / 2 / E;
  return Shape{rot / 2, pairs, pairs + (head_dim - rot) / E};
}

template <typename T, int E>
int launch(Params<T> p, int head_dim, int rot, bool il, cudaStream_t stream) {
  p.s = shape_of(head_dim, rot, E, il);
  // About 256 threads a block: enough of them on an SM to cover the loads' latency.
  const int nc = p.s.n_chunks;
  const int hy = std::max(1, std::min(p.H, 256 / nc));
  const int tz = std::max(1, std::min(16, 256 / (nc * hy)));
  const dim3 block(nc, hy, tz);
  const unsigned grid = static_cast<unsigned>((static_cast<long long>(p.T_) + tz - 1) / tz);
  if (il)
    rope_kernel<T, E, true><<<grid, block, 0, stream>>>(p);
  else
    rope_kernel<T, E, false><<<grid, block, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

template <typename T>
int run(const void* x, void* y, const int32_t* positions, const float* cos, const float* sin, int T_, int H, int head_dim,
        int rot, int rows, long long x_t, long long x_h, long long y_t, long long y_h, int flags, cudaStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  if (T_ < 0 || H <= 0 || head_dim <= 0 || rot <= 0 || rot > head_dim || (rot & 1) || rows <= 0)
    return GQA_ERR_INVALID_ARGUMENT;
  if (flags & ~(GQA_FLAG_INTERLEAVED | GQA_FLAG_INVERSE)) return GQA_ERR_INVALID_ARGUMENT;
  if (head_dim > 512) return GQA_ERR_UNSUPPORTED;
  if (x_t < 0 || x_h < 0 || y_t < 0 || y_h < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (T_ == 0) return GQA_OK;
  if (!x || !y || !positions || !cos || !sin) return GQA_ERR_INVALID_ARGUMENT;
  // rows written once each: tokens and heads of y must not share memory
  if (!rows_apart(T_, H, y_t, y_h, head_dim)) return GQA_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(x) % sizeof(T) || reinterpret_cast<uintptr_t>(y) % sizeof(T) ||
      reinterpret_cast<uintptr_t>(cos) % 4 || reinterpret_cast<uintptr_t>(sin) % 4 ||
      reinterpret_cast<uintptr_t>(positions) % 4)
    return GQA_ERR_MISALIGNED;
  Params<T> p;
  p.x = static_cast<const T*>(x);
  p.y = static_cast<T*>(y);
  p.positions = positions;
  p.cos = cos;
  p.sin = sin;
  p.x_t = x_t, p.x_h = x_h, p.y_t = y_t, p.y_h = y_h;
  p.T_ = T_;
  p.H = H;
  p.rows = rows;
  p.sign = (flags & GQA_FLAG_INVERSE) ? -1.0f : 1.0f;
  const bool il = (flags & GQA_FLAG_INTERLEAVED) != 0;
  const bool vec = (il ? rot : rot / 2) % E == 0 && head_dim % E == 0 && vec_ok(x, sizeof(T), x_t, x_h, H) &&
                   vec_ok(y, sizeof(T), y_t, y_h, H) && aligned16(cos) && aligned16(sin);
  return vec ? launch<T, E>(p, head_dim, rot, il, stream) : launch<T, 1>(p, head_dim, rot, il, stream);
}

}  // namespace ropepos

GQA_ERROR_FLAG_ACCESSOR(error_flag_rope_positions)

}  // namespace gqa

using namespace gqa;

extern "C" int gqa_rope_table_f32(const double* inv_freq, float* cos, float* sin, int rows, int half_dim, int pos0,
                                  double mscale, gqa_stream_t stream) {
  if (!inv_freq || !cos || !sin || rows <= 0 || half_dim <= 0 || pos0 < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (!(mscale > 0.0) || !(mscale < 1e30)) return GQA_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(inv_freq) % 8 || reinterpret_cast<uintptr_t>(cos) % 4 ||
      reinterpret_cast<uintptr_t>(sin) % 4)
    return GQA_ERR_MISALIGNED;
  const long long n = static_cast<long long>(rows) * half_dim;
  if ((n + 255) / 256 > 0x7FFFFFFFLL) return GQA_ERR_UNSUPPORTED;
  ropepos::table_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(inv_freq, cos, sin, n, half_dim,
                                                                                  pos0, mscale);
  return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}

extern "C" int gqa_rope_positions_bf16(const void* x, void* y, const int32_t* positions, const float* cos,
                                       const float* sin, int T, int H, int head_dim, int rot_dim, int table_rows,
                                       long long x_token_stride, long long x_head_stride, long long y_token_stride,
                                       long long y_head_stride, int flags, gqa_stream_t stream) {
  return ropepos::run<uint16_t>(x, y, positions, cos, sin, T, H, head_dim, rot_dim, table_rows, x_token_stride,
                                x_head_stride, y_token_stride, y_head_stride, flags, stream);
}

extern "C" int gqa_rope_positions_f32(const void* x, void* y, const int32_t* positions, const float* cos,
                                      const float* sin, int T, int H, int head_dim, int rot_dim, int table_rows,
                                      long long x_token_stride, long long x_head_stride, long long y_token_stride,
                                      long long y_head_stride, int flags, gqa_stream_t stream) {
  return ropepos::run<float>(x, y, positions, cos, sin, T, H, head_dim, rot_dim, table_rows, x_token_stride,
                             x_head_stride, y_token_stride, y_head_stride, flags, stream);
}

extern "C" int gqa_kv_extend_bf16(const void* k, const void* v, long long k_token_stride, long long k_head_stride,
                                  long long v_token_stride, long long v_head_stride, void* kpages, void* vpages,
                                  const int32_t* block_table, int max_pages_per_seq, int page_size, int num_pages,
                                  const int32_t* q_start, const int32_t* lens, const int32_t* positions,
                                  const float* cos, const float* sin, int table_rows, int rot_dim, const void* q,
                                  long long q_token_stride, long long q_head_stride, void* q_out,
                                  long long q_out_token_stride, long long q_out_head_stride, int32_t* slot_pos, int B,
                                  int T, int Hq, int Hkv, int head_dim, int flags, gqa_stream_t stream) {
  using namespace ropepos;
  if (B <= 0 || T < 0 || Hkv <= 0 || Hq < 0 || max_pages_per_seq <= 0 || page_size <= 0 || num_pages <= 0)
    return GQA_ERR_INVALID_ARGUMENT;
  if (head_dim != kD) return GQA_ERR_UNSUPPORTED;
  if (rot_dim < 0 || rot_dim > head_dim || (rot_dim & 1)) return GQA_ERR_INVALID_ARGUMENT;
  if (flags & ~GQA_FLAG_INTERLEAVED) return GQA_ERR_INVALID_ARGUMENT;
  if (T == 0) return GQA_OK;
  if (!k || !v || !kpages || !vpages || !block_table || !q_start || !lens) return GQA_ERR_INVALID_ARGUMENT;
  if (rot_dim > 0 && (!cos || !sin || table_rows <= 0)) return GQA_ERR_INVALID_ARGUMENT;
  if ((q != nullptr) != (q_out != nullptr) || (q != nullptr) != (Hq > 0)) return GQA_ERR_INVALID_ARGUMENT;
  const long long st[] = {k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  for (long long x : st)
    if (x < 0) return GQA_ERR_INVALID_ARGUMENT;
  if (q) {
    if (q_token_stride < 0 || q_head_stride < 0 || q_out_token_stride < 0 || q_out_head_stride < 0)
      return GQA_ERR_INVALID_ARGUMENT;
    if (!rows_apart(T, Hq, q_out_token_stride, q_out_head_stride, kD)) return GQA_ERR_INVALID_ARGUMENT;
  }
  auto odd = [](const void* ptr, int a) { return reinterpret_cast<uintptr_t>(ptr) % a != 0; };
  if (odd(k, 2) || odd(v, 2) || odd(q, 2) || odd(q_out, 2) || !aligned16(kpages) || !aligned16(vpages) ||
      odd(block_table, 4) || odd(q_start, 4) || odd(lens, 4) || odd(positions, 4) || odd(slot_pos, 4) || odd(cos, 4) ||
      odd(sin, 4))
    return GQA_ERR_MISALIGNED;
  ExtendParams p;
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q = static_cast<const uint16_t*>(q);
  p.q_out = static_cast<uint16_t*>(q_out);
  p.kp = static_cast<uint16_t*>(kpages);
  p.vp = static_cast<uint16_t*>(vpages);
  p.table = block_table;
  p.q_start = q_start;
  p.lens = lens;
  p.positions = positions;
  p.cos = cos;
  p.sin = sin;
  p.slot_pos = slot_pos;
  p.k_t = k_token_stride, p.k_h = k_head_stride, p.v_t = v_token_stride, p.v_h = v_head_stride;
  p.q_t = q_token_stride, p.q_h = q_head_stride, p.o_t = q_out_token_stride, p.o_h = q_out_head_stride;
  p.B = B, p.T = T, p.Hq = Hq, p.Hkv = Hkv;
  p.max_pages = max_pages_per_seq, p.page_size = page_size, p.num_pages = num_pages, p.rows = table_rows;
  const bool vec = rot_dim % ((flags & GQA_FLAG_INTERLEAVED) ? 8 : 16) == 0 && vec_ok(k, 2, k_token_stride, k_head_stride, Hkv) &&
                   vec_ok(v, 2, v_token_stride, v_head_stride, Hkv) &&
                   (!q || (vec_ok(q, 2, q_token_stride, q_head_stride, Hq) &&
                           vec_ok(q_out, 2, q_out_token_stride, q_out_head_stride, Hq))) &&
                   aligned16(cos) && aligned16(sin);
  const bool il = (flags & GQA_FLAG_INTERLEAVED) != 0;
  p.s = shape_of(kD, rot_dim, vec ? 8 : 1, il);
  // Few tokens: one a block, a thread for every chunk, so that one load's latency is all.
  // Many: small blocks of four tokens, of which some look up their slots while others move
  // rows.  Both at 32 + 2 x 8 heads, us for few / many: 256 tokens 4 to 6 / 8 to 9, 512
  // tokens 7 to 9 / 8 to 10, 768 level, 1024 tokens 10 / 9, 2048 tokens 18 / 12, 8192 tokens 80 / 40.
  const int n_rows = Hq + 2 * Hkv;
  p.tokens = T <= 512 ? 1 : 4;
  const dim3 block(p.s.n_chunks, std::max(1, std::min(n_rows, (T <= 512 ? 512 : 128) / p.s.n_chunks)));
  const unsigned grid = static_cast<unsigned>((static_cast<long long>(T) + p.tokens - 1) / p.tokens);
  if (vec && il)
    extend_kernel<8, true><<<grid, block, 0, stream>>>(p);
  else if (vec)
    extend_kernel<8, false><<<grid, block, 0, stream>>>(p);
  else if (il)
    extend_kernel<1, true><<<grid, block, 0, stream>>>(p);
  else
    extend_kernel<1, false><<<grid, block, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? GQA_OK : GQA_ERR_CUDA;
}
