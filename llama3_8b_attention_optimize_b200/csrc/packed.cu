// packed.cu -- gqa_packed_call: the chunked-serving entry points with their arguments in
// one int64 array.
#include <cstdint>
#include <tuple>
#include <type_traits>

#include "gqa_internal.h"

namespace gqa {
namespace {

struct Scalars {  // what comes from outside the array
  float scale;
  gqa_stream_t stream;
};

template <typename A>
constexpr bool kPacked = !std::is_same_v<A, float> && !std::is_same_v<A, gqa_stream_t>;

// The next argument, of type A; `fits` turns false where an integer does not hold its value.
template <typename A>
A take(const int64_t* args, int& at, bool& fits, const Scalars& s) {
  if constexpr (std::is_same_v<A, float>) {
    return s.scale;
  } else if constexpr (std::is_same_v<A, gqa_stream_t>) {
    return s.stream;
  } else if constexpr (std::is_pointer_v<A>) {
    return reinterpret_cast<A>(static_cast<intptr_t>(args[at++]));
  } else {
    const int64_t v = args[at++];
    const A a = static_cast<A>(v);
    fits = fits && static_cast<int64_t>(a) == v;
    return a;
  }
}

template <typename... A>
int unpack(int (*fn)(A...), const int64_t* args, int n, const Scalars& s) {
  if (n != (0 + ... + (kPacked<A> ? 1 : 0))) return GQA_ERR_INVALID_ARGUMENT;
  int at = 0;
  bool fits = true;
  std::tuple<A...> v{take<A>(args, at, fits, s)...};  // a braced list takes them in order
  return fits ? std::apply(fn, v) : GQA_ERR_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace gqa

using namespace gqa;

extern "C" int gqa_packed_call(int entry, const int64_t* args, int n, float scale, gqa_stream_t stream) {
  if (!args) return GQA_ERR_INVALID_ARGUMENT;
  const Scalars s = {scale, stream};
  switch (entry) {
    case GQA_PACKED_ROPE_POSITIONS_BF16: return unpack(gqa_rope_positions_bf16, args, n, s);
    case GQA_PACKED_ROPE_POSITIONS_F32: return unpack(gqa_rope_positions_f32, args, n, s);
    case GQA_PACKED_KV_EXTEND_BF16: return unpack(gqa_kv_extend_bf16, args, n, s);
    case GQA_PACKED_ATTEND_CHUNK_BF16: return unpack(gqa_attend_chunk_bf16, args, n, s);
    case GQA_PACKED_ATTN_WEIGHT_SUMS_F32: return unpack(gqa_attn_weight_sums_f32, args, n, s);
    case GQA_PACKED_KV_EVICT_BF16: return unpack(gqa_kv_evict_bf16, args, n, s);
    default: return GQA_ERR_INVALID_ARGUMENT;
  }
}
