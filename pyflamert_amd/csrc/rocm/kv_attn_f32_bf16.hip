// Attention kernels for float32 queries and a bfloat16 cache.
#include "kv_attn.hpp"

namespace pfr {
namespace attn {
template void launch<float, __bf16>(hipStream_t, const Args&, Kind, unsigned);
}  // namespace attn
}  // namespace pfr
