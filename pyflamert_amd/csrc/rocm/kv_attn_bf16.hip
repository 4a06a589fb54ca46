// Attention kernels for bfloat16 queries and cache.
#include "kv_attn.hpp"

namespace pfr {
namespace attn {
template void launch<__bf16, __bf16>(hipStream_t, const Args&, Kind, unsigned);
}  // namespace attn
}  // namespace pfr
