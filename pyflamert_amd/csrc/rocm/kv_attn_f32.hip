// Attention kernels for float32 queries and cache.
#include "kv_attn.hpp"

namespace pfr {
namespace attn {
template void launch<float, float>(hipStream_t, const Args&, Kind, unsigned);
}  // namespace attn
}  // namespace pfr
