// Attention kernels for float32 queries and a float16 cache.
#include "kv_attn.hpp"

namespace pfr {
namespace attn {
template void launch<float, _Float16>(hipStream_t, const Args&, Kind, unsigned);
}  // namespace attn
}  // namespace pfr
