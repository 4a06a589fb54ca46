// Attention kernels for float16 queries and cache.
#include "kv_attn.hpp"

namespace pfr {
namespace attn {
template void launch<_Float16, _Float16>(hipStream_t, const Args&, Kind, unsigned);
}  // namespace attn
}  // namespace pfr
