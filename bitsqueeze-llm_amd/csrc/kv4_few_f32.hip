// Attention of few queries over the paged MX4 cache: FP32 queries or results.
#include "kv4_few.hpp"

namespace bsq {
template void launch_kv4_few<3>(const AttentionArgs &, uint32_t, hipStream_t);
}  // namespace bsq
