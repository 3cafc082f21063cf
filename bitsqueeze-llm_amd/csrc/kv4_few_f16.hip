// Attention of few queries over the paged MX4 cache: FP16 queries or results.
#include "kv4_few.hpp"

namespace bsq {
template void launch_kv4_few<2>(const AttentionArgs &, uint32_t, hipStream_t);
}  // namespace bsq
