// Attention of few queries over the paged MX4 cache: BF16 queries and results.
#include "kv4_few.hpp"

namespace bsq {
template void launch_kv4_few<1>(const AttentionArgs &, uint32_t, hipStream_t);
}  // namespace bsq
