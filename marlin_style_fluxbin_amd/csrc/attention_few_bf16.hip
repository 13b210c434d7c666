// attention_few.h for bf16 queries over a 16-bit cache.
#include "attention_few.h"

namespace fx {
template void launch_attention_few<kBF16, 64, false>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
template void launch_attention_few<kBF16, 128, false>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
template void launch_attention_few<kBF16, 256, false>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
}  // namespace fx
