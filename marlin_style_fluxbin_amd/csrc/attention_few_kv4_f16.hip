// attention_few.h for f16 queries over the 4-bit cache.
#include "attention_few.h"

namespace fx {
template void launch_attention_few<kF16, 64, true>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
template void launch_attention_few<kF16, 128, true>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
template void launch_attention_few<kF16, 256, true>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
}  // namespace fx
