// attention_rows.h for bf16 queries over the 4-bit cache.
#include "attention_rows.h"

namespace fx {
template void launch_attention_rows<kBF16, 64, true>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
template void launch_attention_rows<kBF16, 128, true>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
template void launch_attention_rows<kBF16, 256, true>(const CachedAttentionPlan&, const CachedAttentionArgs&, hipStream_t);
}  // namespace fx
