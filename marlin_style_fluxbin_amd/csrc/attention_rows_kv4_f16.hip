// attention_rows.h for f16 queries over the 4-bit cache.
#include "attention_rows.h"

namespace fx {
template void launch_attention_rows<kF16, 64, true>(const CachedAttentionArgs&, hipStream_t);
template void launch_attention_rows<kF16, 128, true>(const CachedAttentionArgs&, hipStream_t);
template void launch_attention_rows<kF16, 256, true>(const CachedAttentionArgs&, hipStream_t);
}  // namespace fx
