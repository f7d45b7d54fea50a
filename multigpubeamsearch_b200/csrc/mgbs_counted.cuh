// Forms of the operators for callers inside the library: the number of batch entries comes from the device.
#pragma once
#include <stdint.h>

#include "mgbs.h"

namespace mgbs {

// Batch entries done: min(batch, *count_dev - count_offset), none where that is negative; all with count_dev null.
int rel_attention_counted(const MgbsRelAttentionArgs* args, const uint32_t* count_dev, int64_t count_offset, void* stream);
int qk_norm_rope_counted(const MgbsQkNormArgs* args, const uint32_t* count_dev, int64_t count_offset, void* stream);

}  // namespace mgbs
