// kv_wide.h -- the tensor-core attention kernel's launch (kv_attend_wide.cu).
#pragma once
#include "kv.h"

namespace iq {
// `ctas`: tiles of 128 query rows x KV heads x slots.
cudaError_t kv_attend_wide_launch(const KvAttnArgs& a, int64_t ctas, bool vec, cudaStream_t st);
}  // namespace iq
