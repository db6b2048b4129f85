// Paged attention: bf16 queries and cache.
#include "paged_attention_kernel.hpp"

namespace ba {
template int launch_paged_dtype<1, false>(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream);
}  // namespace ba
