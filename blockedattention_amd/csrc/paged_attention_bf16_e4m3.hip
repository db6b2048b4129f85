// Paged attention: bf16 queries, cache in 8 bits.
#include "paged_attention_kernel.hpp"

namespace ba {
template int launch_paged_dtype<1, true>(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream);
}  // namespace ba
