// Attention of drafted tokens: bf16 queries, 8-bit cache.
#include "paged_tree_attention_kernel.hpp"

namespace ba {
template int launch_tree_types<1, true>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);
}  // namespace ba
