// Attention of drafted tokens, many rows: fp16 queries, 8-bit cache.
#include "paged_tree_wide.hpp"

namespace ba {
template int launch_tree_wide<0, true>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);
}  // namespace ba
