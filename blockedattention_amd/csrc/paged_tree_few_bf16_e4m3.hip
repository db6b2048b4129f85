// Attention of drafted tokens, few rows: bf16 queries, 8-bit cache.
#include "paged_tree_few.hpp"

namespace ba {
template int launch_tree_few<1, true>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int sets, hipStream_t stream);
}  // namespace ba
