// Attention of drafted tokens over a paged cache: what a call's workgroups are, and which build takes it (the kernels:
// paged_tree_attention_kernel.hpp).
#include "paged_tree_attention_kernel.hpp"

namespace ba {

extern template int launch_tree_types<0, false>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);
extern template int launch_tree_types<1, false>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);
extern template int launch_tree_types<0, true>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);
extern template int launch_tree_types<1, true>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);

static int resident_of(int dims) { return dims == 64 ? TreeTile<64, 4>::kResident : dims == 128 ? TreeTile<128, 4>::kResident : TreeTile<256, 4>::kResident; }

// Workgroups: as many as are resident, or fewer where the longest possible requests would not give each its least share.
static TreeWork tree_work(int64_t heads, int64_t group, int64_t dim, int64_t tokens, int64_t requests, int64_t width, int64_t page, int64_t window,
                          void *workspace, size_t *bytes) {
    TreeWork w{};
    const int waves = tree_waves(tokens, requests, group), dims = tree_dims(dim);
    const int64_t rows = 32 * waves, tile = waves == 1 ? 128 : dims == 256 ? 32 : 64;
    const int64_t resident = (int64_t)device_cu_count() * resident_of(dims);
    const double units = (double)heads * (tokens * group / rows + requests);
    const double longest = window > 0 ? std::min((double)width * page, (double)window + tokens + tile) : (double)width * page;
    const double most = std::max(units, units * (longest / tile + 1) / kTreeShare + 1);
    w.groups = (int32_t)std::max<int64_t>(1, std::min<int64_t>(BA_PAGED_COUNTERS, (int64_t)std::min<double>((double)resident, most)));
    w.pitch = (int32_t)((dim + 3) & ~int64_t(3));
    w.group = PageDiv::of((uint32_t)group);
    auto whole = [](size_t n) { return (n + 255) & ~size_t(255); };
    const size_t left = whole((size_t)w.groups * sizeof(TreeLeft)), parts = whole(2 * (size_t)w.groups * rows * sizeof(TreePart));
    const size_t sums = 2 * (size_t)w.groups * rows * w.pitch * sizeof(float);
    if (bytes) *bytes = left + parts + sums;
    if (workspace) {
        w.left = (TreeLeft *)workspace;
        w.parts = (TreePart *)((char *)workspace + left);
        w.sums = (float *)((char *)workspace + left + parts);
    }
    return w;
}

size_t paged_tree_attention_workspace(int64_t heads, int64_t group, int64_t dim, int, int64_t tokens, int64_t requests, int64_t width, int64_t page) {
    size_t bytes = 0;                        // (windows have fewer workgroups, which need no more)
    tree_work(heads, group, dim, tokens, requests, width, page, 0, nullptr, &bytes);
    return bytes;
}

int launch_paged_tree_attention(const PagedTreeAttentionArgs &a, int dtype, int cache_dtype, int32_t *counters, void *workspace, hipStream_t stream) {
    const bool f8 = cache_dtype == BA_F8_E4M3;
    const int waves = tree_waves(a.tokens, a.requests, a.group);
    TreeWork w = tree_work(a.heads, a.group, a.dim, a.tokens, a.requests, a.width, a.page.d, a.window, workspace, nullptr);
    w.counters = counters;
    // Joining within the kernel saves the second launch, but one workgroup then reads all parts of a unit.
    if (waves == 1 && w.groups <= kTreeFewParts * std::max<int64_t>(1, a.tokens * a.group / (32 * waves)) * a.heads) w.left = nullptr;
    const uint64_t bits = (uint64_t)a.k.base | (uint64_t)a.v.base | (uint64_t)a.k.page_bytes | (uint64_t)a.v.page_bytes | (uint64_t)a.k.head_bytes |
                          (uint64_t)a.v.head_bytes | (uint64_t)a.k.token_bytes | (uint64_t)a.v.token_bytes;
    const TreeRows rows = a.dim * (f8 ? 1 : 2) < 16 ? kTreeShort : bits % 16 != 0 || a.dim % (f8 ? 16 : 8) != 0 ? kTreeAny : kTreePieces;
    if (dtype == BA_F16) return f8 ? launch_tree_types<0, true>(a, w, rows, waves, stream) : launch_tree_types<0, false>(a, w, rows, waves, stream);
    return f8 ? launch_tree_types<1, true>(a, w, rows, waves, stream) : launch_tree_types<1, false>(a, w, rows, waves, stream);
}

}  // namespace ba
