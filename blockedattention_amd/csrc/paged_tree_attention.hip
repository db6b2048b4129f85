// Attention of drafted tokens over a paged cache: what a call's workgroups are, and which kernel takes it (paged_tree_few.hpp, paged_tree_wide.hpp).
#include "paged_tree_few.hpp"
#include "paged_tree_wide.hpp"

namespace ba {

#define BA_TREE(DT, F8) \
    extern template int launch_tree_few<DT, F8>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int sets, hipStream_t stream); \
    extern template int launch_tree_wide<DT, F8>(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);
BA_TREE(0, false)
BA_TREE(1, false)
BA_TREE(0, true)
BA_TREE(1, true)

template <int DC> static int resident_of(int rows) {
    if constexpr (DC <= 128)
        if (rows == 32) return TreeFew<DC, 2>::kResident;
    return rows == 128 ? TreeWide<DC, 4>::kResident : rows == 64 ? TreeWide<64, 2>::kResident : TreeFew<DC, 1>::kResident;
}

// Tokens that a row sees at most, as far as the call's sizes tell.
static int64_t longest_of(int64_t tokens, int64_t width, int64_t page, int64_t window) {
    return window > 0 ? std::min(width * page, window + tokens) : width * page;
}

// Workgroups: as many as are resident, or fewer where the longest possible requests would not give each its least share.
static TreeWork tree_work(int rows, int64_t heads, int64_t group, int64_t dim, int64_t tokens, int64_t requests, int64_t longest, void *workspace, size_t *bytes) {
    TreeWork w{};
    const int dims = dim_class(dim);
    const int64_t tile = rows < 64 ? 32 * kTreeWaves : rows == 128 && dims == 256 ? 32 : 64;
    const int64_t resident = (int64_t)device_cu_count() * (dims == 64 ? resident_of<64>(rows) : dims == 128 ? resident_of<128>(rows) : resident_of<256>(rows));
    const double units = (double)heads * (tokens * group / rows + requests);
    const double most = units * ((double)longest / tile + 2 + kTreeUnit) / kTreeShare + 1;
    w.groups = (int32_t)std::max<int64_t>(1, std::min<int64_t>(BA_PAGED_COUNTERS, (int64_t)std::min<double>((double)resident, most)));
    w.pitch = (int32_t)((dim + 3) & ~int64_t(3));
    w.group = PageDiv::of((uint32_t)group);
    auto whole = [](size_t n) { return (n + 255) & ~size_t(255); };
    const size_t left = whole((size_t)w.groups * sizeof(TreeLeft)), parts = whole(2 * (size_t)w.groups * rows * sizeof(PagedPart));
    const size_t sums = 2 * (size_t)w.groups * rows * w.pitch * sizeof(float);
    if (bytes) *bytes = left + parts + sums;
    if (workspace) {
        w.left = (TreeLeft *)workspace;
        w.parts = (PagedPart *)((char *)workspace + left);
        w.sums = (float *)((char *)workspace + left + parts);
    }
    return w;
}

// (a window can make a call brief, which then has other units; else fewer workgroups, which need no more)
size_t paged_tree_attention_workspace(int64_t heads, int64_t group, int64_t dim, int64_t tokens, int64_t requests, int64_t width, int64_t page) {
    size_t most = 0;
    for (const int64_t longest : {width * page, std::min(width * page, kTreeBrief)}) {
        size_t bytes = 0;
        tree_work(tree_rows(heads, tokens, requests, group, dim, longest), heads, group, dim, tokens, requests, longest, nullptr, &bytes);
        most = std::max(most, bytes);
    }
    return most;
}

int launch_paged_tree_attention(const PagedTreeAttentionArgs &a, int dtype, int cache_dtype, int32_t *counters, void *workspace, hipStream_t stream) {
    const bool f8 = cache_dtype == BA_F8_E4M3;
    const int64_t longest = longest_of(a.tokens, a.width, a.page.d, a.window);
    const int unit = tree_rows(a.heads, a.tokens, a.requests, a.group, a.dim, longest);
    const uint64_t bits = (uint64_t)a.k.base | (uint64_t)a.v.base | (uint64_t)a.k.page_bytes | (uint64_t)a.v.page_bytes | (uint64_t)a.k.head_bytes |
                          (uint64_t)a.v.head_bytes | (uint64_t)a.k.token_bytes | (uint64_t)a.v.token_bytes;
    const TreeRows rows = a.dim * (f8 ? 1 : 2) < 16 ? kTreeShort : bits % 16 != 0 || a.dim % (f8 ? 16 : 8) != 0 ? kTreeAny : kTreePieces;
    TreeWork w = tree_work(unit, a.heads, a.group, a.dim, a.tokens, a.requests, longest, workspace, nullptr);
    w.counters = counters;
    // Joining within the kernel saves the second launch, but one workgroup then reads all parts of a unit.
    if (unit < 64 && w.groups <= kTreeFewParts * std::max<int64_t>(1, a.tokens * a.group / unit) * a.heads) w.left = nullptr;
    if (dtype == BA_F16) {
        if (unit >= 64) return f8 ? launch_tree_wide<0, true>(a, w, rows, unit / 32, stream) : launch_tree_wide<0, false>(a, w, rows, unit / 32, stream);
        return f8 ? launch_tree_few<0, true>(a, w, rows, unit / 16, stream) : launch_tree_few<0, false>(a, w, rows, unit / 16, stream);
    }
    if (unit >= 64) return f8 ? launch_tree_wide<1, true>(a, w, rows, unit / 32, stream) : launch_tree_wide<1, false>(a, w, rows, unit / 32, stream);
    return f8 ? launch_tree_few<1, true>(a, w, rows, unit / 16, stream) : launch_tree_few<1, false>(a, w, rows, unit / 16, stream);
}

}  // namespace ba
