// Paged attention: what a call's workgroups are, and which build takes it (the kernels: paged_attention_kernel.hpp).
#include "paged_attention_kernel.hpp"

namespace ba {

extern template int launch_paged_dtype<0, false>(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream);
extern template int launch_paged_dtype<1, false>(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream);
extern template int launch_paged_dtype<0, true>(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream);
extern template int launch_paged_dtype<1, true>(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream);

// Workgroups: as many as are resident, or fewer where the longest possible requests would not give each its least share.
// (The window counts: three requests that look at 69 tokens 7.4 us, with workgroups for the length and thus a joining kernel 15.)
static PagedWork work_of(int64_t heads, int64_t group, int64_t dim, bool f8, bool any, int64_t requests, int64_t width, int64_t page, int64_t window, void *workspace, size_t *bytes) {
    PagedWork w{};
    const int sets = group > kPagedHeads ? 2 : 1;
    w.tiles_a_head = (int32_t)((group + sets * kPagedHeads - 1) / (sets * kPagedHeads));
    w.rows = (int32_t)((group + w.tiles_a_head - 1) / w.tiles_a_head);
    const int64_t resident = (int64_t)device_cu_count() * resident_groups(dim_class(dim), f8, sets, any);
    const int64_t units = requests * heads * w.tiles_a_head;
    const double longest = window > 0 ? std::min((double)width * page, (double)window + kPagedTile) : (double)width * page;
    const double most = std::max((double)units, (double)units * (longest / kPagedTile + 1) / kPagedShare + 1);
    w.groups = (int32_t)std::max<int64_t>(1, std::min<int64_t>(BA_PAGED_COUNTERS, (int64_t)std::min<double>((double)resident, most)));
    // (the list is only used where units are far fewer than workgroups, see below)
    const size_t split = ((size_t)std::min<int64_t>(units, w.groups) * sizeof(Left) + 255) & ~size_t(255);
    const size_t parts = (2 * (size_t)w.groups * w.rows * sizeof(PagedPart) + 255) & ~size_t(255);
    w.pitch = (int32_t)((dim + 3) & ~int64_t(3));
    const size_t sums = 2 * (size_t)w.groups * w.rows * w.pitch * sizeof(float);
    if (bytes) *bytes = split + parts + sums;
    if (workspace) {
        w.split = (Left *)workspace;
        w.parts = (PagedPart *)((char *)workspace + split);
        w.sums = (float *)((char *)workspace + split + parts);
    }
    return w;
}

size_t paged_attention_workspace(int64_t heads, int64_t group, int64_t dim, int cache_dtype, int64_t requests, int64_t width, int64_t page) {
    size_t bytes = 0;                        // (rows at any address and windows have fewer workgroups, which need no more)
    work_of(heads, group, dim, cache_dtype == BA_F8_E4M3, false, requests, width, page, 0, nullptr, &bytes);
    return bytes;
}

int launch_paged_attention(const PagedAttentionArgs &a, int dtype, int cache_dtype, int32_t *counters, void *workspace, hipStream_t stream) {
    const bool f8 = cache_dtype == BA_F8_E4M3;
    PagedWork w = work_of(a.heads, a.group, a.dim, f8, build_of(a, f8).shape != kFull, a.requests, a.width, a.page.d, a.window, workspace, nullptr);
    w.counters = counters;
    // Joining within the kernel saves the second launch (about 3 us), but one workgroup then reads all parts of a unit: at 32 parts
    // of 8 heads it takes 5 us more than a kernel that spreads them, at 96 parts 14 us.
    if (w.groups <= kPagedFewParts * a.requests * (int64_t)a.heads * w.tiles_a_head) w.split = nullptr;
    if (dtype == BA_F16) return f8 ? launch_paged_dtype<0, true>(a, w, stream) : launch_paged_dtype<0, false>(a, w, stream);
    return f8 ? launch_paged_dtype<1, true>(a, w, stream) : launch_paged_dtype<1, false>(a, w, stream);
}

}  // namespace ba
