// Page tables and slot maps from the requests' lengths before and after a call.
#include "ba_device.hpp"
#include "paged.hpp"

namespace ba {

__device__ __forceinline__ int pages_of(const PageDiv &page, int tokens) {
    return tokens > 0 ? (int)page.div((uint32_t)(tokens - 1)) + 1 : 0;
}

// One thread, one request after the other.
__global__ void paged_tables_kernel(PagedTablesArgs a) {
    if (threadIdx.x) return;
    const int64_t count = a.state_in[0], limit = (int64_t)a.width * a.page.d;
    int64_t verdict = a.state_in[1], take = 0, drop = 0, grow = 0;
    for (int r = 0; r < a.requests; ++r) {
        const int64_t o = a.lens[r], n = a.new_lens[r];
        a.accum[r] = grow;
        if (o < 0 || n < 0 || o > limit) { verdict |= BA_PAGED_BAD_LENGTH; continue; }
        if (n > limit) { verdict |= BA_PAGED_ROW_SHORT; continue; }
        const int po = pages_of(a.page, (int)o), pn = pages_of(a.page, (int)n);
        take += max(pn - po, 0); drop += max(po - pn, 0); grow += n > o ? n - o : 0;
    }
    a.accum[a.requests] = grow;
    if (count < 0 || count + drop > a.pool) verdict |= BA_PAGED_BAD_STATE;
    if (!verdict) verdict = (take > count + drop ? BA_PAGED_NO_PAGES : 0) | (grow > a.tokens ? BA_PAGED_NO_SLOTS : 0);
    a.state_out[0] = verdict ? count : count + drop - take;
    a.state_out[1] = verdict;
    int64_t slot = 0, taken = 0;
    if (!verdict) {
        // the pages given back lie on the stack first, the last one lowest
        int64_t j = 0;
        for (int r = 0; r < a.requests; ++r) {
            const int po = pages_of(a.page, (int)a.lens[r]), pn = pages_of(a.page, (int)a.new_lens[r]);
            for (int c = pn; c < po; ++c, ++j)
                if (j >= take) a.free_pages[count + drop - 1 - j] = a.table[r * a.table_stride + c];
        }
        int r2 = -1, c2 = 0, e2 = 0;              // the next page given back
        for (int r = 0; r < a.requests; ++r) {
            const int o = (int)a.lens[r], n = (int)a.new_lens[r];
            const int po = pages_of(a.page, o), pn = pages_of(a.page, n);
            for (int c = po; c < pn; ++c, ++taken) {
                int32_t page;
                if (taken < drop) {
                    while (c2 >= e2) { ++r2; e2 = pages_of(a.page, (int)a.lens[r2]); c2 = pages_of(a.page, (int)a.new_lens[r2]); }
                    page = a.table[r2 * a.table_stride + c2++];
                } else {
                    page = a.free_pages[count - 1 - (taken - drop)];
                }
                a.table[r * a.table_stride + c] = page;
            }
            for (int t = o; t < n; ++t) {
                const uint32_t c = a.page.div((uint32_t)t);
                a.slots[slot++] = (int64_t)a.table[r * a.table_stride + c] * a.page.d + ((uint32_t)t - c * a.page.d);
            }
        }
    }
    for (; slot < a.tokens; ++slot) a.slots[slot] = -1;
    for (int r = 0; r < a.requests; ++r) a.lens_out[r] = verdict ? a.lens[r] : a.new_lens[r];
    for (int r = 0; verdict && r <= a.requests; ++r) a.accum[r] = 0;
}

int launch_paged_tables(const PagedTablesArgs &a, void *, hipStream_t stream) {
    paged_tables_kernel<<<1, 64, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
