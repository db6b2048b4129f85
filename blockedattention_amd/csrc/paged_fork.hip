// Rows of a page table that go on from other rows: full pages are shared, a last page that is not full is copied for all but one of
// those that go on from the same row, and pages that no row holds any more return to the stack.
//
// With k the number of rows that go on from a row, each of its full pages has k - 1 holders more, its last page, if not full,
// min(k, 1) - 1.  `shares` counts the holders of a page beyond the first; whole-number atomics add the changes up, whose
// order does not matter, and a page is free when that makes it -1: every holder takes 1 away, so only the last one sees it,
// and marks the page in a bitmap.  Freed pages go on the stack in ascending order, which is their place among the marks; fresh pages
// are numbered by row and come from the end of the stack, so every one of them is found by itself, as in pagedResize.
// Three launches, since counts have to be there before they are changed and whole before they are used:
//   begin   shares are copied, marks cleared; one workgroup counts who goes on from whom and numbers the fresh pages
//   change  the rows' pages, as far as their holders change
//   finish  every workgroup adds up the marks, then rows, stack and verdict
// A step of 32 rows of up to 2000 tokens 13.2 us, 1024 rows of up to 16000 (8 MB) 188.
#include <algorithm>

#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kForkThreads = 256;
constexpr int kForkBegin = 1024;             // threads of the first kernel
constexpr int kForkChunk = 32 * kForkThreads;          // pages whose marks a workgroup of the last kernel has, a word a thread
constexpr int kForkEach = (BA_PAGED_FORK_ROWS + kForkBegin - 1) / kForkBegin;

struct ForkWork {
    int32_t *rows;                           // [requests][2]: how many go on from the row; number of its fresh page or -1
    int32_t *totals;                         // fresh pages, verdict so far
    int32_t *chunks;                         // marks of a chunk
    uint32_t *marks;
    int32_t n_chunks;
};
static ForkWork fork_work(int64_t requests, int64_t pages, void *workspace, size_t *bytes) {
    ForkWork w{};
    w.n_chunks = (int32_t)((pages + kForkChunk - 1) / kForkChunk);
    char *p = (char *)workspace;
    auto take = [&](int64_t n) {
        char *const at = p;
        p += (4 * n + 255) & ~int64_t(255);
        return at;
    };
    w.rows = (int32_t *)take(2 * requests);
    w.totals = (int32_t *)take(2);
    w.chunks = (int32_t *)take(w.n_chunks);
    w.marks = (uint32_t *)take((int64_t)w.n_chunks * kForkThreads);
    if (bytes) *bytes = (size_t)(p - (char *)workspace);
    return w;
}

// Pages of a row, full ones, and whether its length is one.
struct Held {
    int full, all;
    bool bad;
};
__device__ __forceinline__ Held held(const PagedForkArgs &a, int64_t len) {
    Held h;
    h.bad = len < 0 || len > (int64_t)a.width * a.page.d;
    const uint32_t n = h.bad ? 0u : (uint32_t)len;
    h.full = (int)a.page.div(n);
    h.all = h.full + (h.full * a.page.d < n ? 1 : 0);
    return h;
}

__global__ void __launch_bounds__(kForkBegin) paged_fork_begin_kernel(PagedForkArgs a, ForkWork w) {
    if (blockIdx.x > 0) {
        const int64_t at = (int64_t)(blockIdx.x - 1) * kForkBegin + threadIdx.x, step = (int64_t)(gridDim.x - 1) * kForkBegin;
        for (int64_t i = at; i < a.pages; i += step) a.shares_out[i] = a.shares[i];
        for (int64_t i = at; i < (int64_t)w.n_chunks * kForkThreads; i += step) w.marks[i] = 0;
        for (int64_t i = at; i < w.n_chunks; i += step) w.chunks[i] = 0;
        return;
    }
    __shared__ int32_t children[BA_PAGED_FORK_ROWS], keeper[BA_PAGED_FORK_ROWS];
    __shared__ int32_t verdict, scan[kForkBegin / 64];
    const int tid = (int)threadIdx.x, wave = tid >> 6;
    for (int r = tid; r < a.requests; r += kForkBegin) { children[r] = 0; keeper[r] = INT32_MAX; }
    if (tid == 0) verdict = 0;
    __syncthreads();
    int bad = 0;
    for (int r = tid; r < a.requests; r += kForkBegin) {
        const int64_t o = a.origin[r];
        if (held(a, a.lens[r]).bad) bad |= BA_PAGED_BAD_LENGTH;
        if (o < -1 || o >= a.requests) bad |= BA_PAGED_BAD_ORIGIN;
        else if (o >= 0) {
            atomicAdd(&children[o], 1);
            atomicMin(&keeper[o], o == r ? -1 : r);          // the row itself comes before the others
        }
    }
    if (bad) atomicOr(&verdict, bad);
    __syncthreads();
    // fresh pages, numbered by row: thread i has rows [i each, (i + 1) each)
    const int each = (a.requests + kForkBegin - 1) / kForkBegin;
    bool fresh[kForkEach];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kForkEach; ++i) {
        const int r = tid * each + i;
        fresh[i] = false;
        if (i < each && r < a.requests) {
            const int64_t o = a.origin[r];
            if (o >= 0 && o < a.requests && o != r && keeper[o] != r) {
                const Held h = held(a, a.lens[o]);
                fresh[i] = h.all > h.full;
            }
        }
        mine += fresh[i];
    }
    int upto = wave_inclusive_scan(mine);
    if (lane_id() == 63) scan[wave] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kForkBegin / 64; ++i) {
        if (i < wave) upto += scan[i];
        total += scan[i];
    }
    int number = upto - mine;
#pragma unroll
    for (int i = 0; i < kForkEach; ++i) {
        const int r = tid * each + i;
        if (i < each && r < a.requests) {
            w.rows[2 * r] = children[r];
            w.rows[2 * r + 1] = fresh[i] ? number : -1;
        }
        number += fresh[i];
    }
    if (tid == 0) { w.totals[0] = total; w.totals[1] = verdict; }
}

// Workgroup r: the pages of row r, unless as many rows hold them as before.
__global__ void __launch_bounds__(kForkThreads) paged_fork_change_kernel(PagedForkArgs a, ForkWork w) {
    const int r = (int)blockIdx.x;
    const int children = w.rows[2 * r];
    if (children == 1 || w.totals[1]) return;
    const Held h = held(a, a.lens[r]);
    const int32_t *const row = a.table + r * a.table_stride;
    int bad = 0;
    for (int c = (int)threadIdx.x; c < h.all; c += kForkThreads) {
        const int change = (c < h.full ? children : min(children, 1)) - 1;
        if (change == 0) continue;
        const int32_t p = row[c];
        if ((uint32_t)p >= (uint32_t)a.pages) {
            bad = BA_PAGED_BAD_SHARES;
            continue;
        }
        const int was = atomicAdd(&a.shares_out[p], change), now = was + change;
        if (was < 0 || now < -1) {
            bad = BA_PAGED_BAD_SHARES;
        } else if (now == -1) {
            atomicOr(&w.marks[p >> 5], 1u << (p & 31));
            atomicAdd(&w.chunks[p / kForkChunk], 1);
        }
    }
    if (bad) atomicOr(&w.totals[1], bad);
}

// Workgroups 0 .. requests - 1: their row; behind them a chunk each, whose freed pages they put on the stack.
__global__ void __launch_bounds__(kForkThreads) paged_fork_finish_kernel(PagedForkArgs a, ForkWork w) {
    __shared__ int32_t scan[kForkThreads / 64], picked, rest;
    const int tid = (int)threadIdx.x, wave = tid >> 6;
    const bool row_group = (int)blockIdx.x < a.requests;
    const int chunk = (int)blockIdx.x - a.requests;
    // marks of all chunks, of those before this one, and (rows) the chunk that has a given one
    auto block_sum = [&](int v) {
        const int s = wave_inclusive_scan(v);
        __syncthreads();
        if (lane_id() == 63) scan[wave] = s;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int i = 0; i < kForkThreads / 64; ++i) all += scan[i];
        return all;
    };
    int all = 0, before = 0;
    for (int i = tid; i < w.n_chunks; i += kForkThreads) {
        all += w.chunks[i];
        before += i < chunk ? w.chunks[i] : 0;
    }
    const int back = block_sum(all);
    before = row_group ? 0 : block_sum(before);
    const int taken = w.totals[0];
    const int64_t count = a.state_in[0], said = a.state_in[1];
    int64_t verdict = w.totals[1] | said;
    if (count < 0 || count + back > a.pool) verdict |= BA_PAGED_BAD_STATE;
    else if (verdict == 0 && taken > count + back) verdict = BA_PAGED_NO_PAGES;
    const bool fine = verdict == 0;
    const int64_t left = count + back - taken;
    if (blockIdx.x == 0 && tid == 0) {
        a.state_out[0] = fine ? left : count;
        a.state_out[1] = verdict;
    }
    if (!row_group) {
        if (!fine) {
            const int64_t p0 = (int64_t)chunk * kForkChunk, p1 = min(p0 + kForkChunk, (int64_t)a.pages);
            for (int64_t p = p0 + tid; p < p1; p += kForkThreads) a.shares_out[p] = a.shares[p];
            return;
        }
        const int64_t word = (int64_t)chunk * kForkThreads + tid;
        uint32_t marks = w.marks[word];
        const int mine = __builtin_popcount(marks);
        int upto = wave_inclusive_scan(mine);
        __syncthreads();
        if (lane_id() == 63) scan[wave] = upto;
        __syncthreads();
        for (int i = 0; i < wave; ++i) upto += scan[i];
        int64_t place = count + before + upto - mine;
        for (; marks; marks &= marks - 1, ++place) {
            const int32_t p = (int32_t)(32 * word + __builtin_ctz(marks));
            a.shares_out[p] = 0;
            if (place < left) a.free_pages[place] = p;
        }
        return;
    }
    const int r = (int)blockIdx.x;
    int32_t *const out = a.table_out + r * a.table_out_stride;
    if (!fine) {
        for (int c = tid; c < a.width; c += kForkThreads) out[c] = a.table[r * a.table_stride + c];
        if (tid == 0) { a.lens_out[r] = a.lens[r]; a.source[r] = -1; a.target[r] = -1; }
        return;
    }
    const int64_t o = a.origin[r];
    const int number = w.rows[2 * r + 1];
    const int64_t len = o >= 0 ? a.lens[o] : 0;
    const Held h = held(a, len);
    const int32_t *const from = a.table + (o >= 0 ? o : 0) * a.table_stride;
    int32_t page = -1;
    if (number >= 0) {
        // place of the fresh page on the stack; past what was on it, the freed pages in ascending order
        const int64_t place = count + back - 1 - number;
        if (place < count) {
            page = a.free_pages[place];
        } else {
            int want = (int)(place - count), c = 0;
            for (int i0 = 0; i0 < w.n_chunks; i0 += kForkThreads) {
                const int i = i0 + tid, mine = i < w.n_chunks ? w.chunks[i] : 0;
                int upto = wave_inclusive_scan(mine);
                __syncthreads();
                if (tid == 0) picked = -1;
                if (lane_id() == 63) scan[wave] = upto;
                __syncthreads();
                int sum = 0;
                for (int k = 0; k < kForkThreads / 64; ++k) {
                    if (k < wave) upto += scan[k];
                    sum += scan[k];
                }
                if (want >= upto - mine && want < upto) { picked = i; rest = want - (upto - mine); }
                __syncthreads();
                if (picked >= 0) {
                    c = picked;
                    want = rest;
                    break;
                }
                want -= sum;
            }
            uint32_t marks = w.marks[(int64_t)c * kForkThreads + tid];
            const int mine = __builtin_popcount(marks);
            int upto = wave_inclusive_scan(mine);
            __syncthreads();
            if (lane_id() == 63) scan[wave] = upto;
            __syncthreads();
            for (int i = 0; i < wave; ++i) upto += scan[i];
            int nth = want - (upto - mine);
            if (nth >= 0 && nth < mine) {
                for (; nth > 0; --nth) marks &= marks - 1;
                picked = c * kForkChunk + 32 * tid + __builtin_ctz(marks);
            }
            __syncthreads();
            page = picked;
        }
    }
    for (int c = tid; c < a.width; c += kForkThreads) out[c] = c < h.all ? (number >= 0 && c == h.full ? page : from[c]) : -1;
    if (tid == 0) {
        a.lens_out[r] = len;
        a.source[r] = number >= 0 ? from[h.full] : -1;
        a.target[r] = page;
    }
}

size_t paged_fork_workspace(int64_t requests, int64_t pages) {
    size_t bytes = 0;
    fork_work(requests, pages, nullptr, &bytes);
    return bytes;
}

int launch_paged_fork(const PagedForkArgs &a, void *workspace, hipStream_t stream) {
    const ForkWork w = fork_work(a.requests, a.pages, workspace, nullptr);
    const int64_t groups = std::min<int64_t>(1024, (a.pages + kForkBegin - 1) / kForkBegin);
    paged_fork_begin_kernel<<<(unsigned)(1 + groups), kForkBegin, 0, stream>>>(a, w);
    if (a.requests > 0) paged_fork_change_kernel<<<(unsigned)a.requests, kForkThreads, 0, stream>>>(a, w);
    paged_fork_finish_kernel<<<(unsigned)std::max(1, a.requests + w.n_chunks), kForkThreads, 0, stream>>>(a, w);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
