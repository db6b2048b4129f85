// Rows of a page table that go on from other rows: full pages are shared, a last page that is not full is copied for all but one of
// those that go on from the same row, and pages that no row holds any more return to the stack.
//
// With k the number of rows that go on from a row, each of its full pages has k - 1 holders more, its last page, if not full,
// min(k, 1) - 1.  `shares` counts the holders of a page beyond the first; whole-number atomics add the changes up, whose
// order does not matter, and a page is free when that makes it -1.  Counts below that are refused.  Both go by the counts when all changes are in: on
// the way there, with counts that are not right, others may come up, in whatever order the atomics run.
// Freed pages go on the stack in ascending order, fresh pages are numbered by row and come from its end: the place of either is known
// from counts alone, so whoever finds a freed page puts it where it belongs, on the stack or into the row that has its number.
// Three launches, since counts have to be there before they are changed and whole before they are used:
//   begin   shares are copied, counts below 0 found (one of -1 would pass for a page that became free); one workgroup counts who goes on from whom and numbers the fresh pages
//   change  the rows' pages, as far as their holders change, and how many become free in each chunk of pages
//   finish  every workgroup adds up those numbers, then rows, stack and verdict
// A small table takes one launch, all of it in the LDS of one workgroup.  What bounds either are the launches and the round trips to memory in
// each: 32 rows of up to 2000 tokens 8.0 us (three launches 14), 1024 rows of up to 16000 (8 MB) 24.8.
#include <algorithm>

#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kForkThreads = 256;
constexpr int kForkBegin = 1024;             // threads of the first kernel
// Pages that a workgroup of the last kernel looks through, a thread's share of them: few, so that many workgroups look (70 000 pages: 5.3 us, with
// eight a thread 8.8, with sixteen 14), but every workgroup adds up all chunks' numbers, so more where there are many pages.
constexpr int kForkFew = 2, kForkMany = 16;
constexpr int64_t kForkManyPages = 1 << 20;
constexpr int kForkCopies = 1024;            // workgroups that copy the counts, at most
constexpr int kForkRows = 8;                 // rows whose pages a workgroup changes
constexpr int kForkLocal = 2048;             // chunks whose freed pages a workgroup counts in LDS
constexpr int kForkSmall = 8192;            // pages, and entries of the table, that one workgroup deals with

struct ForkWork {
    int32_t *rows;                           // [requests][2]: how many go on from the row; number of its fresh page or -1
    int32_t *totals;                         // fresh pages, verdict of the first kernel, of the second, pages that it leaves below -1
    int32_t *owners;                         // [requests]: the row of a fresh page
    int32_t *chunks;                         // freed pages of a chunk
    int32_t *negative;                       // [copies]: whether a workgroup that copies counts has seen one below 0
    int32_t n_chunks, chunk_log, copies;     // chunks have 2^chunk_log pages
};
static ForkWork fork_work(int64_t requests, int64_t pages, void *workspace, size_t *bytes) {
    ForkWork w{};
    const int64_t chunk = kForkThreads * (pages <= kForkManyPages ? kForkFew : kForkMany);
    w.chunk_log = __builtin_ctzll(chunk);
    w.n_chunks = (int32_t)((pages + chunk - 1) / chunk);
    w.copies = (int32_t)std::min<int64_t>(kForkCopies, (pages + kForkBegin - 1) / kForkBegin);
    char *p = (char *)workspace;
    auto take = [&](int64_t n) {
        char *const at = p;
        p += (4 * n + 255) & ~int64_t(255);
        return at;
    };
    w.rows = (int32_t *)take(2 * requests);
    w.totals = (int32_t *)take(4);
    w.owners = (int32_t *)take(requests);
    w.chunks = (int32_t *)take(w.n_chunks);
    w.negative = (int32_t *)take(w.copies);
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

// Who goes on from whom, by a workgroup of kForkBegin threads with ROWS rows at most: how many from each row, and which of the others
// has its last page (-1: the row itself); put(row, number) with the number of its fresh page or -1.  The number of those; the verdict.
template <int ROWS> struct ForkRows {
    int32_t children[ROWS], keeper[ROWS];
    int32_t verdict, scan[kForkBegin / 64];
};
template <int ROWS, class F> __device__ __forceinline__ int fork_rows(const PagedForkArgs &a, ForkRows<ROWS> &sh, F put) {
    constexpr int kEach = (ROWS + kForkBegin - 1) / kForkBegin;
    const int tid = (int)threadIdx.x, wave = tid >> 6;
    for (int r = tid; r < a.requests; r += kForkBegin) { sh.children[r] = 0; sh.keeper[r] = INT32_MAX; }
    if (tid == 0) sh.verdict = 0;
    __syncthreads();
    int bad = 0;
    for (int r = tid; r < a.requests; r += kForkBegin) {
        const int64_t o = a.origin[r];
        if (held(a, a.lens[r]).bad) bad |= BA_PAGED_BAD_LENGTH;
        if (o < -1 || o >= a.requests) bad |= BA_PAGED_BAD_ORIGIN;
        else if (o >= 0) {
            atomicAdd(&sh.children[o], 1);
            atomicMin(&sh.keeper[o], o == r ? -1 : r);       // the row itself comes before the others
        }
    }
    if (bad) atomicOr(&sh.verdict, bad);
    __syncthreads();
    // fresh pages, numbered by row: thread i has rows [i each, (i + 1) each)
    const int each = (a.requests + kForkBegin - 1) / kForkBegin;
    bool fresh[kEach];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int r = tid * each + i;
        fresh[i] = false;
        if (i < each && r < a.requests) {
            const int64_t o = a.origin[r];
            if (o >= 0 && o < a.requests && o != r && sh.keeper[o] != r) {
                const Held h = held(a, a.lens[o]);
                fresh[i] = h.all > h.full;
            }
        }
        mine += fresh[i];
    }
    int upto = wave_inclusive_scan(mine);
    if (lane_id() == 63) sh.scan[wave] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kForkBegin / 64; ++i) {
        if (i < wave) upto += sh.scan[i];
        total += sh.scan[i];
    }
    int number = upto - mine;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int r = tid * each + i;
        if (i < each && r < a.requests) put(r, fresh[i] ? number : -1);
        number += fresh[i];
    }
    return total;
}

// What becomes of the call: verdict bits, and the pages left on the stack.
struct Outcome {
    int64_t count, left, verdict;
};
__device__ __forceinline__ Outcome outcome(const PagedForkArgs &a, int verdict, int back, int taken) {
    Outcome t{a.state_in[0], 0, a.state_in[1] | verdict};
    if (t.count < 0 || t.count > a.pool || (t.verdict == 0 && t.count + back > a.pool)) t.verdict |= BA_PAGED_BAD_STATE;
    else if (t.verdict == 0 && taken > t.count + back) t.verdict = BA_PAGED_NO_PAGES;
    t.left = t.verdict ? t.count : t.count + back - taken;
    return t;
}

// All of it by one workgroup: at most kForkSmall entries of the table and kForkSmall pages, which are in LDS.  4000 entries 10.0 us, against 15.2
// in three launches; 8000 13.3 against 15.9; 16384 20.5 against 16.4.
constexpr int kForkSmallRows = 1024;
__global__ void __launch_bounds__(kForkBegin) paged_fork_small_kernel(PagedForkArgs a) {
    constexpr int kWaves = kForkBegin / 64, kRounds = kForkSmall / kForkBegin;
    __shared__ int32_t table[kForkSmall], shares[kForkSmall];
    __shared__ int32_t number[kForkSmallRows], owner[kForkSmallRows], page[kForkSmallRows], full[kForkSmallRows], pages_of[kForkSmallRows];
    __shared__ int32_t freed_by[kWaves], bad_shares;
    __shared__ ForkRows<kForkSmallRows> rows;
    const int tid = (int)threadIdx.x, wave = tid >> 6, lane = (int)lane_id();
    const int entries = a.requests * a.width;
    int negative = 0;
#pragma unroll 4
    for (int i = tid; i < a.pages; i += kForkBegin) {
        const int32_t n = a.shares[i];
        shares[i] = n;
        negative |= n < 0;
    }
#pragma unroll 4
    for (int i = tid; i < entries; i += kForkBegin) {
        const int r = (int)a.columns.div((uint32_t)i);
        table[i] = a.table[r * a.table_stride + (i - r * a.width)];
    }
    for (int r = tid; r < a.requests; r += kForkBegin) {
        const Held h = held(a, a.lens[r]);
        full[r] = h.full;
        pages_of[r] = h.all;
    }
    if (tid == 0) bad_shares = 0;
    const int taken = fork_rows(a, rows, [&](int r, int n) {
        number[r] = n;
        if (n >= 0) owner[n] = r;
    });
    if (negative) bad_shares = BA_PAGED_BAD_SHARES;
    __syncthreads();
    if (rows.verdict == 0) {
        int bad = 0;
        for (int i = tid; i < entries; i += kForkBegin) {
            const int r = (int)a.columns.div((uint32_t)i), c = i - r * a.width;
            const int children = rows.children[r], change = c < full[r] ? children - 1 : min(children, 1) - 1;
            if (c >= pages_of[r]) continue;
            if ((uint32_t)table[i] >= (uint32_t)a.pages) bad = BA_PAGED_BAD_SHARES;
            else if (change != 0) atomicAdd(&shares[table[i]], change);
        }
        if (bad) bad_shares = bad;
    }
    __syncthreads();
    uint64_t freed[kRounds];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const int p = (wave * kRounds + i) * 64 + lane;
        const int n = p < a.pages ? shares[p] : 0;
        if (n < -1) bad_shares = BA_PAGED_BAD_SHARES;
        freed[i] = __ballot(n == -1);
        mine += __popcll(freed[i]);
    }
    if (lane == 0) freed_by[wave] = mine;
    __syncthreads();
    int back = 0, ahead = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        ahead += i < wave ? freed_by[i] : 0;
        back += freed_by[i];
    }
    const Outcome t = outcome(a, rows.verdict | bad_shares, back, taken);
    if (tid == 0) { a.state_out[0] = t.left; a.state_out[1] = t.verdict; }
    if (t.verdict) {
        for (int i = tid; i < a.pages; i += kForkBegin) a.shares_out[i] = a.shares[i];
        for (int i = tid; i < entries; i += kForkBegin) {
            const int r = (int)a.columns.div((uint32_t)i);
            a.table_out[r * a.table_out_stride + (i - r * a.width)] = table[i];
        }
        for (int r = tid; r < a.requests; r += kForkBegin) { a.lens_out[r] = a.lens[r]; a.source[r] = -1; a.target[r] = -1; }
        return;
    }
    int64_t place = t.count + ahead;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        if (freed[i] >> lane & 1) {
            const int p = (wave * kRounds + i) * 64 + lane;
            const int64_t at = place + __popcll(freed[i] & ((1ull << lane) - 1));
            shares[p] = 0;
            if (at < t.left) a.free_pages[at] = p;
            else page[owner[t.count + back - 1 - at]] = p;
        }
        place += __popcll(freed[i]);
    }
    for (int r = tid; r < a.requests; r += kForkBegin) {
        const int64_t at = t.count + back - 1 - number[r];
        if (number[r] >= 0 && at < t.count) page[r] = a.free_pages[at];
    }
    __syncthreads();
    for (int i = tid; i < a.pages; i += kForkBegin) a.shares_out[i] = shares[i];
    for (int i = tid; i < entries; i += kForkBegin) {
        const int r = (int)a.columns.div((uint32_t)i), c = i - r * a.width;
        const int o = (int)a.origin[r];
        int32_t p = -1;
        if (o >= 0 && c < pages_of[o]) p = number[r] >= 0 && c == full[o] ? page[r] : table[o * a.width + c];
        a.table_out[r * a.table_out_stride + c] = p;
    }
    for (int r = tid; r < a.requests; r += kForkBegin) {
        const int o = (int)a.origin[r];
        a.lens_out[r] = o >= 0 ? a.lens[o] : 0;
        a.source[r] = number[r] >= 0 ? table[o * a.width + full[o]] : -1;
        a.target[r] = number[r] >= 0 ? page[r] : -1;
    }
}

__global__ void __launch_bounds__(kForkBegin) paged_fork_begin_kernel(PagedForkArgs a, ForkWork w) {
    if (blockIdx.x > 0) {
        const int64_t at = (int64_t)(blockIdx.x - 1) * kForkBegin + threadIdx.x, step = (int64_t)(gridDim.x - 1) * kForkBegin;
        int negative = 0;
        for (int64_t i = at; i < a.pages; i += step) {
            const int32_t n = a.shares[i];
            a.shares_out[i] = n;
            negative |= n < 0;
        }
        for (int64_t i = at; i < w.n_chunks; i += step) w.chunks[i] = 0;
        negative = __syncthreads_or(negative);
        if (threadIdx.x == 0) w.negative[blockIdx.x - 1] = negative;
        return;
    }
    __shared__ ForkRows<BA_PAGED_FORK_ROWS> sh;
    const int total = fork_rows(a, sh, [&](int r, int number) {
        w.rows[2 * r] = sh.children[r];
        w.rows[2 * r + 1] = number;
        if (number >= 0) w.owners[number] = r;
    });
    if (threadIdx.x == 0) { w.totals[0] = total; w.totals[1] = sh.verdict; w.totals[2] = w.totals[3] = 0; }
}

// A workgroup has kForkRows rows and a column a thread.  Rows next to each other that hold the same page there, which those that went on from one
// row do, add their changes up first, and a workgroup counts the freed pages of a chunk in LDS first: atomics on the same few addresses
// wait for each other (1024 rows in sets of 16: 188 us with neither, 41 with the second, 28 with both).  Many chunks need no such care.
__global__ void __launch_bounds__(kForkThreads) paged_fork_change_kernel(PagedForkArgs a, ForkWork w) {
    __shared__ int32_t count[kForkLocal];
    if (w.totals[1]) return;
    const bool local = w.n_chunks <= kForkLocal;
    if (local) {
        for (int i = (int)threadIdx.x; i < w.n_chunks; i += kForkThreads) count[i] = 0;
        __syncthreads();
    }
    const int r0 = (int)blockIdx.x * kForkRows;
    int bad = 0, below = 0;
    for (int64_t c = (int64_t)blockIdx.y * kForkThreads + threadIdx.x; c < a.width; c += (int64_t)gridDim.y * kForkThreads) {
        int32_t page[kForkRows], change[kForkRows], was[kForkRows];
        bool there[kForkRows];
#pragma unroll
        for (int i = 0; i < kForkRows; ++i) {
            const int r = min(r0 + i, a.requests - 1);
            const int children = w.rows[2 * r];
            const Held h = held(a, r0 + i < a.requests ? a.lens[r] : 0);
            change[i] = c < h.full ? children - 1 : c < h.all ? min(children, 1) - 1 : 0;
            page[i] = c < h.all ? a.table[r * a.table_stride + c] : -1;
            there[i] = c < h.all;
        }
#pragma unroll
        for (int i = 0; i < kForkRows; ++i) {
            if ((uint32_t)page[i] >= (uint32_t)a.pages) {
                if (there[i]) bad = BA_PAGED_BAD_SHARES;
                change[i] = 0;
            } else if (i > 0 && page[i] == page[i - 1]) {
                change[i] += change[i - 1];
                change[i - 1] = 0;
            }
        }
#pragma unroll
        for (int i = 0; i < kForkRows; ++i) was[i] = change[i] ? atomicAdd(&a.shares_out[page[i]], change[i]) : 0;
#pragma unroll
        for (int i = 0; i < kForkRows; ++i) {
            // (the steps that a count takes add up to what it is in the end)
            const int now = (int)((uint32_t)was[i] + (uint32_t)change[i]), freed = (now == -1 ? 1 : 0) - (was[i] == -1 ? 1 : 0);
            below += (now < -1 ? 1 : 0) - (was[i] < -1 ? 1 : 0);
            if (freed) {
                if (local) atomicAdd(&count[page[i] >> w.chunk_log], freed);
                else atomicAdd(&w.chunks[page[i] >> w.chunk_log], freed);
            }
        }
    }
    if (local) {
        __syncthreads();
        for (int i = (int)threadIdx.x; i < w.n_chunks; i += kForkThreads)
            if (count[i]) atomicAdd(&w.chunks[i], count[i]);
    }
    if (bad) atomicOr(&w.totals[2], bad);
    if (below) atomicAdd(&w.totals[3], below);
}

// Workgroups 0 .. requests - 1: their row; behind them a chunk each, with the pages that became free.
template <int kRounds> __global__ void __launch_bounds__(kForkThreads) paged_fork_finish_kernel(PagedForkArgs a, ForkWork w) {
    constexpr int kWaves = kForkThreads / 64;
    __shared__ int32_t sums[2][kWaves];
    const int tid = (int)threadIdx.x, wave = tid >> 6, lane = (int)lane_id();
    const bool row_group = (int)blockIdx.x < a.requests;
    const int r = (int)blockIdx.x, chunk = (int)blockIdx.x - a.requests;
    // a wavefront of a chunk has kRounds times 64 pages in order
    const int64_t first = ((int64_t)chunk << w.chunk_log) + wave * 64 * kRounds + lane;
    const int64_t o = row_group ? a.origin[r] : -1;
    const int number = row_group ? w.rows[2 * r + 1] : -1;
    const int64_t len = row_group && o >= 0 && o < a.requests ? a.lens[o] : 0;
    int all = 0, before = 0;
    uint64_t freed[kRounds];
    if (!row_group) {
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int64_t p = first + 64 * i;
            freed[i] = __ballot(p < a.pages && a.shares_out[p] == -1);
        }
    }
    for (int i = tid; i < w.n_chunks; i += kForkThreads) {
        const int n = w.chunks[i];
        all += n;
        before += i < chunk ? n : 0;
    }
    all = wave_inclusive_scan(all);
    before = wave_inclusive_scan(before);
    if (lane == 63) { sums[0][wave] = all; sums[1][wave] = before; }
    int negative = 0;
    for (int i = tid; i < w.copies; i += kForkThreads) negative |= w.negative[i];
    negative = __syncthreads_or(negative);
    int back = 0, ahead = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) { back += sums[0][i]; ahead += sums[1][i]; }
    const int taken = w.totals[0];
    const Outcome t = outcome(a, w.totals[1] | w.totals[2] | (negative || w.totals[3] ? BA_PAGED_BAD_SHARES : 0), back, taken);
    const bool fine = t.verdict == 0;
    const int64_t count = t.count, left = t.left;
    if (blockIdx.x == 0 && tid == 0) {
        a.state_out[0] = left;
        a.state_out[1] = t.verdict;
    }
    if (!row_group) {
        if (!fine) {
            for (int i = 0; i < kRounds; ++i)
                if (first + 64 * i < a.pages) a.shares_out[first + 64 * i] = a.shares[first + 64 * i];
            return;
        }
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kRounds; ++i) mine += __popcll(freed[i]);
        __syncthreads();
        if (lane == 0) sums[0][wave] = mine;
        __syncthreads();
        int64_t place = count + ahead;
        for (int i = 0; i < wave; ++i) place += sums[0][i];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            if (freed[i] >> lane & 1) {
                const int32_t p = (int32_t)(first + 64 * i);
                const int64_t at = place + __popcll(freed[i] & ((1ull << lane) - 1));
                a.shares_out[p] = 0;
                if (at < left) {
                    a.free_pages[at] = p;
                } else {
                    const int owner = w.owners[count + back - 1 - at];
                    a.table_out[owner * a.table_out_stride + held(a, a.lens[a.origin[owner]]).full] = p;
                    a.target[owner] = p;
                }
            }
            place += __popcll(freed[i]);
        }
        return;
    }
    int32_t *const out = a.table_out + r * a.table_out_stride;
    if (!fine) {
        for (int c = tid; c < a.width; c += kForkThreads) out[c] = a.table[r * a.table_stride + c];
        if (tid == 0) { a.lens_out[r] = a.lens[r]; a.source[r] = -1; a.target[r] = -1; }
        return;
    }
    const Held h = held(a, len);
    const int32_t *const from = a.table + (o >= 0 ? o : 0) * a.table_stride;
    const int64_t place = count + back - 1 - number;         // of the fresh page; from `count` on it is a freed one, which its chunk's workgroup writes
    const bool fresh = number >= 0, here = fresh && place < count;
    for (int c = tid; c < a.width; c += kForkThreads)
        if (!fresh || c != h.full) out[c] = c < h.all ? from[c] : -1;
        else if (here) out[c] = a.free_pages[place];
    if (tid == 0) {
        a.lens_out[r] = len;
        a.source[r] = fresh ? from[h.full] : -1;
        if (!fresh || here) a.target[r] = fresh ? a.free_pages[place] : -1;
    }
}

size_t paged_fork_workspace(int64_t requests, int64_t pages) {
    size_t bytes = 0;
    fork_work(requests, pages, nullptr, &bytes);
    return bytes;
}

int launch_paged_fork(const PagedForkArgs &a, void *workspace, hipStream_t stream) {
    if (a.pages <= kForkSmall && a.requests <= kForkSmallRows && (int64_t)a.requests * a.width <= kForkSmall) {
        paged_fork_small_kernel<<<1, kForkBegin, 0, stream>>>(a);
        return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
    }
    const ForkWork w = fork_work(a.requests, a.pages, workspace, nullptr);
    paged_fork_begin_kernel<<<(unsigned)(1 + w.copies), kForkBegin, 0, stream>>>(a, w);
    const dim3 rows((unsigned)(a.requests + kForkRows - 1) / kForkRows, (unsigned)std::min((a.width + kForkThreads - 1) / kForkThreads, 1024));
    if (a.requests > 0 && a.width > 0) paged_fork_change_kernel<<<rows, kForkThreads, 0, stream>>>(a, w);
    const unsigned last = (unsigned)std::max(1, a.requests + w.n_chunks);
    if (a.pages <= kForkManyPages) paged_fork_finish_kernel<kForkFew><<<last, kForkThreads, 0, stream>>>(a, w);
    else paged_fork_finish_kernel<kForkMany><<<last, kForkThreads, 0, stream>>>(a, w);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
