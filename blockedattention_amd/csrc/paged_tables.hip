// Page tables and slot maps from the requests' lengths before and after a call.
//
// With o and n the pages of a request before and after, take = max(n - o, 0), drop = max(o - n, 0), grow = max(new - old, 0):
// three prefix sums over the requests give every new token its request (the place of its number in the sums of grow) and
// every new page its number i, and i tells where the page comes from without anyone having moved anything: the i-th
// page given back (found in the sums of drop, read from the row of the request that gives it) or, past those, a place
// of the free stack.  So every token works out its own slot, nothing waits for a write of another thread, and the
// call writes the same when it is made again.  It is bound by latency: the lengths, one page and one table entry are
// loads one behind the other (256 requests with a token each 4.0 us, an empty launch 3.6).
#include <algorithm>

#include "ba_device.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kTableThreads = 512;
constexpr int kTableWaves = kTableThreads / 64;
constexpr int kTableRequests = 4096;         // with so many requests every workgroup keeps the three sums in LDS
// Workgroups: each makes the sums again, and a token is a chain of loads.  So one token a thread up to kTableGroups workgroups,
// beyond those four at once (49 495 tokens of 2000 requests 7.4 us, with four 9.4; 300 168 of 64 prompts 7.6, with one 7.5;
// 1.2 million of 64 17.3, with one 19.6; 1.04 million of 1000 17.3, with one 21.3).
constexpr int kTableGroups = 128;
constexpr int kTableEach = kTableRequests / kTableThreads;      // requests of a thread at most

__device__ __forceinline__ int pages_of(const PageDiv &page, int tokens) {
    return tokens > 0 ? (int)page.div((uint32_t)(tokens - 1)) + 1 : 0;
}

struct Change {
    int64_t take, drop, grow;
    int verdict;
};
__device__ __forceinline__ Change change_of(const PagedTablesArgs &a, int64_t o, int64_t n) {
    const int64_t limit = (int64_t)a.width * a.page.d;
    if (o < 0 || n < 0 || o > limit || n > limit)
        return {0, 0, 0, (o < 0 || n < 0 || o > limit ? BA_PAGED_BAD_LENGTH : 0) | (n > limit ? BA_PAGED_ROW_SHORT : 0)};
    const int d = pages_of(a.page, (int)n) - pages_of(a.page, (int)o);
    return {max(d, 0), max(-d, 0), n > o ? n - o : 0, 0};
}

// What all requests together change, and the verdict on it (the state given may hold any two numbers).
struct Totals {
    int64_t count, take, drop, grow, verdict;
};
__device__ __forceinline__ void judge(const PagedTablesArgs &a, Totals &t) {
    if (t.count < 0 || t.count > a.pool - t.drop) t.verdict |= BA_PAGED_BAD_STATE;
    if (!t.verdict) t.verdict = (t.take > t.count + t.drop ? BA_PAGED_NO_PAGES : 0) | (t.grow > a.tokens ? BA_PAGED_NO_SLOTS : 0);
}

// Prefix sums of `v` over the workgroup: exclusive for each thread; `sum` gets the total.
template <int WAVES> __device__ __forceinline__ Change scan_changes(const Change &v, Change &sum, Change *waves) {
    const int lane = lane_id(), wave = (int)threadIdx.x >> 6;
    Change upto = {wave_inclusive_scan(v.take), wave_inclusive_scan(v.drop), wave_inclusive_scan(v.grow), v.verdict};
#pragma unroll
    for (int bit = 1; bit <= BA_PAGED_BAD_STATE; bit *= 2) upto.verdict |= __any(v.verdict & bit) ? bit : 0;
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    sum = {0, 0, 0, 0};
    Change before = {upto.take - v.take, upto.drop - v.drop, upto.grow - v.grow, 0};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        if (i < wave) { before.take += waves[i].take; before.drop += waves[i].drop; before.grow += waves[i].grow; }
        sum.take += waves[i].take; sum.drop += waves[i].drop; sum.grow += waves[i].grow; sum.verdict |= waves[i].verdict;
    }
    __syncthreads();
    return before;
}

// The requests r with sums[r] <= i < sums[r + 1], for several i at once: the steps of their searches overlap.
template <int K, typename T> __device__ __forceinline__ void owners(int (&r)[K], const T *sums, int requests, const int64_t (&i)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) r[k] = 0;
    for (int len = requests; len > 1;) {
        const int half = len >> 1;
#pragma unroll
        for (int k = 0; k < K; ++k) r[k] += (int64_t)sums[r[k] + half] <= i[k] ? half : 0;
        len -= half;
    }
}

// Slots, pages and stack entries, thread `me` of `all`.
template <int K, typename P, typename G>
__device__ __forceinline__ void fill(const PagedTablesArgs &a, const Totals &t, const P *take, const P *drop, const G *grow, int64_t me, int64_t all) {
    // page numbers that are given back
    auto given = [&](int32_t (&page)[K], const int64_t (&j)[K], const bool (&wanted)[K]) {
        int r[K];
        owners(r, drop, a.requests, j);
        int64_t n[K];
#pragma unroll
        for (int k = 0; k < K; ++k) n[k] = wanted[k] ? a.new_lens[r[k]] : 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (wanted[k]) page[k] = a.table[r[k] * a.table_stride + pages_of(a.page, (int)n[k]) + (j[k] - (int64_t)drop[r[k]])];
    };
    for (int64_t i0 = me; i0 < a.tokens; i0 += K * all) {
        int64_t i[K], old[K], number[K];
        int r[K], column[K], line[K], had[K];
        int32_t page[K];
        bool mine[K], given_back[K];
        bool some = false;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            i[k] = i0 + k * all;
            mine[k] = i[k] < a.tokens && i[k] < t.grow && !t.verdict;
        }
        if (a.requests) owners(r, grow, a.requests, i);
#pragma unroll
        for (int k = 0; k < K; ++k) old[k] = mine[k] ? a.lens[r[k]] : 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            given_back[k] = false;
            page[k] = 0;
            number[k] = 0;
            if (!mine[k]) continue;
            const int at = (int)old[k] + (int)(i[k] - (int64_t)grow[r[k]]);
            column[k] = (int)a.page.div((uint32_t)at);
            line[k] = at - column[k] * (int)a.page.d;
            had[k] = pages_of(a.page, (int)old[k]);
            number[k] = (int64_t)take[r[k]] + column[k] - had[k];
            if (column[k] < had[k]) page[k] = a.table[r[k] * a.table_stride + column[k]];
            else if (number[k] < t.drop) given_back[k] = some = true;
            else page[k] = a.free_pages[t.count - 1 - (number[k] - t.drop)];
        }
        if (some) given(page, number, given_back);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            // (a page's first token is always new where the page is)
            if (mine[k] && column[k] >= had[k] && line[k] == 0) a.table[r[k] * a.table_stride + column[k]] = page[k];
            if (i[k] < a.tokens) a.slots[i[k]] = mine[k] ? (int64_t)page[k] * a.page.d + line[k] : -1;
        }
    }
    if (!t.verdict)
        for (int64_t j0 = t.take + me; j0 < t.drop; j0 += K * all) {
            int64_t j[K];
            int32_t page[K];
            bool wanted[K];
#pragma unroll
            for (int k = 0; k < K; ++k) { j[k] = j0 + k * all; wanted[k] = j[k] < t.drop; }
            given(page, j, wanted);
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (wanted[k]) a.free_pages[t.count + t.drop - 1 - j[k]] = page[k];
        }
    if (me == 0) {
        a.state_out[0] = t.verdict ? t.count : t.count + t.drop - t.take;
        a.state_out[1] = t.verdict;
    }
}

// Every workgroup makes the three sums for itself, in LDS.
template <int K> __global__ void __launch_bounds__(kTableThreads) paged_tables_kernel(PagedTablesArgs a) {
    __shared__ Change waves[kTableWaves];
    extern __shared__ int32_t sums[];               // take, drop, grow: [requests] each
    int32_t *const take = sums, *const drop = sums + a.requests, *const grow = drop + a.requests;
    const int c = (a.requests + kTableThreads - 1) / kTableThreads;
    const int r0 = min(a.requests, (int)threadIdx.x * c), r1 = min(a.requests, r0 + c);
    Totals t = {a.state_in[0], 0, 0, 0, a.state_in[1]};
    // all lengths of the thread are asked for before the first is used
    int64_t o[kTableEach], n[kTableEach];
#pragma unroll
    for (int i = 0; i < kTableEach; ++i) {
        if (i >= c) break;
        o[i] = r0 + i < r1 ? a.lens[r0 + i] : 0;
        n[i] = r0 + i < r1 ? a.new_lens[r0 + i] : 0;
    }
    Change mine = {0, 0, 0, 0}, all;
#pragma unroll
    for (int i = 0; i < kTableEach; ++i) {
        if (i >= c) break;
        const Change x = change_of(a, o[i], n[i]);
        mine = {mine.take + x.take, mine.drop + x.drop, mine.grow + x.grow, mine.verdict | x.verdict};
    }
    Change before = scan_changes<kTableWaves>(mine, all, waves);
    t.take = all.take; t.drop = all.drop; t.grow = all.grow; t.verdict |= all.verdict;
    judge(a, t);
#pragma unroll
    for (int i = 0; i < kTableEach; ++i) {
        const int r = r0 + i;
        if (r >= r1) break;
        const Change x = change_of(a, o[i], n[i]);
        take[r] = (int32_t)before.take; drop[r] = (int32_t)before.drop; grow[r] = (int32_t)before.grow;
        if (blockIdx.x == 0) {
            a.accum[r] = t.verdict ? 0 : before.grow;
            a.lens_out[r] = t.verdict ? o[i] : n[i];
        }
        before = {before.take + x.take, before.drop + x.drop, before.grow + x.grow, 0};
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.accum[a.requests] = t.verdict ? 0 : t.grow;
    __syncthreads();
    fill<K>(a, t, take, drop, grow, (int64_t)blockIdx.x * kTableThreads + threadIdx.x, (int64_t)gridDim.x * kTableThreads);
}

// More requests: one workgroup makes the sums (grow: the accum result), a second launch reads them (5000 requests, 124 000 tokens
// 32 + 16 us).
struct TableSums {
    Totals totals;
    int64_t sums[];                                  // take, drop: [requests] each
};
__global__ void __launch_bounds__(1024) paged_table_sums_kernel(PagedTablesArgs a, TableSums *w) {
    __shared__ Change waves[16];
    Totals t = {a.state_in[0], 0, 0, 0, a.state_in[1]};
    for (int first = 0; first < a.requests; first += 1024) {
        const int r = first + (int)threadIdx.x;
        Change all;
        const Change mine = r < a.requests ? change_of(a, a.lens[r], a.new_lens[r]) : Change{0, 0, 0, 0}, before = scan_changes<16>(mine, all, waves);
        if (r < a.requests) {
            w->sums[r] = t.take + before.take;
            w->sums[a.requests + r] = t.drop + before.drop;
            a.accum[r] = t.grow + before.grow;
        }
        t.take += all.take; t.drop += all.drop; t.grow += all.grow; t.verdict |= all.verdict;
    }
    judge(a, t);
    if (threadIdx.x == 0) {
        w->totals = t;
        a.accum[a.requests] = t.verdict ? 0 : t.grow;
    }
    for (int r = (int)threadIdx.x; r < a.requests; r += 1024) {
        a.lens_out[r] = t.verdict ? a.lens[r] : a.new_lens[r];
        if (t.verdict) a.accum[r] = 0;              // (this thread's own writes)
    }
}
template <int K> __global__ void __launch_bounds__(kTableThreads) paged_table_fill_kernel(PagedTablesArgs a, const TableSums *w) {
    fill<K>(a, w->totals, w->sums, w->sums + a.requests, a.accum, (int64_t)blockIdx.x * kTableThreads + threadIdx.x, (int64_t)gridDim.x * kTableThreads);
}

size_t paged_tables_workspace(int64_t requests) {
    return requests > kTableRequests ? sizeof(TableSums) + 2 * (size_t)requests * sizeof(int64_t) : 0;
}

int launch_paged_tables(const PagedTablesArgs &a, void *workspace, hipStream_t stream) {
    const int64_t rounds = ((int64_t)a.tokens + kTableThreads - 1) / kTableThreads;
    const unsigned groups = (unsigned)std::min<int64_t>(kTableGroups, std::max<int64_t>(1, rounds));
    const bool many = rounds > kTableGroups;
    if (a.requests > kTableRequests) {
        paged_table_sums_kernel<<<1, 1024, 0, stream>>>(a, (TableSums *)workspace);
        if (many) paged_table_fill_kernel<4><<<groups, kTableThreads, 0, stream>>>(a, (const TableSums *)workspace);
        else paged_table_fill_kernel<1><<<groups, kTableThreads, 0, stream>>>(a, (const TableSums *)workspace);
    } else {
        const size_t lds = 3 * (size_t)a.requests * sizeof(int32_t);
        if (many) paged_tables_kernel<4><<<groups, kTableThreads, lds, stream>>>(a);
        else paged_tables_kernel<1><<<groups, kTableThreads, lds, stream>>>(a);
    }
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
