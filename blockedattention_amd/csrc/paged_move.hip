// Keys and values that move within a paged cache: the tokens of an accepted path to the front of their draft, whole pages to other
// pages.  Copies: what they read and write is their floor.  4096 pages of 64 KiB in both arrays (1.07 GB read and written) take 217 us, 4.9 TB/s, a
// large copy's rate; 200 drafts of up to 40 accepted nodes 6.2 us, 32 of up to 6 4.8, 32 pages 4.1, which is launches and the chain
// list, page number, row.
#include <algorithm>

#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 4;               // 16-byte pieces of a thread in flight

// The first `bytes` (1 .. 16) of a piece.
__device__ __forceinline__ void store_some(char *p, const uint32_t (&x)[4], int bytes) {
    if (bytes >= 16) {
        *(u32x4_any *)p = u32x4_any{x[0], x[1], x[2], x[3]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = bytes - 4 * i;
        if (left >= 4) *(u32_any *)(p + 4 * i) = x[i];
        else if (left > 0) {
            if (left >= 2) *(u16_any *)(p + 4 * i) = (uint16_t)x[i];
            if (left & 1) *(uint8_t *)(p + 4 * i + (left & 2)) = (uint8_t)(x[i] >> (8 * (left & 2)));
        }
    }
}

// Place lens[r] + i takes what place lens[r] + path[r][i] has.  A path's entries increase, so entry i comes from place i or behind:
// what an entry overwrites is read by entries before it only.  A workgroup has some heads of a request to itself and takes the path's
// entries in order, loads of a round before its stores; that is the same as if all were read first.
// Grid (request, heads / heads of a workgroup, keys and values).
__global__ void __launch_bounds__(kMoveThreads) paged_keep_kernel(PagedKeepArgs a) {
    __shared__ int32_t ends;
    __shared__ int64_t from[kMoveThreads], to[kMoveThreads];
    const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (group >= (int64_t)a.requests * a.splits) return;
    const int r = (int)(group / a.splits), part = (int)(group - (int64_t)r * a.splits);
    const int h0 = part * a.group_heads, heads = min(a.group_heads, a.heads - h0);
    const PagedArray array = a.arrays[blockIdx.z];
    const PageDiv per_entry = heads == a.group_heads ? a.per_entry : a.per_rest;
    const int64_t *const path = a.path + r * a.path_stride;
    const int64_t base = a.lens[r], room = (int64_t)a.width * a.page.d;
    const int32_t *const row = a.table + r * a.table_stride;
    const uint32_t row_pieces = a.per_row.d;
    const int bytes = a.row_bytes;
    if (threadIdx.x == 0) ends = a.depth;
    __syncthreads();
    for (int i0 = 0; i0 < a.depth; i0 += kMoveThreads) {
        const int i = i0 + (int)threadIdx.x;
        int64_t by = -1, onto = -1;
        if (i < a.depth) {
            const int64_t node = path[i], before = i > 0 ? path[i - 1] : -1;
            if (base < 0 || node < i || node <= before || node >= room - base) atomicMin(&ends, i);
            else if (node != i) {
                const uint32_t s = (uint32_t)(base + node), d = (uint32_t)(base + i);
                const uint32_t sc = a.page.div(s), dc = a.page.div(d);
                const int32_t sp = row[sc], dp = row[dc];
                if ((uint32_t)sp < (uint32_t)a.pages && (uint32_t)dp < (uint32_t)a.pages) {
                    by = sp * array.page_bytes + (int64_t)(s - sc * a.page.d) * array.token_bytes;
                    onto = dp * array.page_bytes + (int64_t)(d - dc * a.page.d) * array.token_bytes;
                }
            }
        }
        from[threadIdx.x] = by; to[threadIdx.x] = onto;
        __syncthreads();
        const int here = min(kMoveThreads, ends - i0);       // entries of this round; the rest of the path does not count
        const uint32_t all = here > 0 ? (uint32_t)here * heads * row_pieces : 0;
        for (uint32_t x0 = 0; x0 < all; x0 += kMovePieces * kMoveThreads) {
            uint32_t x[kMovePieces][4];
            int64_t at[kMovePieces];
            int left[kMovePieces];
#pragma unroll
            for (int k = 0; k < kMovePieces; ++k) {
                const uint32_t e = x0 + k * kMoveThreads + threadIdx.x;
                at[k] = -1;
                if (e < all) {
                    const uint32_t line = a.per_row.div(e), piece = e - line * row_pieces, entry = per_entry.div(e), h = line - entry * heads;
                    const int64_t by_ = from[entry], side = (h0 + h) * array.head_bytes + 16 * piece;
                    left[k] = bytes - 16 * (int)piece;
                    if (by_ >= 0) {
                        load_part<4>(x[k], array.base + by_ + side, left[k]);
                        at[k] = to[entry] + side;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kMovePieces; ++k)
                if (at[k] >= 0) store_some(array.base + at[k], x[k], left[k]);
        }
        if (ends < i0 + kMoveThreads) break;
        __syncthreads();
    }
    if (blockIdx.z == 0 && part == 0 && threadIdx.x == 0) a.lens_out[r] = base < 0 ? base : base + ends;
}

int launch_paged_keep(PagedKeepArgs a, hipStream_t stream) {
    const int row = (a.row_bytes + 15) / 16;
    a.group_heads = std::max(1, std::min(a.heads, 16 / row));
    a.splits = (a.heads + a.group_heads - 1) / a.group_heads;
    a.per_row = PageDiv::of((uint32_t)row);
    a.per_entry = PageDiv::of((uint32_t)(row * a.group_heads));
    a.per_rest = PageDiv::of((uint32_t)(row * (a.heads - (a.splits - 1) * a.group_heads)));
    dim3 grid = flat_grid((int64_t)a.requests * a.splits);
    grid.z = 2;
    paged_keep_kernel<<<grid, kMoveThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

// Pages source[i] into pages target[i].  What a page holds of all heads and tokens is a run of bytes, or runs with gaps; a workgroup
// takes kCopyPieces pieces a thread of a page.  Grid (copy and part of the page, keys and values).
constexpr int kCopyPieces = 4;

__global__ void __launch_bounds__(kMoveThreads) paged_copy_kernel(PagedCopyArgs a) {
    const int64_t group = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int64_t entry = group / a.parts;
    if (entry >= a.copies) return;
    const int32_t from = a.source[entry], to = a.target[entry];
    if ((uint32_t)from >= (uint32_t)a.pages || (uint32_t)to >= (uint32_t)a.pages) return;
    const PagedRuns &runs = a.runs[blockIdx.z];
    const char *const src = runs.base + from * runs.page_bytes;
    char *const dst = runs.base + to * runs.page_bytes;
    const uint32_t x0 = (uint32_t)(group - entry * a.parts) * (uint32_t)a.part_pieces, x1 = min(x0 + (uint32_t)a.part_pieces, runs.pieces);
    for (uint32_t y0 = x0 + threadIdx.x; y0 < x1; y0 += kCopyPieces * kMoveThreads) {
        uint32_t x[kCopyPieces][4];
        int64_t at[kCopyPieces];
        int left[kCopyPieces];
#pragma unroll
        for (int k = 0; k < kCopyPieces; ++k) {
            const uint32_t y = y0 + k * kMoveThreads;
            at[k] = -1;
            if (y < x1) {
                const uint32_t run = runs.per_run.div(y), piece = y - run * runs.per_run.d, outer = runs.per_outer.div(run), inner = run - outer * runs.per_outer.d;
                at[k] = outer * runs.outer_bytes + inner * runs.inner_bytes + 16 * (int64_t)piece;
                left[k] = (int)min((int64_t)16, runs.run_bytes - 16 * (int64_t)piece);
                load_part<4>(x[k], src + at[k], left[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < kCopyPieces; ++k)
            if (at[k] >= 0) store_some(dst + at[k], x[k], left[k]);
    }
}

// The heads and tokens of a page, as few runs as they are.
static PagedRuns runs_of(const PagedArray &x, int64_t heads, int64_t page, int64_t row) {
    PagedRuns r{};
    r.base = x.base; r.page_bytes = x.page_bytes;
    const bool heads_inner = x.head_bytes < x.token_bytes;
    const int64_t n[2] = {heads_inner ? page : heads, heads_inner ? heads : page};       // outer, inner
    const int64_t step[2] = {heads_inner ? x.token_bytes : x.head_bytes, heads_inner ? x.head_bytes : x.token_bytes};
    int64_t inner = n[1], outer = n[0];
    r.run_bytes = row; r.inner_bytes = step[1]; r.outer_bytes = step[0];
    if (inner == 1 || step[1] == r.run_bytes) {
        r.run_bytes *= inner;
        inner = 1;
        if (outer == 1 || step[0] == r.run_bytes) {
            r.run_bytes *= outer;
            outer = 1;
        }
    }
    const int64_t pieces = (r.run_bytes + 15) / 16;
    r.per_run = PageDiv::of((uint32_t)pieces);
    r.per_outer = PageDiv::of((uint32_t)inner);
    r.pieces = (uint32_t)(pieces * inner * outer);
    return r;
}

int launch_paged_copy(PagedCopyArgs a, const PagedArray (&arrays)[2], int64_t heads, int64_t page, int64_t row, hipStream_t stream) {
    for (int i = 0; i < 2; ++i) a.runs[i] = runs_of(arrays[i], heads, page, row);
    const uint32_t most = std::max(a.runs[0].pieces, a.runs[1].pieces);
    uint32_t part = kCopyPieces * kMoveThreads;
    while (part > kMoveThreads && (most + part - 1) / part * a.copies < 512) part /= 2;
    a.part_pieces = (int32_t)part;
    a.parts = (int32_t)((most + part - 1) / part);
    dim3 grid = flat_grid(a.copies * a.parts);
    grid.z = 2;
    paged_copy_kernel<<<grid, kMoveThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
