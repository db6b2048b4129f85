// What each node of a tree of drafted tokens sees, as bits, and how deep it lies, from every node's parent.
//
// sees(i) = {i} + sees(parent(i)), depth(i) = depth(parent(i)) + 1.  A parent comes before its node, so a node's ancestors lie in
// its own block of 64 nodes and in blocks before.  Within a block, a wavefront unites the sets by doubling: after k rounds
// a lane has its 2^k nearest ancestors there and the number of the next one, so six rounds do for any shape; what it has then is one
// word of the result, and the first ancestor outside the block.  From there every node goes on by itself, a word a step: at most
// as many steps as there are blocks, however deep the tree is.
// 256 requests of up to 500 nodes, most of them in long chains (5.4 MB) 6.8 us, eight of up to 16 4.8: a launch.
#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kTreeThreads = 256;
constexpr int kLost = -2;                    // no ancestor, because a parent on the way is none

// Workgroups 0 .. requests - 1 have a request each, those behind them the rows that are no request's.
__global__ void __launch_bounds__(kTreeThreads) paged_tree_kernel(PagedTreeArgs a) {
    __shared__ uint64_t word[BA_PAGED_TREE_NODES];
    __shared__ int32_t above[BA_PAGED_TREE_NODES];
    const int r = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    if (r >= a.requests) {
        const int64_t head = min(max(a.accum[0], (int64_t)0), a.tokens), tail = min(max(a.accum[a.requests], head), a.tokens);
        const int64_t rows = head + a.tokens - tail, step = (int64_t)kTreePadGroups * kTreeThreads;
        for (int64_t i = (int64_t)(r - a.requests) * kTreeThreads + threadIdx.x; i < rows && r < a.requests + kTreePadGroups; i += step) {
            const int64_t row = i < head ? i : tail + (i - head);
            for (int w = 0; w < a.words; ++w) a.mask[row * a.words + w] = 0;
            a.depth[row] = -1;
        }
        return;
    }
    const int64_t first = min(max(a.accum[r], (int64_t)0), a.tokens), last = min(max(a.accum[r + 1], first), a.tokens);
    const int n = (int)min(last - first, (int64_t)a.nodes);
    for (int i0 = (int)threadIdx.x & ~63; i0 < n; i0 += kTreeThreads) {
        const int lane = lane_id(), i = i0 + lane;
        const int64_t parent = i < n ? a.parents[first + i] : -1;
        const uint64_t lost = __ballot(parent < -1 || parent >= i);
        const int up = (int)max(min(parent, (int64_t)i), (int64_t)-1);
        uint64_t sees = 1ull << lane;
        int next = up >= i0 && up < i ? up - i0 : -1;        // nearest ancestor in the block that is not in `sees`
#pragma unroll
        for (int k = 0; k < 6; ++k) {
            const int from = max(next, 0);
            const uint64_t more = __shfl(sees, from);
            const int then = __shfl(next, from);
            if (next >= 0) { sees |= more; next = then; }
        }
        const int outside = __shfl(up, __builtin_ctzll(sees));
        if (i < n) { word[i] = sees; above[i] = sees & lost ? kLost : outside; }
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < last - first; i += kTreeThreads) {
        int64_t *const row = a.mask + (first + i) * a.words;
        int at = i < n ? (int)i : kLost, depth = -1;
        for (; at >= 0; at = above[at]) depth += __builtin_popcountll(word[at]);
        const bool lost = at == kLost;
        at = lost ? -1 : (int)i;
        for (int w = a.words - 1; w >= 0; --w) {
            const bool here = at >> 6 == w && at >= 0;
            row[w] = here ? (int64_t)word[at] : 0;
            if (here) at = above[at];
        }
        a.depth[first + i] = lost ? -1 : depth;
    }
}

int launch_paged_tree(const PagedTreeArgs &a, hipStream_t stream) {
    paged_tree_kernel<<<flat_grid((int64_t)a.requests + kTreePadGroups), kTreeThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
