// What the kernels of the paged key-value cache share (paged_tables.hip, paged_append.hip, paged_attention.hip) and the
// launchers that capi_paged.hip calls.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/blocked_attention.h"

namespace ba {

// Division of 0 <= n < 2^31 by a number given at run time: with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (mulhi(n, m) + n) >> s (Granlund and Montgomery's round-up method; the sum stays below 2^32).
struct PageDiv {
    uint32_t d, mul, shift;
    static PageDiv of(uint32_t d) {
        uint32_t s = 0;
        while ((uint64_t(1) << s) < d) ++s;
        return {d, (uint32_t)(((((uint64_t)1 << s) - d) << 32) / d + 1), s};
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return (uint32_t)((((uint64_t)n * mul) >> 32) + n) >> shift;
    }
};

// One of the two arrays of a cache.
struct PagedArray {
    char *base;
    const float *scale;                 // per head, 8-bit caches only
    int64_t page_bytes, head_bytes;
    int32_t token_bytes;
};

struct PagedTablesArgs {
    int32_t *table, *free_pages;
    const int64_t *state_in, *lens, *new_lens;
    int64_t *slots, *accum, *lens_out, *state_out;
    int64_t table_stride, pool;
    int32_t requests, width, tokens;
    PageDiv page;
};

struct PagedAppendArgs {
    PagedArray to[2];
    const char *from[2];
    int64_t from_head_bytes[2], from_token_bytes[2];
    const int64_t *slots;
    int64_t tokens, places;             // places: pages * page
    int32_t heads, dim;
    PageDiv page;
};

struct PagedAttentionArgs {
    PagedArray k, v;
    const char *q;
    char *out;
    const int32_t *table;
    const int64_t *lens;
    int64_t q_head_bytes, q_row_bytes, out_head_bytes, out_row_bytes, table_stride;
    int32_t requests, heads, group, dim, pages, width;
    int32_t window;                     // tokens; 0: all
    float scale;
    PageDiv page;
};

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));

// N dwords from any address, past the caches (what streams through once is read at 7.0 TB/s that way, 6.2 otherwise).
template <int N> __device__ __forceinline__ void load_stream(uint32_t (&x)[N], const char *p) {
    static_assert(N == 1 || N == 2 || N == 4);
    if (N == 4) {
        const u32x4_any v = __builtin_nontemporal_load((const u32x4_any *)p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = v[i];
    } else if (N == 2) {
        const u32x2_any v = __builtin_nontemporal_load((const u32x2_any *)p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = v[i];
    } else {
        x[0] = __builtin_nontemporal_load((const u32_any *)p);
    }
}
// The first `bytes` of N dwords (any number, also none or negative), zeros behind.
template <int N> __device__ __forceinline__ void load_part(uint32_t (&x)[N], const char *p, int bytes) {
    if (bytes >= 4 * N) {
        load_stream<N>(x, p);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0;
    if (bytes <= 0) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int left = bytes - 4 * i;
        if (left >= 4) x[i] = *(const u32_any *)(p + 4 * i);
        else if (left >= 2) x[i] = *(const u16_any *)(p + 4 * i) | (left == 3 ? (uint32_t)*(const uint8_t *)(p + 4 * i + 2) << 16 : 0u);
        else if (left == 1) x[i] = *(const uint8_t *)(p + 4 * i);
    }
}

size_t paged_tables_workspace(int64_t requests);
int launch_paged_tables(const PagedTablesArgs &args, void *workspace, hipStream_t stream);
int launch_paged_append(const PagedAppendArgs &args, int dtype, int cache_dtype, hipStream_t stream);
size_t paged_attention_workspace(int64_t cache_heads, int64_t group, int64_t dim, int cache_dtype, int64_t requests, int64_t width, int64_t page);
int launch_paged_attention(const PagedAttentionArgs &args, int dtype, int cache_dtype, int32_t *counters, void *workspace, hipStream_t stream);

}  // namespace ba
