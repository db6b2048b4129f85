// extern "C" entry points of the paged key-value cache: argument checks and launches.  No allocation, no host
// synchronisation, nothing kept between calls.
#include <algorithm>

#include "paged.hpp"

namespace ba {

constexpr int64_t kTokenLimit = int64_t(1) << 31;      // tokens, places and bytes inside a page are 32-bit numbers

static bool bad_stride(int64_t s) { return s < 0 || s > (int64_t(1) << 40); }

// BA_OK, or what a cache that no kernel takes is refused with.  The stride of a dimension of one entry is used by nothing and may
// be anything: `c` becomes the same cache with 0 there (in pages of one token with something in range, which still tells whether
// the heads lie closer together).  moved: what it holds is only moved, so scales do not matter.
static int check_cache(const ba_paged_cache *given, ba_paged_cache *c, bool moved = false) {
    if (!given) return BA_ERR_INVALID_ARG;
    *c = *given;
    if (c->pages <= 1) c->k_page_stride = c->v_page_stride = 0;
    if (c->heads == 1) c->k_head_stride = c->v_head_stride = 0;
    if (c->page == 1)
        for (int64_t *s : {&c->k_token_stride, &c->v_token_stride}) *s = std::clamp<int64_t>(*s, 0, 1 << 28);
    if (c->pages < 0 || c->heads < 1 || c->page < 1 || c->dim < 1) return BA_ERR_INVALID_ARG;
    if (c->dtype != BA_F16 && c->dtype != BA_BF16 && c->dtype != BA_F8_E4M3) return BA_ERR_UNSUPPORTED;
    if (!moved && ((c->dtype == BA_F8_E4M3) != (c->k_scale != nullptr) || (c->dtype == BA_F8_E4M3) != (c->v_scale != nullptr)))
        return BA_ERR_INVALID_ARG;
    if (c->pages > 0 && (!c->k || !c->v)) return BA_ERR_INVALID_ARG;
    const int64_t strides[] = {c->k_page_stride, c->k_head_stride, c->k_token_stride, c->v_page_stride, c->v_head_stride, c->v_token_stride};
    for (int64_t s : strides)
        if (bad_stride(s)) return BA_ERR_INVALID_ARG;
    if (c->dim > 256 || c->pages >= kTokenLimit || c->page >= kTokenLimit || c->heads >= (1 << 20)) return BA_ERR_UNSUPPORTED;
    for (int64_t s : {c->k_token_stride, c->v_token_stride})
        if (s >= kTokenLimit || 2 * ((c->page - 1) * s + c->dim) >= kTokenLimit) return BA_ERR_UNSUPPORTED;
    return BA_OK;
}

static int elem_bytes(int dtype) { return dtype == BA_F8_E4M3 ? 1 : 2; }

static PagedArray array_of(const ba_paged_cache *c, bool values) {
    const int e = elem_bytes(c->dtype);
    if (values) return {(char *)c->v, c->v_scale, c->v_page_stride * e, c->v_head_stride * e, (int32_t)(c->v_token_stride * e)};
    return {(char *)c->k, c->k_scale, c->k_page_stride * e, c->k_head_stride * e, (int32_t)(c->k_token_stride * e)};
}

}  // namespace ba

using namespace ba;

extern "C" {

__attribute__((visibility("default"))) size_t ba_paged_resize_workspace(int64_t requests) {
    return paged_tables_workspace(requests);
}

__attribute__((visibility("default"))) int ba_paged_resize(int32_t *table, int64_t table_stride, int64_t width,
                                                           int32_t *free_pages, int64_t pool, const int64_t *state_in,
                                                           const int64_t *lens, const int64_t *new_lens, int64_t requests,
                                                           int64_t page, int64_t *slots, int64_t tokens, int64_t *accum,
                                                           int64_t *lens_out, int64_t *state_out, void *workspace,
                                                           size_t workspace_bytes, ba_stream_t stream) {
    if (requests < 0 || page < 1 || width < 0 || pool < 0 || tokens < 0 || table_stride < 0) return BA_ERR_INVALID_ARG;
    if (!state_in || !state_out || !accum) return BA_ERR_INVALID_ARG;
    if (requests > 0 && (!lens || !new_lens || !lens_out || (width > 0 && !table))) return BA_ERR_INVALID_ARG;
    if ((pool > 0 && !free_pages) || (tokens > 0 && !slots)) return BA_ERR_INVALID_ARG;
    if (requests > 1 && width > 0 && table_stride < width) return BA_ERR_INVALID_ARG;
    if (requests >= kTokenLimit || width >= kTokenLimit || page >= kTokenLimit || tokens >= kTokenLimit || pool >= kTokenLimit ||
        requests * width >= kTokenLimit || width * page >= kTokenLimit)
        return BA_ERR_UNSUPPORTED;
    const size_t need = ba_paged_resize_workspace(requests);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 7))) return BA_ERR_WORKSPACE;
    PagedTablesArgs a{table, free_pages, state_in, lens, new_lens, slots, accum, lens_out, state_out, table_stride, pool,
                      (int32_t)requests, (int32_t)width, (int32_t)tokens, PageDiv::of((uint32_t)page)};
    return launch_paged_tables(a, workspace, (hipStream_t)stream);
}

__attribute__((visibility("default"))) int ba_paged_append(const ba_paged_cache *cache, int dtype, const void *k,
                                                           int64_t k_head_stride, int64_t k_token_stride, const void *v,
                                                           int64_t v_head_stride, int64_t v_token_stride,
                                                           const int64_t *slots, int64_t tokens, ba_stream_t stream) {
    ba_paged_cache plain;
    const int st = check_cache(cache, &plain);
    if (st != BA_OK) return st;
    cache = &plain;
    if (dtype != BA_F16 && dtype != BA_BF16) return BA_ERR_UNSUPPORTED;
    if (cache->dtype != BA_F8_E4M3 && cache->dtype != dtype) return BA_ERR_UNSUPPORTED;
    if (tokens < 0 || bad_stride(k_head_stride) || bad_stride(k_token_stride) || bad_stride(v_head_stride) || bad_stride(v_token_stride))
        return BA_ERR_INVALID_ARG;
    if (tokens >= kTokenLimit) return BA_ERR_UNSUPPORTED;
    if (tokens == 0 || cache->pages == 0) return BA_OK;
    if (!k || !v || !slots) return BA_ERR_INVALID_ARG;
    PagedAppendArgs a{};
    a.to[0] = array_of(cache, false); a.to[1] = array_of(cache, true);
    a.from[0] = (const char *)k; a.from[1] = (const char *)v;
    a.from_head_bytes[0] = 2 * k_head_stride; a.from_head_bytes[1] = 2 * v_head_stride;
    a.from_token_bytes[0] = 2 * k_token_stride; a.from_token_bytes[1] = 2 * v_token_stride;
    a.slots = slots; a.tokens = tokens; a.places = cache->pages * cache->page;
    a.heads = (int32_t)cache->heads; a.dim = (int32_t)cache->dim; a.page = PageDiv::of((uint32_t)cache->page);
    if (a.places >= kTokenLimit) return BA_ERR_UNSUPPORTED;
    return launch_paged_append(a, dtype, cache->dtype, (hipStream_t)stream);
}

__attribute__((visibility("default"))) size_t ba_paged_attention_workspace(const ba_paged_cache *cache, int64_t heads,
                                                                           int64_t requests, int64_t width) {
    ba_paged_cache plain;
    if (check_cache(cache, &plain) != BA_OK || heads < 1 || heads % cache->heads || requests < 1 || width < 0) return 0;
    return paged_attention_workspace(cache->heads, heads / cache->heads, cache->dim, cache->dtype, requests, width, cache->page);
}

__attribute__((visibility("default"))) int ba_paged_attention(const ba_paged_cache *cache, int dtype, const void *q,
                                                              int64_t q_head_stride, int64_t q_row_stride, int64_t heads,
                                                              int64_t requests, const int32_t *table, int64_t table_stride,
                                                              int64_t width, const int64_t *lens, int64_t window,
                                                              float scale, void *out, int64_t out_head_stride,
                                                              int64_t out_row_stride, int32_t *counters, void *workspace,
                                                              size_t workspace_bytes, ba_stream_t stream) {
    ba_paged_cache plain;
    const int st = check_cache(cache, &plain);
    if (st != BA_OK) return st;
    cache = &plain;
    if (dtype != BA_F16 && dtype != BA_BF16) return BA_ERR_UNSUPPORTED;
    if (cache->dtype != BA_F8_E4M3 && cache->dtype != dtype) return BA_ERR_UNSUPPORTED;
    if (heads < 1 || heads % cache->heads || requests < 0 || width < 0 || window < 0 || table_stride < 0) return BA_ERR_INVALID_ARG;
    if (bad_stride(q_head_stride) || bad_stride(q_row_stride) || bad_stride(out_head_stride) || bad_stride(out_row_stride))
        return BA_ERR_INVALID_ARG;
    if (requests == 0) return BA_OK;
    if (!q || !out || !lens || !counters || (width > 0 && !table)) return BA_ERR_INVALID_ARG;
    if (requests > 1 && width > 0 && table_stride < width && table_stride != 0) return BA_ERR_INVALID_ARG;   // (0: a row for all, only read)
    if (heads >= (1 << 20) || requests >= kTokenLimit / heads || width >= kTokenLimit || width * cache->page >= kTokenLimit)
        return BA_ERR_UNSUPPORTED;
    const size_t need = ba_paged_attention_workspace(cache, heads, requests, width);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255)) return BA_ERR_WORKSPACE;
    PagedAttentionArgs a{};
    a.k = array_of(cache, false); a.v = array_of(cache, true);
    a.q = (const char *)q; a.out = (char *)out; a.table = table; a.lens = lens;
    a.q_head_bytes = 2 * q_head_stride; a.q_row_bytes = 2 * q_row_stride;
    a.out_head_bytes = 2 * out_head_stride; a.out_row_bytes = 2 * out_row_stride;
    a.table_stride = table_stride;
    a.requests = (int32_t)requests; a.heads = (int32_t)cache->heads; a.group = (int32_t)(heads / cache->heads);
    a.dim = (int32_t)cache->dim; a.pages = (int32_t)cache->pages; a.width = (int32_t)width;
    a.window = (int32_t)std::min<int64_t>(window, kTokenLimit - 1);
    a.scale = scale; a.page = PageDiv::of((uint32_t)cache->page);
    return launch_paged_attention(a, dtype, cache->dtype, counters, workspace, (hipStream_t)stream);
}

__attribute__((visibility("default"))) int ba_paged_tree(const int64_t *parents, const int64_t *accum, int64_t requests, int64_t tokens,
                                                         int64_t nodes, int64_t *mask, int64_t *depth, ba_stream_t stream) {
    if (requests < 0 || tokens < 0 || nodes < 1 || !accum) return BA_ERR_INVALID_ARG;
    if (nodes > BA_PAGED_TREE_NODES || requests >= kTokenLimit - kTreePadGroups || tokens >= kTokenLimit) return BA_ERR_UNSUPPORTED;
    if (tokens == 0) return BA_OK;
    if (!parents || !mask || !depth) return BA_ERR_INVALID_ARG;
    const PagedTreeArgs a{parents, accum, mask, depth, tokens, (int32_t)requests, (int32_t)nodes, (int32_t)((nodes + 63) / 64)};
    return launch_paged_tree(a, (hipStream_t)stream);
}

__attribute__((visibility("default"))) size_t ba_paged_tree_attention_workspace(const ba_paged_cache *cache, int64_t heads, int64_t tokens,
                                                                                int64_t requests, int64_t width) {
    ba_paged_cache plain;
    if (check_cache(cache, &plain) != BA_OK || heads < 1 || heads % cache->heads || tokens < 1 || requests < 0 || width < 0) return 0;
    return paged_tree_attention_workspace(cache->heads, heads / cache->heads, cache->dim, tokens, requests, width, cache->page);
}

__attribute__((visibility("default"))) int ba_paged_tree_attention(const ba_paged_cache *cache, int dtype, const void *q, int64_t q_head_stride,
                                                                   int64_t q_row_stride, int64_t heads, int64_t tokens, const int32_t *table,
                                                                   int64_t table_stride, int64_t width, const int64_t *lens,
                                                                   const int64_t *accum, int64_t requests, const int64_t *mask,
                                                                   int64_t mask_stride, int64_t words, int64_t window, float scale, void *out,
                                                                   int64_t out_head_stride, int64_t out_row_stride, int32_t *counters,
                                                                   void *workspace, size_t workspace_bytes, ba_stream_t stream) {
    ba_paged_cache plain;
    const int st = check_cache(cache, &plain);
    if (st != BA_OK) return st;
    cache = &plain;
    if (dtype != BA_F16 && dtype != BA_BF16) return BA_ERR_UNSUPPORTED;
    if (cache->dtype != BA_F8_E4M3 && cache->dtype != dtype) return BA_ERR_UNSUPPORTED;
    if (heads < 1 || heads % cache->heads || tokens < 0 || requests < 0 || width < 0 || window < 0 || table_stride < 0) return BA_ERR_INVALID_ARG;
    if (bad_stride(q_head_stride) || bad_stride(q_row_stride) || bad_stride(out_head_stride) || bad_stride(out_row_stride))
        return BA_ERR_INVALID_ARG;
    if (mask && (words < 1 || bad_stride(mask_stride) || (tokens > 1 && mask_stride < words && mask_stride != 0))) return BA_ERR_INVALID_ARG;
    if (tokens == 0) return BA_OK;
    if (!q || !out || !accum || !counters || (requests > 0 && (!lens || (width > 0 && !table)))) return BA_ERR_INVALID_ARG;
    if (requests > 1 && width > 0 && table_stride < width && table_stride != 0) return BA_ERR_INVALID_ARG;   // (0: a row for all, only read)
    if (heads >= (1 << 20) || tokens >= kTokenLimit / heads || requests >= kTokenLimit / heads || width >= kTokenLimit ||
        width * cache->page >= kTokenLimit || (mask && words >= kTokenLimit / 64))
        return BA_ERR_UNSUPPORTED;
    const size_t need = ba_paged_tree_attention_workspace(cache, heads, tokens, requests, width);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) return BA_ERR_WORKSPACE;
    PagedTreeAttentionArgs a{};
    a.k = array_of(cache, false); a.v = array_of(cache, true);
    a.q = (const char *)q; a.out = (char *)out; a.table = table; a.lens = lens; a.accum = accum; a.mask = mask;
    a.q_head_bytes = 2 * q_head_stride; a.q_row_bytes = 2 * q_row_stride;
    a.out_head_bytes = 2 * out_head_stride; a.out_row_bytes = 2 * out_row_stride;
    a.table_stride = table_stride; a.mask_stride = mask_stride; a.tokens = tokens;
    a.requests = (int32_t)requests; a.heads = (int32_t)cache->heads; a.group = (int32_t)(heads / cache->heads);
    a.dim = (int32_t)cache->dim; a.pages = (int32_t)cache->pages; a.width = (int32_t)width; a.words = mask ? (int32_t)words : 0;
    a.window = (int32_t)std::min<int64_t>(window, kTokenLimit - 1);
    a.scale = scale; a.page = PageDiv::of((uint32_t)cache->page);
    return launch_paged_tree_attention(a, dtype, cache->dtype, counters, workspace, (hipStream_t)stream);
}

__attribute__((visibility("default"))) int ba_paged_keep(const ba_paged_cache *cache, const int32_t *table, int64_t table_stride, int64_t width,
                                                         const int64_t *lens, const int64_t *path, int64_t path_stride, int64_t requests,
                                                         int64_t depth, int64_t *lens_out, ba_stream_t stream) {
    ba_paged_cache plain;
    const int st = check_cache(cache, &plain, true);
    if (st != BA_OK) return st;
    cache = &plain;
    if (requests < 0 || depth < 0 || width < 0 || table_stride < 0 || bad_stride(path_stride)) return BA_ERR_INVALID_ARG;
    if (requests == 0) return BA_OK;
    if (!lens || !lens_out || (depth > 0 && !path) || (width > 0 && !table)) return BA_ERR_INVALID_ARG;
    if (requests > 1 && ((width > 0 && table_stride < width) || (depth > 0 && path_stride < depth && path_stride != 0))) return BA_ERR_INVALID_ARG;
    if (requests >= kTokenLimit || depth >= kTokenLimit || width >= kTokenLimit || width * cache->page >= kTokenLimit) return BA_ERR_UNSUPPORTED;
    PagedKeepArgs a{};
    a.arrays[0] = array_of(cache, false); a.arrays[1] = array_of(cache, true);
    a.table = table; a.lens = lens; a.path = path; a.lens_out = lens_out;
    a.table_stride = table_stride; a.path_stride = path_stride;
    a.requests = (int32_t)requests; a.heads = (int32_t)cache->heads; a.pages = (int32_t)cache->pages; a.width = (int32_t)width;
    a.depth = (int32_t)depth; a.row_bytes = (int32_t)cache->dim * elem_bytes(cache->dtype); a.page = PageDiv::of((uint32_t)cache->page);
    return launch_paged_keep(a, (hipStream_t)stream);
}

__attribute__((visibility("default"))) size_t ba_paged_fork_workspace(int64_t requests, int64_t pages) {
    if (requests < 0 || requests > BA_PAGED_FORK_ROWS || pages < 0 || pages >= kTokenLimit) return 0;
    return paged_fork_workspace(requests, pages);
}

__attribute__((visibility("default"))) int ba_paged_fork(const int32_t *table, int64_t table_stride, int64_t width, int32_t *free_pages, int64_t pool,
                                                         const int64_t *state_in, const int32_t *shares, int64_t pages, const int64_t *lens,
                                                         const int64_t *origin, int64_t requests, int64_t page, int32_t *table_out,
                                                         int64_t table_out_stride, int64_t *lens_out, int64_t *state_out, int32_t *shares_out,
                                                         int32_t *source, int32_t *target, void *workspace, size_t workspace_bytes,
                                                         ba_stream_t stream) {
    if (requests < 0 || page < 1 || width < 0 || pool < 0 || pages < 0 || table_stride < 0 || table_out_stride < 0) return BA_ERR_INVALID_ARG;
    if (!state_in || !state_out || (pool > 0 && !free_pages) || (pages > 0 && (!shares || !shares_out))) return BA_ERR_INVALID_ARG;
    if (requests > 0 && (!lens || !origin || !lens_out || !source || !target || (width > 0 && (!table || !table_out)))) return BA_ERR_INVALID_ARG;
    if (requests > 1 && width > 0 && (table_stride < width || table_out_stride < width)) return BA_ERR_INVALID_ARG;
    if (requests > BA_PAGED_FORK_ROWS || width >= kTokenLimit || page >= kTokenLimit || pool >= kTokenLimit || pages >= kTokenLimit ||
        width * page >= kTokenLimit)
        return BA_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < ba_paged_fork_workspace(requests, pages) || ((uintptr_t)workspace & 255)) return BA_ERR_WORKSPACE;
    const PagedForkArgs a{table, shares, free_pages, table_out, shares_out, source, target, state_in, lens, origin, lens_out, state_out,
                          table_stride, table_out_stride, pool, (int32_t)requests, (int32_t)width, (int32_t)pages, PageDiv::of((uint32_t)page),
                          PageDiv::of((uint32_t)std::max<int64_t>(1, width))};
    return launch_paged_fork(a, workspace, (hipStream_t)stream);
}

__attribute__((visibility("default"))) int ba_paged_copy(const ba_paged_cache *cache, const int32_t *source, const int32_t *target, int64_t copies,
                                                         ba_stream_t stream) {
    ba_paged_cache plain;
    const int st = check_cache(cache, &plain, true);
    if (st != BA_OK) return st;
    cache = &plain;
    if (copies < 0) return BA_ERR_INVALID_ARG;
    const int64_t row = cache->dim * elem_bytes(cache->dtype);
    if (copies >= kTokenLimit || cache->page >= kTokenLimit / ((row + 15) / 16) / cache->heads) return BA_ERR_UNSUPPORTED;
    if (copies == 0 || cache->pages == 0) return BA_OK;
    if (!source || !target) return BA_ERR_INVALID_ARG;
    PagedCopyArgs a{};
    a.source = source; a.target = target; a.copies = copies; a.pages = (int32_t)cache->pages;
    return launch_paged_copy(a, {array_of(cache, false), array_of(cache, true)}, cache->heads, cache->page, row, (hipStream_t)stream);
}

}  // extern "C"
