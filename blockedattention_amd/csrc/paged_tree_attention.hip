// Attention of drafted tokens over a paged cache.
#include <algorithm>

#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

// A wavefront takes a query head of a row; a lane four dimensions.
template <int DT, bool F8> __global__ void __launch_bounds__(64) paged_tree_attention_kernel(PagedTreeAttentionArgs a) {
    const int64_t row = blockIdx.x;
    const int head = (int)blockIdx.y, h = head / a.group, lane = lane_id();
    int r = -1;
    for (int i = 0; i < a.requests; ++i)
        if (a.accum[i] <= row && row < a.accum[i + 1]) r = i;
    char *const out = a.out + head * a.out_head_bytes + row * a.out_row_bytes;
    float q[4] = {}, acc[4] = {}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4; ++i)
        if (4 * lane + i < a.dim) q[i] = Elem<DT>::to_float(((const uint16_t *)(a.q + head * a.q_head_bytes + row * a.q_row_bytes))[4 * lane + i]);
    if (r >= 0) {
        const int64_t node = row - a.accum[r], n = a.accum[r + 1] - a.accum[r], len = a.lens[r], base = max(len - n, (int64_t)0);
        const int64_t room = (int64_t)a.width * a.page.d, end = min(len, room);
        auto sees = [&](int64_t j) {
            if (!a.mask) return j <= node;
            return j < 64 * (int64_t)a.words && ((a.mask[row * a.mask_stride + (j >> 6)] >> (j & 63)) & 1) != 0;
        };
        int64_t left = a.window ? a.window : INT64_MAX;
        for (int64_t t = end - 1; t >= 0 && left > 0; --t) {
            if (t >= base && !sees(t - base)) continue;
            --left;
            const uint32_t c = a.page.div((uint32_t)t);
            const int32_t p = a.table[r * a.table_stride + c];
            if ((uint32_t)p >= (uint32_t)a.pages) { l = NAN; break; }
            const int64_t line = t - (int64_t)c * a.page.d;
            const char *const k = a.k.base + p * a.k.page_bytes + h * a.k.head_bytes + line * a.k.token_bytes;
            const char *const v = a.v.base + p * a.v.page_bytes + h * a.v.head_bytes + line * a.v.token_bytes;
            auto value = [&](const char *x, int d) {
                if (F8) return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)x)[d], 0);
                return Elem<DT>::to_float(((const uint16_t *)x)[d]);
            };
            float s = 0.f, val[4] = {};
            for (int i = 0; i < 4; ++i)
                if (4 * lane + i < a.dim) { s += q[i] * value(k, 4 * lane + i); val[i] = value(v, 4 * lane + i); }
            s = wave_sum(s) * (a.scale * kLog2e * (F8 ? a.k.scale[h] : 1.f));
            const float top = fmaxf(m, s), f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top), p2 = __builtin_amdgcn_exp2f(s - top);
            l = l * f + p2;
            for (int i = 0; i < 4; ++i) acc[i] = acc[i] * f + p2 * val[i];
            m = top;
        }
    }
    const float f = l == 0.f ? 0.f : (F8 ? a.v.scale[h] : 1.f) / l;
    for (int i = 0; i < 4; ++i)
        if (4 * lane + i < a.dim) ((uint16_t *)out)[4 * lane + i] = Elem<DT>::from_float(acc[i] * f);
}

size_t paged_tree_attention_workspace(int64_t, int64_t, int64_t, int, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_paged_tree_attention(const PagedTreeAttentionArgs &a, int dtype, int cache_dtype, int32_t *, void *, hipStream_t stream) {
    const dim3 grid((unsigned)a.tokens, (unsigned)(a.heads * a.group));
    const bool f8 = cache_dtype == BA_F8_E4M3;
    if (dtype == BA_F16 && !f8) paged_tree_attention_kernel<0, false><<<grid, 64, 0, stream>>>(a);
    else if (dtype == BA_F16) paged_tree_attention_kernel<0, true><<<grid, 64, 0, stream>>>(a);
    else if (!f8) paged_tree_attention_kernel<1, false><<<grid, 64, 0, stream>>>(a);
    else paged_tree_attention_kernel<1, true><<<grid, 64, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
