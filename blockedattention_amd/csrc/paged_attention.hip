// Attention of one new query per request over a paged key-value cache.
#include "ba_device.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / 64;

template <int DT, bool F8> __device__ __forceinline__ float cache_value(const char *p, int d) {
    if (F8) return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)p)[d], 0);
    return Elem<DT>::to_float(((const uint16_t *)p)[d]);
}

// One workgroup per request and query head, a wavefront takes every fourth token, a lane every 64th dimension.
template <int DT, bool F8> __global__ void __launch_bounds__(kPagedThreads) paged_attention_kernel(PagedAttentionArgs a) {
    const int r = (int)blockIdx.x, hq = (int)blockIdx.y, h = hq / a.group;
    const int lane = lane_id(), wave = (int)threadIdx.x / 64;
    const int64_t room = (int64_t)a.width * a.page.d, length = a.lens[r];
    const int len = (int)(length < 0 ? 0 : length < room ? length : room);
    const int first = a.window && len > a.window ? len - a.window : 0;
    const uint16_t *q = (const uint16_t *)(a.q + hq * a.q_head_bytes + r * a.q_row_bytes);
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    const float k_scale = a.scale * kLog2e * (F8 ? a.k.scale[h] : 1.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = lane + 64 * i < a.dim ? Elem<DT>::to_float(q[lane + 64 * i]) : 0.f;
    for (int t = first + wave; t < len; t += kPagedWaves) {
        const uint32_t c = a.page.div((uint32_t)t), row = (uint32_t)t - c * a.page.d;
        const int32_t page = a.table[r * a.table_stride + c];
        if (page < 0 || page >= a.pages) { l = NAN; continue; }
        const char *k = a.k.base + page * a.k.page_bytes + h * a.k.head_bytes + (int64_t)row * a.k.token_bytes;
        const char *v = a.v.base + page * a.v.page_bytes + h * a.v.head_bytes + (int64_t)row * a.v.token_bytes;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < a.dim) s += qv[i] * cache_value<DT, F8>(k, lane + 64 * i);
        s = wave_sum(s) * k_scale;
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
        const float shrink = exp2f(m - base), p = exp2f(s - base);
        l = l * shrink + p;
        m = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] *= shrink;
            if (lane + 64 * i < a.dim) o[i] += p * cache_value<DT, F8>(v, lane + 64 * i);
        }
    }
    __shared__ float sm[kPagedWaves], sl[kPagedWaves], so[kPagedWaves][256];
    if (lane == 0) { sm[wave] = m; sl[wave] = l; }
#pragma unroll
    for (int i = 0; i < 4; ++i) so[wave][lane + 64 * i] = o[i];
    __syncthreads();
    const int d = (int)threadIdx.x;
    if (d >= a.dim) return;
    float top = -INFINITY, sum = 0.f, total = 0.f;
    for (int w = 0; w < kPagedWaves; ++w) top = fmaxf(top, sm[w]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < kPagedWaves; ++w) {
        const float f = exp2f(sm[w] - base);
        sum += sl[w] * f;
        total += so[w][d] * f;
    }
    uint16_t *out = (uint16_t *)(a.out + hq * a.out_head_bytes + r * a.out_row_bytes);
    out[d] = Elem<DT>::from_float(len > first ? total * (F8 ? a.v.scale[h] : 1.f) / sum : 0.f);
}

size_t paged_attention_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_paged_attention(const PagedAttentionArgs &a, int dtype, int cache_dtype, void *, hipStream_t stream) {
    const dim3 grid((unsigned)a.requests, (unsigned)(a.heads * a.group));
    const bool f8 = cache_dtype == BA_F8_E4M3;
    if (dtype == BA_F16 && !f8) paged_attention_kernel<0, false><<<grid, kPagedThreads, 0, stream>>>(a);
    else if (dtype == BA_F16) paged_attention_kernel<0, true><<<grid, kPagedThreads, 0, stream>>>(a);
    else if (!f8) paged_attention_kernel<1, false><<<grid, kPagedThreads, 0, stream>>>(a);
    else paged_attention_kernel<1, true><<<grid, kPagedThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
