// Keys and values of new tokens into the pages of a cache, in 16 bits or rounded to 8 (e4m3).
#include <algorithm>

#include "ba_device.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kAppendThreads = 256;

// One element a thread, grid (elements of a token, tokens, keys or values).
template <int DT, bool F8> __global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(PagedAppendArgs a) {
    const int i = (int)(blockIdx.x * kAppendThreads + threadIdx.x), which = (int)blockIdx.z;
    const int h = i / a.dim, d = i - h * a.dim;
    if (h >= a.heads) return;
    for (int64_t t = blockIdx.y; t < a.tokens; t += gridDim.y) {
        const int64_t slot = a.slots[t];
        if (slot < 0 || slot >= a.places) continue;
        const uint32_t page = a.page.div((uint32_t)slot), row = (uint32_t)slot - page * a.page.d;
        const PagedArray &to = a.to[which];
        char *dst = to.base + page * to.page_bytes + h * to.head_bytes + (int64_t)row * to.token_bytes;
        const uint16_t x = ((const uint16_t *)(a.from[which] + h * a.from_head_bytes[which] + t * a.from_token_bytes[which]))[d];
        if (F8) {
            float y = Elem<DT>::to_float(x) / to.scale[h];
            y = y > 448.f ? 448.f : y < -448.f ? -448.f : y;      // (a NaN stays one)
            ((uint8_t *)dst)[d] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
        } else {
            ((uint16_t *)dst)[d] = x;
        }
    }
}

int launch_paged_append(const PagedAppendArgs &a, int dtype, int cache_dtype, hipStream_t stream) {
    const dim3 grid((unsigned)((a.heads * a.dim + kAppendThreads - 1) / kAppendThreads), (unsigned)std::min<int64_t>(a.tokens, 65535), 2);
    if (cache_dtype != BA_F8_E4M3) paged_append_kernel<0, false><<<grid, kAppendThreads, 0, stream>>>(a);
    else if (dtype == BA_F16) paged_append_kernel<0, true><<<grid, kAppendThreads, 0, stream>>>(a);
    else paged_append_kernel<1, true><<<grid, kAppendThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
