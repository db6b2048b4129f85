// Keys and values of new tokens into the pages of a cache, in 16 bits or rounded to 8 (e4m3).  A copy: what it reads and
// writes is its floor.  A thread takes pieces of eight elements (16 bytes of the source); within a workgroup the
// pieces follow each other as they lie in the cache -- the tokens of a head or the heads of a token, whichever are closer --
// so that adjacent lanes write whole lines.  16384 tokens, 8 heads of 128, fp16 (134 MB) 22.8 us, 5.9 TB/s, bound by memory;
// 30011 tokens, 8 heads of 64, bf16 to e4m3 (92 MB) 22.3 us, 4.1 TB/s, bound by the quotients as well; 64 tokens 4.1 us, a launch.
// Rows that are not whole pieces end element by element: the same with dimension 100 (105 and 144 MB) 29 and 51 us.
#include <algorithm>

#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kAppendThreads = 256;
constexpr int kAppendPieces = 2;             // of a thread, their loads in flight together (with 4: 22.6 us for 22.1, with 8: 26.2)
constexpr int kPieceElems = 8;

struct AppendShape {
    PageDiv per_token, per_row;              // pieces of a token in one workgroup's order, of a row
    int32_t tokens, heads_inner;             // tokens of a workgroup; whether it takes all heads of them
};

// The fp32 quotient x / scale, limited to +-448; a NaN stays one.  With r the nearest number to 1 / scale and q = x r, one correction by the residual
// gives the nearest number to x / scale (Markstein's theorem; infinities and zeros stay as they are).  `plain`: a
// scale for which nothing on the way leaves fp32's range (what does has a result that rounds to 0 or 448 all the same);
// others are divided.  30 000 tokens of 8 x 64: 24 us with a division each, which costs
// twice the instructions.  It is rounded once more, to e4m3, as fp32 code that divides and converts does: a quotient that fp32
// makes a tie of goes to even, whichever side of it the exact one is.
__device__ __forceinline__ float scaled_down(float x, float scale, float r, bool plain) {
    float q = x * r;
    if (plain) {
        const float better = fmaf(fmaf(-q, scale, x), r, q);
        q = __builtin_amdgcn_classf(q, 0x198) ? better : q;      // finite and not 0 (which would lose its sign)
    } else {
        q = x / scale;
    }
    const float y = __builtin_amdgcn_fmed3f(q, -448.f, 448.f);
    return q == q ? y : q;
}

template <int DT, bool F8, bool WHOLE> __device__ __forceinline__ void store_piece(char *dst, const uint32_t (&x)[4], float scale, int left) {
    if (F8) {
        uint32_t y[2] = {0, 0};
        const float r = 1.f / scale, size = fabsf(scale);
        const bool plain = size > 0x1p-100f && size < 0x1p100f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = scaled_down(Elem<DT>::to_float((uint16_t)x[i]), scale, r, plain);
            const float hi = scaled_down(Elem<DT>::to_float((uint16_t)(x[i] >> 16)), scale, r, plain);
            if (i % 2) y[i / 2] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, (int)y[i / 2], true);
            else y[i / 2] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, (int)y[i / 2], false);
        }
        if (WHOLE || left >= kPieceElems) {
            *(u32x2_any *)dst = u32x2_any{y[0], y[1]};
        } else {
#pragma unroll
            for (int i = 0; i < kPieceElems - 1; ++i)
                if (i < left) ((uint8_t *)dst)[i] = (uint8_t)(y[i / 4] >> (8 * (i % 4)));
        }
    } else if (WHOLE || left >= kPieceElems) {
        *(u32x4_any *)dst = u32x4_any{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int i = 0; i < kPieceElems - 1; ++i)
            if (i < left) ((u16_any *)dst)[i] = (uint16_t)(x[i / 2] >> (16 * (i % 2)));
    }
}

// Grid (a row of token groups, heads or 1, rows of keys and values by turns): one row but for more groups than flat_grid() puts
// into one.  WHOLE: rows are whole pieces.
template <int DT, bool F8, bool WHOLE> __global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(PagedAppendArgs a, AppendShape s) {
    const int which = (int)blockIdx.z & 1;
    const int64_t t0 = ((int64_t)(blockIdx.z >> 1) * gridDim.x + blockIdx.x) * s.tokens;
    if (t0 >= a.tokens) return;
    const uint32_t most = (uint32_t)(min((int64_t)s.tokens, a.tokens - t0) * s.per_token.d);
    for (uint32_t i0 = threadIdx.x; i0 < most; i0 += kAppendPieces * kAppendThreads) {
        int64_t slot[kAppendPieces];
        int head[kAppendPieces], at[kAppendPieces];
        uint32_t x[kAppendPieces][4];
#pragma unroll
        for (int k = 0; k < kAppendPieces; ++k) {
            const uint32_t i = i0 + k * kAppendThreads;
            slot[k] = -1;
            if (i < most) {
                const uint32_t t = s.per_token.div(i), rest = i - t * s.per_token.d, row = s.per_row.div(rest);
                head[k] = s.heads_inner ? (int)row : (int)blockIdx.y;
                at[k] = (int)(rest - row * s.per_row.d) * kPieceElems;
                slot[k] = a.slots[t0 + t];
                const char *const src = a.from[which] + head[k] * a.from_head_bytes[which] + (t0 + t) * a.from_token_bytes[which] + 2 * at[k];
                if (WHOLE) load_stream<4>(x[k], src);
                else load_part<4>(x[k], src, 2 * (a.dim - at[k]));
            }
        }
        const PagedArray &to = a.to[which];
#pragma unroll
        for (int k = 0; k < kAppendPieces; ++k) {
            if (slot[k] < 0 || slot[k] >= a.places) continue;
            const uint32_t page = a.page.div((uint32_t)slot[k]), row = (uint32_t)slot[k] - page * a.page.d;
            char *const dst = to.base + page * to.page_bytes + head[k] * to.head_bytes + (int64_t)row * to.token_bytes + (F8 ? 1 : 2) * at[k];
            store_piece<DT, F8, WHOLE>(dst, x[k], F8 ? to.scale[head[k]] : 1.f, a.dim - at[k]);
        }
    }
}

template <int DT, bool F8> static void launch_append(const PagedAppendArgs &a, const AppendShape &s, dim3 grid, hipStream_t stream) {
    if (a.dim % kPieceElems == 0) paged_append_kernel<DT, F8, true><<<grid, kAppendThreads, 0, stream>>>(a, s);
    else paged_append_kernel<DT, F8, false><<<grid, kAppendThreads, 0, stream>>>(a, s);
}

int launch_paged_append(const PagedAppendArgs &a, int dtype, int cache_dtype, hipStream_t stream) {
    const uint32_t row = (uint32_t)(a.dim + kPieceElems - 1) / kPieceElems;
    AppendShape s;
    s.heads_inner = a.to[0].head_bytes < a.to[0].token_bytes || a.heads > 65535;
    s.per_row = PageDiv::of(row);
    s.per_token = PageDiv::of(s.heads_inner ? row * a.heads : row);
    // one round of pieces for every thread, or a token if that is more; fewer where the call is small and would otherwise
    // leave compute units idle
    int64_t tokens = std::max<int64_t>(1, kAppendPieces * kAppendThreads / s.per_token.d);
    const int64_t planes = s.heads_inner ? 2 : 2 * a.heads;
    while (tokens > 1 && a.tokens * planes < 256 * tokens) tokens /= 2;
    s.tokens = (int32_t)tokens;
    const dim3 flat = flat_grid((a.tokens + tokens - 1) / tokens);
    const dim3 grid(flat.x, s.heads_inner ? 1u : (unsigned)a.heads, 2 * flat.y);
    if (cache_dtype != BA_F8_E4M3) launch_append<0, false>(a, s, grid, stream);
    else if (dtype == BA_F16) launch_append<0, true>(a, s, grid, stream);
    else launch_append<1, true>(a, s, grid, stream);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

}  // namespace ba
