// Attention of one new query per request over a paged key-value cache.
//
// out[h][r] = sum_t softmax_t(scale q[h][r] . K[t]) V[t] over the request's tokens t.  Every key and value is read once and
// takes part in 4 x group operations a byte pair, so memory traffic is the floor; what the kernel is built for is bytes in
// flight on every compute unit, whatever the lengths are.
//
// Split.  A unit is a request and up to 32 query heads that share a key head.  Its tokens are cut into tiles of 32, and
// the tiles of all units, in order, are dealt out to the workgroups in equal shares (the lengths are on the GPU only, so
// every workgroup adds them up itself).  A workgroup goes through its share unit by unit, its four wavefronts taking every
// fourth tile each; at the end of a unit their results are joined in LDS.  A unit that lies in one share is done
// then; for others each workgroup leaves its maximum, sum and fp32 accumulators in memory.  Where units have few parts, each
// counts itself in and the last one there joins them all, in the order of the tokens whoever it is; else a second kernel does.
//
// One tile; nothing of the cache passes through LDS.  With lane = 16 g + 4 q + c:
//   Scores, S[token][head] = K Q^T on the 16 x 16 x 32 matrix instruction, tokens as rows.
//     16-bit caches: a lane loads 16 bytes of tokens lane % 16 and 16 + lane % 16, which is what the instruction wants.
//     8-bit caches: so loaded every lane is a memory access of its own for few bytes, and every line is asked for twice.
//     Instead load j gives the lane piece 4 g + c of token 4 q + j, four lanes 32 bytes in a row.  Multiplied with piece 4 g + c'
//     of the queries, for c' = 0 .. 3, the rows 4 q + c of the result are right where c = c', and those lie in register c
//     of the lanes that hold the rows of q: the score is the sum of register c' of product c'.  Four times the products:
//     96 requests of up to 8192 tokens, 128 dimensions 165 us against 191; in 16 bits, 128 requests of up to 16384, 603
//     against 588, so there it is not done.
//   A lane then holds the scores of tokens 4 g + j of both halves of the tile for head lane % 16: packed to 16 bits these
//   are, as they are, its operand of the second product if that runs over the tokens in the order (half, g, j).
//   Values, O[d][head] = V^T P.  A lane loads a piece of its eight tokens, sixteen lanes a row, and turns the small matrix in
//   registers: the operand of dimension j is made of the j-th halves of its eight rows.
//   The next tile's keys are asked for as soon as the scores have used this one's, its values behind the second product, and the
//   page numbers of the tile after that before both: loads come back in order.
//
// Bound and figures.  Loads that pass the caches reach 7.05 TB/s here, others 6.2.  128 requests of 1 to 16384 tokens, 32 query
// heads on 8, 128 dimensions, bf16 (3.8 GB): 582 us, 6.6 TB/s; 64 requests of up to 4096 (500 MB): 92 us, 5.4 TB/s, of which
// about 12 us do not depend on the lengths (launch, adding up the lengths, first loads, joining).  8-bit caches are bound by
// instructions as much as by memory: 96 requests of up to 8192 tokens (876 MB) 164 us, 5.3 TB/s, and about the same time at 64 dimensions.
#pragma once
#include <algorithm>
#include <type_traits>

#include "ba_device.hpp"
#include "ba_gemm_common.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kPagedWaves = 4;
constexpr int kPagedThreads = 64 * kPagedWaves;
constexpr int kPagedTile = 32;               // tokens
constexpr int kPagedHeads = 16;              // query heads of an operand of the matrix instruction; a unit has one or two such sets
constexpr int kPagedShare = kPagedWaves;     // tiles of a workgroup at least, one a wavefront, unless units are shorter
constexpr int kPagedFewParts = 8;            // parts of a unit, on the average, up to which the kernel itself joins them
constexpr int kPagedJoins = 512;             // workgroups of the joining kernel, where it has a choice
constexpr int kPagedWhole = 8;               // units of up to so many tiles are not split between workgroups

// Probabilities are scaled by a power of two that keeps those of 2^-39 (and not 2^-24) of the largest apart from
// zero in fp16; it is in the sums as well and drops out.
template <int DT> constexpr float kLift = DT == 0 ? 14.f : 0.f;

// Workgroups of a compute unit, by the registers that the tiles in flight and the results take.  (One or two less: 128 dimensions
// 94 -> 97 us for 64 requests of up to 4096 tokens; one more, 8-bit, 167 -> 198; 256 dimensions in 16 bits at two, with registers in
// memory, 244 against 183.)
// `any`: rows at any address, whose addresses and shifting take more (64 requests of up to 4096 tokens, 100 dimensions 140 us,
// with a workgroup more 169; but 8-bit, 96 of up to 8192, 276 us with three, 282 with two, and 200 dimensions 437 with two, 504 with one).
constexpr int resident_groups(int dim_class, bool f8, int sets, bool any) {
    if (any)
        return dim_class == 64 ? (sets == 2 ? 2 : 3) : dim_class == 128 ? (f8 && sets == 1 ? 3 : 2) : f8 && sets == 1 ? 2 : 1;
    return dim_class == 64 ? (sets == 2 ? 3 : 4) : dim_class == 128 ? (sets == 2 ? 2 : 3) : f8 && sets == 1 ? 2 : 1;
}

struct alignas(8) PagedPart {                // what a workgroup leaves for a unit that others work on too
    float m, l;
};
// A unit of which several workgroups did a part each: the one that has its first tile, how many they are (0: not split).
struct Left {
    int32_t begins, parts, request, h, q0, rows;
};

struct PagedWork {
    int32_t *counters;                       // [groups]: how many have left their part of the unit begun by a workgroup; 0 between calls
    Left *split;                             // not NULL: instead of counting, one entry a unit for the joining kernel
    // Brings what follows to a multiple of 32 bytes in the kernel's arguments.  Else the compiler fetches it in pieces with what is before,
    // moves whole pieces to and from vector registers (367 moves for 144), and 64 dimensions take 64 us for 60.
    int64_t pad;
    PagedPart *parts;                        // [2 * groups][rows]
    float *sums;                             // [2 * groups][rows][pitch]
    int32_t groups, tiles_a_head, rows, pitch;     // tiles_a_head: units of a key head; rows: query heads of the largest unit
};

// Two e4m3 values (HI: the upper two bytes) as two 16-bit numbers: exact in either type.
template <int DT, bool HI> __device__ __forceinline__ uint32_t widen(uint32_t x) {
    if (DT == 0) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x, 1.f, HI));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, 1.f, HI));
}

// A probability as two 16-bit terms, the first for two of them, rounded down.  The error is 2^-16 of the probability or less.
// Down, because in fp16 the lifted probability of the largest score is 2^16, past the type, where scores are so large (2^25 and
// more) that subtracting the lift rounds, and because 16-bit values may be infinite, where a negative term would make NaN of an
// infinity.  A term of 0 would as well: there the second one is the type's smallest (bf16: smallest normal) number at least,
// unless the probability itself is less.  (128 requests of up to 16384 tokens 582 us with and without that.)
template <int DT> __device__ __forceinline__ uint32_t first_term(float p0, float p1) {
    if (DT == 0) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, p1), __builtin_bit_cast(uint32_t, p0), 0x07060302u);
}
template <int DT, bool F8> __device__ __forceinline__ float second_term(float p, float first) {
    return F8 ? p - first : __builtin_amdgcn_fmed3f(p - first, DT == 0 ? 0x1p-24f : 0x1p-126f, p);
}

// Dimensions d .. d + 3 of a result, as far as there are `dim`.
template <int DT> __device__ __forceinline__ void store_result(char *row, int d, int dim, f32x4 x) {
    u16_any *const p = (u16_any *)row + d;
    if (d + 4 <= dim) {
        *(u32x2_any *)p = u32x2_any{Elem<DT>::pack2(x[0], x[1]), Elem<DT>::pack2(x[2], x[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (d + i < dim) p[i] = Elem<DT>::from_float(x[i]);
    }
}

// What is known of the rows: at multiples of 16 bytes they fill the registers (64, 128, 256) or are whole pieces (16 bytes of
// a key); at any address they have 16 bytes or more, or fewer.
enum Shape { kFull, kPieces, kAny, kShort };
// What is known of the pages: whole halves of tiles, whole groups of four tokens, nothing.
enum Pages { kHalves, kFours, kTokens };

// The matrix product of part x of a load of a key (rows) with the same dimensions of the queries (columns).
template <int DT, bool F8, int E, int N> __device__ __forceinline__ f32x4 product(const uint32_t (&k)[N], int x, u32x4 q, f32x4 c) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (F8) {
#pragma unroll
        for (int i = 0; i < (E < 8 ? 1 : 2); ++i) { w[2 * i] = widen<DT, false>(k[2 * x + i]); w[2 * i + 1] = widen<DT, true>(k[2 * x + i]); }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = k[i];
    }
    if constexpr (E < 8) {                   // four dimensions a lane
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        const u32x2 ka = {w[0], w[1]}, qa = {q[0], q[1]};
        if constexpr (DT == 0) return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, ka), __builtin_bit_cast(f16x4, qa), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, ka), __builtin_bit_cast(s16x4, qa), c, 0, 0, 0);
    }
    return Elem<DT>::mfma(u32x4{w[0], w[1], w[2], w[3]}, q, c);
}

// Whether keys are loaded in whole lines (see above; rows at any address take 509 us that way, 276 without).
template <bool F8, Shape SHAPE> constexpr bool quad_keys = SHAPE != kAny && SHAPE != kShort && F8;

// kAny: the piece of a row that its end cuts off is loaded from so many bytes before (nothing past the row is read), and brought
// into place, zeros behind, when it is used.  `past` may be the whole piece and more.
template <int N> __device__ __forceinline__ void shift_down(uint32_t (&x)[N], int past) {
    if constexpr (N == 4) {
        const bool two = past & 8;
        x[0] = two ? x[2] : x[0]; x[1] = two ? x[3] : x[1]; x[2] = two ? 0u : x[2]; x[3] = two ? 0u : x[3];
    }
    if constexpr (N >= 2) {
        const bool one = past & 4;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = one ? (i + 1 < N ? x[(i + 1) % N] : 0u) : x[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = __builtin_amdgcn_alignbyte(i + 1 < N ? x[(i + 1) % N] : 0u, x[i], past & 3);
        x[i] = past >= 4 * N ? 0u : x[i];
    }
}

// Loads through a buffer descriptor: the base in scalar registers, one offset a lane, and what is past the range reads as zeros.
constexpr uint32_t kNowhere = 0x80000000u;
constexpr int kStreamAux = 2;                // past the caches, as load_stream
__device__ __forceinline__ __amdgpu_buffer_rsrc_t stream_resource(const char *base) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7fffffff, kRsrcFlags);
}
template <int N> __device__ __forceinline__ void buffer_stream(uint32_t (&x)[N], __amdgpu_buffer_rsrc_t res, uint32_t off, int soff) {
    static_assert(N == 1 || N == 2 || N == 4);
    soff = uniform(soff);                    // (in a vector register it would make the load a loop)
    if constexpr (N == 4) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(res, off, soff, kStreamAux);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = v[i];
    } else if constexpr (N == 2) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(res, off, soff, kStreamAux);
        x[0] = v[0]; x[1] = v[1];
    } else {
        x[0] = __builtin_amdgcn_raw_buffer_load_b32(res, off, soff, kStreamAux);
    }
}

// Barrier that waits for this wavefront's LDS traffic only (the loads of the next unit stay in flight).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct Visible {
    int first, len;                          // tokens first .. len - 1 are seen
    __device__ __forceinline__ int start() const { return first & ~(kPagedTile - 1); }
    // a request without tokens has one tile: its zeros are written by whoever gets it.  (The tile of the last token less that of the
    // first: lengths go up to 2^31 - 1.)
    __device__ __forceinline__ int tiles() const { return len > first ? (int)((uint32_t)(len - 1) / kPagedTile - (uint32_t)first / kPagedTile) + 1 : 1; }
};
__device__ __forceinline__ Visible visible(const PagedAttentionArgs &a, int r) {
    const int64_t room = (int64_t)a.width * a.page.d, length = a.lens[r];
    const int len = (int)(length < 0 ? 0 : length < room ? length : room);
    return {a.window && len > a.window ? len - a.window : 0, len};
}

// Position of the tile that the share of a workgroup begins with: request, unit of the request, tile of the unit.
struct Place {
    int request, unit, tile;
    Visible see;                             // of the request
    int64_t at;                              // number of the tile in the order of all
};

// x y / z, rounded down, z > 0: most often all of it fits 32 bits, where a division costs a fifth.
__device__ __forceinline__ int64_t scaled(int64_t x, int64_t y, int64_t z) {
    const int64_t p = x * y;
    return ((uint64_t)p | (uint64_t)z) >> 32 ? p / z : (int64_t)((uint32_t)p / (uint32_t)z);
}

// x y / z, rounded up.
__device__ __forceinline__ int64_t scaled_up(int64_t x, int64_t y, int64_t z) {
    const int64_t q = scaled(x, y, z);
    return q + (q * z < x * y);
}

// Parts travel between workgroups of different dies, whose caches know nothing of each other.  Fences for that write back and
// drop a whole cache (measured: 70 us more for a call of 100); stores and loads that go to where all meet by
// themselves only have to be in order, so a workgroup waits for its stores before it counts itself in.
constexpr int kSharedAux = 16;               // scope of the device
struct Shared {
    __amdgpu_buffer_rsrc_t parts, sums;
    int rows, pitch;
    __device__ __forceinline__ uint32_t part_at(int slot, int hd) const { return (uint32_t)((slot * rows + hd) * sizeof(PagedPart)); }
    __device__ __forceinline__ uint32_t sum_at(int slot, int hd, int d) const { return (uint32_t)((slot * rows + hd) * pitch + d) * 4u; }
    __device__ __forceinline__ void store(int slot, int hd, int d, f32x4 x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), sums, sum_at(slot, hd, d), 0, kSharedAux);
    }
    __device__ __forceinline__ void store(int slot, int hd, PagedPart x) const {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), parts, part_at(slot, hd), 0, kSharedAux);
    }
    __device__ __forceinline__ f32x4 sum(int slot, int hd, int d) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(sums, sum_at(slot, hd, d), 0, kSharedAux));
    }
    __device__ __forceinline__ PagedPart part(int slot, int hd) const {
        return __builtin_bit_cast(PagedPart, __builtin_amdgcn_raw_buffer_load_b64(parts, part_at(slot, hd), 0, kSharedAux));
    }
};
__device__ __forceinline__ Shared shared_of(const PagedWork &w) {
    return {__builtin_amdgcn_make_buffer_rsrc(w.parts, 0, 2 * w.groups * w.rows * (int)sizeof(PagedPart), kRsrcFlags),
            __builtin_amdgcn_make_buffer_rsrc(w.sums, 0, 2 * w.groups * w.rows * w.pitch * 4, kRsrcFlags), w.rows, w.pitch};
}

// Joins the parts of a unit for its query heads [hd0, hd1), by a whole workgroup.  DC / 4 threads read a row of partial sums;
// the rest of the threads take other heads, or every so manieth part of the same ones.
template <int DT, int DC>
__device__ __forceinline__ void join_parts(const PagedAttentionArgs &a, const PagedWork &w, const Left &u, int hd0, int hd1, float v_scale) {
    constexpr int kLanes = DC / 4, kRows = kPagedThreads / kLanes, kAhead = DC == 64 ? 8 : 16;
    __shared__ float rest_m[kRows], rest_l[kRows];
    __shared__ f32x4 rest_acc[kRows][kLanes];
    const int begins = u.begins, parts = u.parts, rows = min(u.rows, hd1);
    const Shared shared = shared_of(w);
    int heads = 1;
    while (heads < rows - hd0 && heads < kRows) heads *= 2;
    const int mine = (int)threadIdx.x / kLanes, d = 4 * ((int)threadIdx.x % kLanes), deep = kRows / heads, sub = mine / heads;
    for (int hd = hd0 + mine % heads; hd < hd0 + (rows - hd0 + heads - 1) / heads * heads; hd += heads) {
        float m = -INFINITY, l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (hd < rows && d < a.dim)
            for (int p0 = sub; p0 < parts; p0 += kAhead * deep) {
                PagedPart x[kAhead];
                f32x4 y[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int p = p0 + i * deep;
                    x[i] = {-INFINITY, 0.f};
                    y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (p < parts) {
                        const int slot = 2 * (begins + p) + (p == 0 ? 1 : 0);
                        x[i] = shared.part(slot, hd);
                        y[i] = shared.sum(slot, hd, d);
                    }
                }
                float top = m;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) top = fmaxf(top, x[i].m);
                const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m - base);
                l *= old;
                acc *= old;
                m = top;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const float f = __builtin_amdgcn_exp2f(x[i].m - base);
                    l += f * x[i].l;
                    acc += f * y[i];
                }
            }
        if (deep > 1) {
            rest_acc[mine][d / 4] = acc;
            if (d == 0) { rest_m[mine] = m; rest_l[mine] = l; }
            __syncthreads();
            float top = m;
            for (int i = 1; i < deep && sub == 0; ++i) top = fmaxf(top, rest_m[mine + i * heads]);
            const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m - base);
            l *= old;
            acc *= old;
            for (int i = 1; i < deep && sub == 0; ++i) {
                const float f = __builtin_amdgcn_exp2f(rest_m[mine + i * heads] - base);
                l += f * rest_l[mine + i * heads];
                acc += f * rest_acc[mine + i * heads][d / 4];
            }
        }
        if (deep > 1) __syncthreads();
        if (sub == 0 && hd < rows && d < a.dim)
            store_result<DT>(a.out + (u.q0 + hd) * a.out_head_bytes + u.request * a.out_row_bytes, d, a.dim, acc * (v_scale / l));
    }
}

// DC: dimensions that the registers hold (64, 128, 256).
template <int DT, bool F8, int DC, int SETS, Shape SHAPE, Pages PAGES>
__global__ void __launch_bounds__(kPagedThreads, resident_groups(DC, F8, SETS, SHAPE == kAny || SHAPE == kShort))
paged_attention_kernel(PagedAttentionArgs a, PagedWork w) {
    constexpr int EB = F8 ? 1 : 2;           // bytes of an element
    constexpr int PW = DC / 16;              // dimensions of a row that a lane holds
    constexpr int E = PW * EB < 16 ? PW : 16 / EB, N = E * EB / 4;      // those of one load, its dwords
    constexpr int L = PW / E;                // loads; load k of lane x of a row: dimensions 16 E k + E x ..
    constexpr bool QUAD = quad_keys<F8, SHAPE>;
    constexpr int PARTS = QUAD && E > 8 ? E / 8 : 1;           // matrix instructions that a load of a key feeds (for each c')
    constexpr int KR = QUAD ? 8 : 2, KL = QUAD ? L : DC * EB / 64, KN = QUAD ? N : 4;      // a lane's tokens of a tile, loads of each, dwords
    constexpr int QC = QUAD ? 4 : 1, QK = QUAD ? L * PARTS : DC / 32;                    // operands of the queries
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4, q4 = l16 >> 2, c4 = l16 & 3, wave = uniform((int)threadIdx.x >> 6);
    const int units = a.heads * w.tiles_a_head;

    extern __shared__ __attribute__((aligned(16))) float lds[];           // [waves][rows][DC + 4]
    __shared__ int64_t scan[kPagedWaves];
    __shared__ Place places[2];
    __shared__ float wave_m[kPagedWaves][SETS * kPagedHeads], wave_l[kPagedWaves][SETS * kPagedHeads];
    __shared__ Left left[2];
    __shared__ bool joins[2];
    int unfinished = 0;

    // ---- the share.  Thread i adds up the tiles of requests [i c, (i + 1) c).
    const int c = (a.requests + kPagedThreads - 1) / kPagedThreads, r0 = (int)threadIdx.x * c;
    const int r1 = min(a.requests, r0 + c);
    int64_t mine = 0;
    Visible front = {0, 0};
    for (int r = r0; r < r1; ++r) {
        const Visible v = visible(a, r);
        if (r == r0) front = v;
        mine += v.tiles();
    }
    int64_t upto = wave_inclusive_scan(mine);
    if (lane == 63) scan[wave] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int i = 0; i < kPagedWaves; ++i) {
        if (i < wave) upto += scan[i];
        total += scan[i];
    }
    total = uniform64(total) * units;
    // (a workgroup for every unit while there are enough: a request of 5 tokens, 14 key heads of 80, 8-bit 7.7 us,
    // four units to a workgroup 17.4)
    const int64_t groups = min((int64_t)w.groups, max((total + kPagedShare - 1) / kPagedShare, (int64_t)a.requests * units));
    const int64_t group = blockIdx.x;
    if (group >= groups) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int64_t at = scaled(group + k, total, groups);
        if (at >= total) {
            if (threadIdx.x == 0) places[k] = {a.requests, 0, 0, {0, 0}, total};
        } else if (at < upto * units && at >= (upto - mine) * units) {
            int64_t before = (upto - mine) * units;
            Visible see = front;
            int r = r0, n = see.tiles();
            while (at >= before + (int64_t)n * units) {
                before += (int64_t)n * units;
                see = visible(a, ++r);
                n = see.tiles();
            }
            int unit = (int)scaled(at - before, 1, n), tile = (int)((at - before) - (int64_t)unit * n);
            if (n <= kPagedWhole && tile) {                    // short units go where most of them lies
                at -= tile;
                if (2 * tile > n) {
                    at += n;
                    if (++unit == units) {
                        unit = 0;
                        if (++r < a.requests) see = visible(a, r);
                    }
                }
                tile = 0;
            }
            places[k] = {r, unit, tile, see, at};
        }
    }
    __syncthreads();
    // What a workgroup does of a unit: tiles [tile, last) of n.
    struct Unit {
        int request, unit, tile, last, n, first, len, start, h, q0, rows;
        int64_t at;                          // number of tile `tile` in the order of all
    };
    const int64_t end = uniform64(places[1].at);
    auto unit_of = [&](int request, int unit, int tile, int64_t at, Visible see) {
        Unit u;
        u.request = request; u.unit = unit; u.tile = tile; u.at = at;
        u.first = see.first; u.len = see.len; u.n = see.tiles(); u.start = see.start();
        u.last = (int)min((int64_t)u.n, tile + (end - at));
        u.h = unit / w.tiles_a_head;
        u.q0 = u.h * a.group + (unit - u.h * w.tiles_a_head) * w.rows;
        u.rows = min(w.rows, (u.h + 1) * a.group - u.q0);
        return u;
    };
    const Place place = places[0];
    if (place.at >= end) return;
    Unit cur = unit_of(uniform(place.request), uniform(place.unit), uniform(place.tile), uniform64(place.at),
                       {uniform(place.see.first), uniform(place.see.len)});

    // queries: of heads l16 and 16 + l16, in the order of dimensions in which the keys arrive
    u32x4 qf[SETS][QC][QK];
    auto load_queries = [&](const Unit &u) {
#pragma unroll
        for (int z = 0; z < SETS; ++z)
#pragma unroll
            for (int c = 0; c < QC; ++c)
#pragma unroll
                for (int k = 0; k < QK; ++k) {
                    constexpr int QN = QUAD && E < 8 ? 2 : 4;
                    const int d = QUAD ? 16 * E * (k / PARTS) + E * (4 * g + c) + 8 * (k % PARTS)
                                  : F8 ? 64 * (k / 2) + 16 * g + 8 * (k % 2) : 32 * k + 8 * g;
                    uint32_t x[QN] = {};
                    const int hd = kPagedHeads * z + l16;
                    const char *const p = a.q + (u.q0 + hd) * a.q_head_bytes + u.request * a.q_row_bytes + 2 * d;
                    if (hd < u.rows) {
                        if (SHAPE == kAny || SHAPE == kShort) load_part<QN>(x, p, 2 * (a.dim - d));
                        else if (SHAPE == kFull || d < a.dim) load_stream<QN>(x, p);
                    }
                    qf[z][c][k] = u32x4{x[0], x[1], x[QN - 2], x[QN - 1]};
                }
    };

    // Pages of a tile.  Tokens that are not seen may have no page (any more): a half, a group of four or a token
    // without any that is seen borrows the place of the nearest one with (so tiles past the unit's last may be asked for).
    // Page numbers outside the cache become page 0 and poison the result.
    // kHalves: the pages of both halves, the same in all lanes; else lane i has that of the i-th group of four or token.
    struct Spot {
        int32_t page[PAGES == kHalves ? 2 : 1], line[PAGES == kHalves ? 2 : 1];      // (line: kHalves only)
    };
    bool poison = false;
    constexpr int low = PAGES == kHalves ? 15 : PAGES == kFours ? 3 : 0;
    auto borrowed = [&](const Unit &u, int t) { return min(max(t & ~low, u.first & ~low), (u.len - 1) & ~low) + (t & low); };
    // (Tiles are looked up ahead, past the last one too: with lengths up to 2^31 - 1 such a place may wrap round to below zero, where
    // it borrows that of the first token.)
    auto look_up = [&](const Unit &u, uint32_t t0) {
        Spot s;
        const int32_t *const row = a.table + u.request * a.table_stride;
        if (PAGES == kHalves) {
            typedef const __attribute__((address_space(4))) int32_t *Row;      // scalar loads
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t t = (uint32_t)borrowed(u, (int)(t0 + 16 * i)), c = a.page.div(t);
                s.page[i] = ((Row)(uintptr_t)row)[c];
                s.line[i] = (int)(t - c * a.page.d);
            }
        } else {
            s.page[0] = row[a.page.div((uint32_t)borrowed(u, (int)(t0 + (PAGES == kFours ? 4 * (lane & 7) : lane & 31))))];
        }
        return s;
    };
    // kHalves: the page numbers, once they are there.
    auto check = [&](Spot &s) {
        if (PAGES != kHalves) return;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s.page[i % 2] = uniform(s.page[i % 2]);
            const bool bad = (uint32_t)s.page[i % 2] >= (uint32_t)a.pages;
            poison |= bad;
            s.page[i % 2] = bad ? 0 : s.page[i % 2];
        }
    };
    // Where token t0 + i (kHalves: half i of the tile) lies in an array, from the first token of the head on.
    auto place_of = [&](const PagedArray &array, const Unit &u, const Spot &s, int t0, int i) {
        if (PAGES == kHalves)
            return (int64_t)((uint64_t)(uint32_t)s.page[i % 2] * (uint32_t)array.page_bytes + (uint32_t)(uniform(s.line[i % 2]) * array.token_bytes));
        const uint32_t t = (uint32_t)borrowed(u, t0 + i);
        const int32_t p = __shfl(s.page[0], PAGES == kFours ? i / 4 : i);
        const int32_t line = (int)(t - a.page.div(t) * a.page.d);
        const bool bad = (uint32_t)p >= (uint32_t)a.pages;
        poison |= bad;
        return (bad ? 0 : p) * array.page_bytes + (int64_t)line * array.token_bytes;
    };
    // The rows of a tile.  With kHalves and kFours through descriptors, whose range check reads pieces that are not there as zeros.
    uint32_t kx[KR][KL][KN], vx[8][L][N];
    auto may_miss = [](int k, int loads) { return SHAPE == kPieces && (DC == 64 || 2 * k + 1 >= loads); };      // (more than half of DC there are always)
    auto load_keys = [&](const Unit &u, const Spot &s, int t0) {
        constexpr int kNext = QUAD ? 16 * EB * E : 64;
        const int b = QUAD ? EB * E * (4 * g + c4) : 16 * g, row = EB * a.dim;
        const char *const base = a.k.base + u.h * a.k.head_bytes;
        if (SHAPE == kAny || SHAPE == kShort) {
            const char *p[KR];
#pragma unroll
            for (int i = 0; i < KR; ++i)
                p[i] = base + place_of(a.k, u, s, t0, PAGES == kHalves ? i : 16 * i + l16) + (PAGES == kHalves ? (uint32_t)(l16 * a.k.token_bytes) : 0u);
#pragma unroll
            for (int k = 0; k < KL; ++k)
#pragma unroll
                for (int i = 0; i < KR; ++i) {
                    if (SHAPE == kAny) load_stream<KN>(kx[i][k], p[i] + (uint32_t)min(b + kNext * k, row - 4 * KN));
                    else load_part<KN>(kx[i][k], p[i] + b + kNext * k, row - b - kNext * k);
                }
            return;
        }
        __amdgpu_buffer_rsrc_t res[2];
        uint32_t off[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t at = place_of(a.k, u, s, t0, PAGES == kHalves ? i : 16 * i + (QUAD ? 4 * q4 : l16));
            res[i] = stream_resource(PAGES == kHalves ? base + at : base);
            off[i] = b + (PAGES == kHalves ? (uint32_t)((QUAD ? 4 * q4 : l16) * a.k.token_bytes) : (uint32_t)at);
        }
#pragma unroll
        for (int k = 0; k < KL; ++k)
#pragma unroll
            for (int i = 0; i < KR; ++i) {
                const int half = QUAD ? i / 4 : i;
                buffer_stream<KN>(kx[i][k], res[half], may_miss(k, KL) && b + kNext * k >= row ? kNowhere : off[half] + kNext * k, QUAD ? i % 4 * a.k.token_bytes : 0);
            }
    };
    auto load_values = [&](const Unit &u, const Spot &s, int t0) {
        constexpr int kNext = 16 * EB * E;
        const int b = EB * E * l16, row = EB * a.dim;
        const char *const base = a.v.base + u.h * a.v.head_bytes;
        if (SHAPE == kAny || SHAPE == kShort) {
            const char *p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                p[i] = base + place_of(a.v, u, s, t0, PAGES == kHalves ? i / 4 : 16 * (i / 4) + 4 * g + i % 4) +
                       (PAGES == kHalves ? (uint32_t)((4 * g + i % 4) * a.v.token_bytes) : 0u);
#pragma unroll
            for (int k = 0; k < L; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (SHAPE == kAny) load_stream<N>(vx[i][k], p[i] + (uint32_t)min(b + kNext * k, row - 4 * N));
                    else load_part<N>(vx[i][k], p[i] + b + kNext * k, row - b - kNext * k);
                }
            return;
        }
        __amdgpu_buffer_rsrc_t res[2];
        uint32_t off[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t at = place_of(a.v, u, s, t0, PAGES == kHalves ? i : 16 * i + 4 * g);
            res[i] = stream_resource(PAGES == kHalves ? base + at : base);
            off[i] = b + (PAGES == kHalves ? (uint32_t)(4 * g * a.v.token_bytes) : (uint32_t)at);
        }
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                buffer_stream<N>(vx[i][k], res[i / 4], may_miss(k, L) && b + kNext * k >= row ? kNowhere : off[i / 4] + kNext * k, i % 4 * a.v.token_bytes);
    };
    // kAny: pieces that the rows' end cuts off, once they are there.
    auto settle_keys = [&]() {
        if (SHAPE != kAny) return;
        const int row = EB * a.dim;
#pragma unroll
        for (int k = 0; k < KL; ++k)
            if (64 * (k + 1) > row)
#pragma unroll
                for (int i = 0; i < KR; ++i) shift_down<KN>(kx[i][k], max(16 * g + 64 * k - (row - 4 * KN), 0));
    };
    auto settle_values = [&]() {
        if (SHAPE != kAny) return;
        constexpr int kNext = 16 * EB * E;
        const int row = EB * a.dim;
#pragma unroll
        for (int k = 0; k < L; ++k)
            if (kNext * (k + 1) > row)
#pragma unroll
                for (int i = 0; i < 8; ++i) shift_down<N>(vx[i][k], max(EB * E * l16 + kNext * k - (row - 4 * N), 0));
    };
    // The wavefront's first tile of a unit.  Loads come back in the order in which they were asked for, so page numbers are asked
    // for before the loads that others wait for: those of a tile two tiles ahead.
    constexpr int kStep = kPagedWaves * kPagedTile;
    Spot ahead;
    auto has_tile = [&](const Unit &u) { return u.tile + wave < u.last && u.len > u.first && a.pages > 0; };
    auto load_first = [&](const Unit &u) {
        load_queries(u);
        if (has_tile(u)) {
            const int t0 = u.start + (u.tile + wave) * kPagedTile;
            Spot s = look_up(u, t0);
            ahead = look_up(u, (uint32_t)t0 + kStep);
            check(s);
            __builtin_amdgcn_sched_barrier(0);
            load_keys(u, s, t0);
            __builtin_amdgcn_sched_barrier(0);
            load_values(u, s, t0);
        }
    };

    f32x4 o[SETS][PW];
    float m[SETS], l[SETS];
    // The tile that begins with token t0; MORE: the wavefront's next one of the unit follows, whose keys are asked for as soon
    // as the scores have used this one's, and its values likewise.
    auto attend = [&](const Unit &u, auto more, int t0, float to_log2) {
        constexpr bool MORE = decltype(more)::value;
        Spot after;
        if (MORE) after = look_up(u, (uint32_t)t0 + 2 * kStep);
        // ---- scores of tokens t0 + 16 i + 4 g + j
        settle_keys();
        f32x4 sc[SETS][2];
#pragma unroll
        for (int z = 0; z < SETS; ++z)
#pragma unroll
            for (int i = 0; i < KR; ++i) {
                if (QUAD) {
                    f32x4 s4[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        s4[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < QK; ++k) s4[c] = product<DT, F8, E>(kx[i][k / PARTS], k % PARTS, qf[z][c % QC][k], s4[c]);
                    }
                    sc[z][i / 4][i % 4] = ((s4[0][0] + s4[1][1]) + (s4[2][2] + s4[3][3])) * to_log2;
                } else {
                    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < QK; ++k) s = product<DT, F8, F8 ? 16 : 8>(kx[i][F8 ? k / 2 : k], F8 ? k % 2 : 0, qf[z][0][k], s);
                    sc[z][i % 2] = s * to_log2;
                }
            }
        if (MORE) {
            check(ahead);
            load_keys(u, ahead, t0 + kStep);
            __builtin_amdgcn_sched_barrier(0);
        }
        settle_values();
        if (t0 < u.first || (uint32_t)t0 + kPagedTile > (uint32_t)u.len) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
                const bool seen = t >= u.first && t < u.len;
#pragma unroll
                for (int z = 0; z < SETS; ++z) sc[z][i / 4][i % 4] = seen ? sc[z][i / 4][i % 4] : -INFINITY;
#pragma unroll
                for (int k = 0; k < L; ++k)
#pragma unroll
                    for (int x = 0; x < N; ++x) vx[i][k][x] = seen ? vx[i][k][x] : 0u;    // (a probability of 0 times what lies there may be NaN)
            }
        }
        // Probabilities in two 16-bit terms: one alone would cost as much accuracy as the rounding of the result, and the
        // matrix unit has time to spare.
        u32x4 hi[SETS], lo[SETS];
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            float top = fmaxf(fmaxf(fmaxf(sc[z][0][0], sc[z][0][1]), fmaxf(sc[z][0][2], sc[z][0][3])),
                              fmaxf(fmaxf(sc[z][1][0], sc[z][1][1]), fmaxf(sc[z][1][2], sc[z][1][3])));
            top = fmaxf(m[z], quad_column_max(top));
            const float base = (top == -INFINITY ? 0.f : top) - kLift<DT>;
            if (__any(top != m[z])) {
                const float shrink = __builtin_amdgcn_exp2f(m[z] - kLift<DT> - base);
                l[z] *= shrink;
#pragma unroll
                for (int j = 0; j < PW; ++j) o[z][j] *= shrink;
                m[z] = top;
            }
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(sc[z][i / 4][i % 4] - base);
                l[z] += p[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hi[z][i] = first_term<DT>(p[2 * i], p[2 * i + 1]);
                lo[z][i] = Elem<DT>::pack2(second_term<DT, F8>(p[2 * i], Elem<DT>::to_float((uint16_t)hi[z][i])),
                                           second_term<DT, F8>(p[2 * i + 1], Elem<DT>::to_float((uint16_t)(hi[z][i] >> 16))));
            }
        }
        // ---- values
#pragma unroll
        for (int j = 0; j < PW; ++j) {
            uint32_t f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = j / E, x = j % E;
                if (F8) {
                    // byte x of both rows next to each other, then widened together
                    const uint32_t both = __builtin_amdgcn_perm(vx[2 * i + 1][k][x / 4], vx[2 * i][k][x / 4], 0x0c0c0400u + (uint32_t)(x % 4) * 0x0101u);
                    f[i] = widen<DT, false>(both);
                } else {
                    f[i] = __builtin_amdgcn_perm(vx[2 * i + 1][k][x / 2], vx[2 * i][k][x / 2], x % 2 ? 0x07060302u : 0x05040100u);
                }
            }
            const u32x4 v = {f[0], f[1], f[2], f[3]};
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                o[z][j] = Elem<DT>::mfma(v, hi[z], o[z][j]);
                o[z][j] = Elem<DT>::mfma(v, lo[z], o[z][j]);
            }
        }
        if (MORE) {
            load_values(u, ahead, t0 + kStep);
            ahead = after;
        }
    };

    load_first(cur);
    for (;;) {
        const float to_log2 = a.scale * kLog2e * (F8 ? a.k.scale[cur.h] : 1.f);
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            m[z] = -INFINITY; l[z] = 0.f;
#pragma unroll
            for (int j = 0; j < PW; ++j) o[z][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (has_tile(cur)) {
            int s = cur.tile + wave, t0 = cur.start + s * kPagedTile;
            for (; s + kPagedWaves < cur.last; s += kPagedWaves, t0 += kStep) attend(cur, std::true_type{}, t0, to_log2);
            attend(cur, std::false_type{}, t0, to_log2);
        }
        if (__any(poison) || (a.pages == 0 && cur.len > cur.first))
#pragma unroll
            for (int z = 0; z < SETS; ++z) l[z] = NAN;
        poison = false;
        // the next unit's first tile is on its way while this one is finished
        Unit next = cur;
        const int64_t at = cur.at + (cur.last - cur.tile);
        if (at < end) {
            if (cur.unit + 1 < units) {
                next = unit_of(cur.request, cur.unit + 1, 0, at, {cur.first, cur.len});
            } else {
                const Visible v = visible(a, cur.request + 1);
                next = unit_of(cur.request + 1, 0, 0, at, {uniform(v.first), uniform(v.len)});
            }
            load_first(next);
        }

        // ---- join the wavefronts: lane (g, l16) has dimensions 16 E k + E (4 g + i) + x of heads l16 and 16 + l16, j = E k + x
        constexpr int pitch = DC + 4;
        const int busy = min(cur.last - cur.tile, kPagedWaves);
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            const int hd = kPagedHeads * z + l16;
            l[z] = quad_column_sum(l[z]);
            if (wave < busy) {
                if (g == 0) { wave_m[wave][hd] = m[z]; wave_l[wave][hd] = l[z]; }
                if (hd < cur.rows) {
                    float *const mineo = lds + (wave * w.rows + hd) * pitch;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < PW; j += 4) {
                            const int d = 16 * E * (j / E) + E * (4 * g + i) + j % E;
                            if (SHAPE == kFull || d < a.dim) *(f32x4 *)(mineo + d) = f32x4{o[z][j][i], o[z][j + 1][i], o[z][j + 2][i], o[z][j + 3][i]};
                        }
                }
            }
        }
        lds_barrier();
        const bool begun = cur.tile == 0, done = cur.last == cur.n, whole = begun && done;
        const int slot = 2 * (int)group + (begun ? 1 : 0);
        for (int x = 4 * (int)threadIdx.x; x < cur.rows * DC; x += 4 * kPagedThreads) {
            const int hd = x / DC, d = x % DC;
            if (d >= a.dim) continue;
            float top = -INFINITY, sum = 0.f;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            for (int i = 0; i < busy; ++i) top = fmaxf(top, wave_m[i][hd]);
            const float base = top == -INFINITY ? 0.f : top;
            for (int i = 0; i < busy; ++i) {
                const float f = __builtin_amdgcn_exp2f(wave_m[i][hd] - base);
                sum += f * wave_l[i][hd];
                acc += f * *(const f32x4 *)(lds + (i * w.rows + hd) * pitch + d);
            }
            if (whole) {
                const float f = cur.len > cur.first ? (F8 ? a.v.scale[cur.h] : 1.f) / sum : 0.f;
                if (cur.len <= cur.first) acc = f32x4{0.f, 0.f, 0.f, 0.f};
                store_result<DT>(a.out + (cur.q0 + hd) * a.out_head_bytes + cur.request * a.out_row_bytes, d, a.dim, acc * f);
            } else {
                const Shared shared = shared_of(w);
                shared.store(slot, hd, d, acc);
                if (d == 0) shared.store(slot, hd, PagedPart{top, sum});
            }
        }
        // the workgroups that have the unit's first and last tile
        Left u = {0, 0, cur.request, cur.h, cur.q0, cur.rows};
        if (!whole) {
            const int64_t from = cur.at - cur.tile;
            u.begins = begun ? (int)group : (int)scaled_up(from + 1, groups, total) - 1;
            u.parts = (int)scaled_up(from + cur.n, groups, total) - u.begins;
        }
        if (w.split) {
            if (begun && threadIdx.x == 0) w.split[(int64_t)cur.request * units + cur.unit] = u;
        } else if (!whole) {
            if (threadIdx.x == 0) left[unfinished] = u;
            ++unfinished;                    // (the first unit of the share at most, and its last)
        }
        if (at >= end) break;
        lds_barrier();
        cur = next;
    }
    if (w.split || unfinished == 0) return;  // (with a list nothing is unfinished; said for the compiler, as the padding is)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 0; i < unfinished; ++i) {
            int32_t *const counter = w.counters + left[i].begins;
            joins[i] = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == left[i].parts - 1;
            if (joins[i]) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    __syncthreads();
    for (int i = 0; i < unfinished; ++i)
        if (joins[i]) join_parts<DT, DC>(a, w, left[i], 0, w.rows, F8 ? a.v.scale[left[i].h] : 1.f);
}

// The same as a kernel of its own: grid (entries of the list, query heads / `heads`).
template <int DT, int DC> __global__ void __launch_bounds__(kPagedThreads) paged_join_kernel(PagedAttentionArgs a, PagedWork w, int heads) {
    const Left u = w.split[blockIdx.x];
    const int hd = (int)blockIdx.y * heads;
    if (u.parts && hd < u.rows) join_parts<DT, DC>(a, w, u, hd, hd + heads, a.v.scale ? a.v.scale[u.h] : 1.f);
}

// ------------------------------------------------------------------ host
static inline int dim_class(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

template <int DT, bool F8, int DC, int SETS, Shape SHAPE, Pages PAGES>
static int launch_split(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream) {
    constexpr int kMostLds = kPagedWaves * SETS * kPagedHeads * (DC + 4) * (int)sizeof(float);
    if constexpr (kMostLds > 65536) {
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_attention_kernel<DT, F8, DC, SETS, SHAPE, PAGES>),
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
        if (attr != hipSuccess) return BA_ERR_LAUNCH;
    }
    const size_t lds = (size_t)kPagedWaves * w.rows * (DC + 4) * sizeof(float);
    paged_attention_kernel<DT, F8, DC, SETS, SHAPE, PAGES><<<w.groups, kPagedThreads, lds, stream>>>(a, w);
    if (w.split) {
        const int64_t entries = a.requests * (int64_t)a.heads * w.tiles_a_head;
        const int most = kPagedThreads / (DC / 4);
        int heads = 1;
        while (heads < most && heads < w.rows && entries * ((w.rows + heads - 1) / heads) > kPagedJoins) heads *= 2;
        paged_join_kernel<DT, DC><<<dim3((unsigned)entries, (unsigned)((w.rows + heads - 1) / heads)), kPagedThreads, 0, stream>>>(a, w, heads);
    }
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

// Bytes from the first element of an array to the end of the last one of a head.
static int64_t span(const PagedArray &x, const PagedAttentionArgs &a) {
    return (a.pages - 1) * x.page_bytes + ((int64_t)a.page.d - 1) * x.token_bytes + 2 * a.dim;
}

// Rows of whole pieces at addresses that are multiples of 16 go through descriptors: pages of 16, 32, ... tokens with one a page,
// pages of 4, 8, 12, 20, ... with one for all pages, whose offsets have 31 bits.  All else runs through the builds for any
// address, by page for pages of 16, 32, ..., else token by token; rows shorter than a load take byte by byte.
struct PagedBuild {
    Shape shape;                             // (kFull for kPieces as well)
    Pages pages;
};
static inline PagedBuild build_of(const PagedAttentionArgs &a, bool f8) {
    const uint64_t bits = (uint64_t)a.k.base | (uint64_t)a.v.base | (uint64_t)a.k.page_bytes | (uint64_t)a.v.page_bytes | (uint64_t)a.k.head_bytes |
                          (uint64_t)a.v.head_bytes | (uint64_t)a.k.token_bytes | (uint64_t)a.v.token_bytes;
    const bool pieces = bits % 16 == 0 && a.dim % (f8 ? 16 : 8) == 0;
    // (the page stride as 32 bits: one scalar multiplication less a tile and array)
    const bool near = ((uint64_t)a.k.page_bytes | (uint64_t)a.v.page_bytes) >> 32 == 0;
    if (near && a.page.d % 16 == 0 && a.dim * (f8 ? 1 : 2) >= 16) return {pieces ? kFull : kAny, kHalves};
    if (near && pieces && a.page.d % 4 == 0 && span(a.k, a) < kNowhere && span(a.v, a) < kNowhere) return {kFull, kFours};
    return {a.dim * (f8 ? 1 : 2) < 16 ? kShort : kAny, kTokens};
}

template <int DT, bool F8, int DC, int SETS> static int launch_class(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream) {
    const PagedBuild build = build_of(a, F8);
    if (build.shape == kFull && build.pages == kHalves)
        return a.dim == DC ? launch_split<DT, F8, DC, SETS, kFull, kHalves>(a, w, stream) : launch_split<DT, F8, DC, SETS, kPieces, kHalves>(a, w, stream);
    if (build.shape == kFull)
        return a.dim == DC ? launch_split<DT, F8, DC, SETS, kFull, kFours>(a, w, stream) : launch_split<DT, F8, DC, SETS, kPieces, kFours>(a, w, stream);
    if constexpr (DC == 64)
        if (build.shape == kShort) return launch_split<DT, F8, DC, SETS, kShort, kTokens>(a, w, stream);
    return build.pages == kHalves ? launch_split<DT, F8, DC, SETS, kAny, kHalves>(a, w, stream) : launch_split<DT, F8, DC, SETS, kAny, kTokens>(a, w, stream);
}

template <int DT, bool F8> int launch_paged_dtype(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream) {
    const bool two = w.rows > kPagedHeads;
    switch (dim_class(a.dim)) {
        case 64: return two ? launch_class<DT, F8, 64, 2>(a, w, stream) : launch_class<DT, F8, 64, 1>(a, w, stream);
        case 128: return two ? launch_class<DT, F8, 128, 2>(a, w, stream) : launch_class<DT, F8, 128, 1>(a, w, stream);
        default: return two ? launch_class<DT, F8, 256, 2>(a, w, stream) : launch_class<DT, F8, 256, 1>(a, w, stream);
    }
}

}  // namespace ba
