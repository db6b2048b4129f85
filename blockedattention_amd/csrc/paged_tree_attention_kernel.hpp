// Attention of the drafted tokens of each request over a paged key-value cache.
//
// out[h][i] = sum_t softmax_t(scale q[h][i] . K[t]) V[t] over the tokens t that row i sees: those before the draft, of the draft
// those with a bit in the row's mask, of these the last `window`.  A key takes part in one product for every row and query head that
// shares it, n x group of them: up to about a hundred rows the cache's bytes are the floor, beyond that the products.
#pragma once
#include <algorithm>
#include <type_traits>

#include "ba_device.hpp"
#include "ba_gemm_common.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char *LdsPtr;
typedef __attribute__((address_space(3))) s16x4 *LdsPiece;

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
constexpr int kTreeUnit = 3;                 // what a unit costs besides its tiles, in tiles: queries, first loads, joining, results
constexpr int kTreeShare = 5;                // of both, what a workgroup has at least, unless units are shorter
constexpr int kTreeWhole = 4;                // units of up to so many tiles are not split between workgroups
constexpr int kTreeFewParts = 8;             // parts of a unit, on the average, up to which the kernel itself joins them

// What is known when it is launched: what a workgroup's four wavefronts share out, and how much is in flight.
//   rows   wavefronts side by side over 32 rows each; the others take other tokens of the same tile
template <int DC, int WR> struct TreeTile {
    static constexpr int kRows = 32 * WR, kGroups = kTreeWaves / WR;     // rows of a unit, groups of wavefronts with the same tokens
    static constexpr int kMine = WR == 4 && DC < 256 ? 64 : 32;           // tokens of a wavefront in a tile
    static constexpr int kTokens = kMine * kGroups;
    static constexpr bool kAlone = WR == 1;                               // every wavefront loads its own tokens
    static constexpr int kBuffers = kAlone ? 1 : 2;
    // Bytes between rows in LDS: keys 16 more than whole lines of banks, so that sixteen rows' pieces lie side by side; values 64 more, so
    // that four rows' 64 bytes do.
    static constexpr int kPitchK = 2 * DC + 16, kPitchV = 2 * DC + 64;
    static constexpr int kStaged = kAlone ? kMine : kTokens;              // tokens that are loaded together
    static constexpr int kBuffer = kStaged * (kPitchK + kPitchV);
    static constexpr int kLds = (kAlone ? kTreeWaves : kBuffers) * kBuffer;
    static constexpr int kResident = DC == 64 ? 3 : DC == 128 ? 2 : 1;    // workgroups of a compute unit, by LDS and registers
};

struct alignas(8) TreePart {                 // what a workgroup leaves for a unit that others work on too
    float m, l;
};
// A unit of which several workgroups did a part each: the one that has its first tile, how many they are (0: not split).
struct TreeLeft {
    int32_t begins, parts, request, h, block;
};
struct TreeWork {
    int32_t *counters;                       // [groups]: how many have left their part of the unit begun by a workgroup; 0 between calls
    TreeLeft *left;                          // not NULL: instead of counting, an entry a workgroup for the joining kernel
    TreePart *parts;                         // [2 * groups][kRows]
    float *sums;                             // [2 * groups][kRows][pitch]
    PageDiv group;                           // query heads of a key head
    int32_t groups, pitch;
};

struct TreeArgs {
    PagedTreeAttentionArgs a;
    TreeWork w;
};
// The kernel's arguments, fetched again.  Held in scalar registers from the start they, and what is derived from them, are twice what there is; the
// compiler then moves whole groups of them to and from vector registers within the loop over tiles (ELSEWHERE us).
__device__ __forceinline__ const TreeArgs &tree_args() {
    auto p = (const __attribute__((address_space(4))) TreeArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const TreeArgs *)p;
}

// A request's draft.
struct Draft {
    int64_t node0;                           // number of the node of its first row
    int32_t row0, rows;                      // rows of q and out
    int32_t before, end;                     // tokens before the draft, tokens; as far as the table's row holds them
    int32_t blocks, start, tiles;            // of kRows rows; first token of the first tile that may be seen, tiles
};
// UNIFORM: r is the same in all lanes (scalar loads).
template <int DC, int WR, bool UNIFORM> __device__ __forceinline__ Draft draft_of(const PagedTreeAttentionArgs &a, int r) {
    typedef TreeTile<DC, WR> T;
    typedef typename std::conditional<UNIFORM, ConstI64, const int64_t *>::type Numbers;
    const Numbers accum = (Numbers)(uintptr_t)a.accum, lens = (Numbers)(uintptr_t)a.lens;
    constexpr int64_t kFar = int64_t(1) << 40;               // sums and lengths beyond any array
    const int64_t a0 = min(max(accum[r], -kFar), kFar), a1 = min(max(accum[r + 1], -kFar), kFar), length = min(max(lens[r], (int64_t)0), kFar);
    const int64_t n = max(a1 - a0, (int64_t)0), room = (int64_t)a.width * a.page.d;
    const int64_t first = min(max(a0, (int64_t)0), a.tokens), last = min(max(a1, first), a.tokens);
    Draft d;
    d.row0 = (int)first;
    d.rows = (int)(last - first);
    d.node0 = first - a0;
    d.end = (int)min(length, room);
    d.before = (int)min(max(length - n, (int64_t)0), (int64_t)d.end);
    d.blocks = (int)(((int64_t)d.rows * a.group + T::kRows - 1) / T::kRows);
    d.start = a.window && d.before > a.window ? (d.before - a.window) & ~(T::kTokens - 1) : 0;
    d.tiles = d.end > d.start ? (int)((uint32_t)(d.end - 1 - d.start) / T::kTokens) + 1 : 1;
    return d;
}

// x y / z, rounded down and up, for 0 <= x y < 2^62 and 0 < z: the quotient of fp64 numbers is off by one at most while it is below 2^51
// (a division of 64-bit integers is ten times the code).
__device__ __forceinline__ int64_t tree_ratio(int64_t x, int64_t y, int64_t z) {
    const int64_t p = x * y;
    int64_t q = (int64_t)((double)p / (double)z);
    q -= q * z > p ? 1 : 0;
    q += p - q * z >= z ? 1 : 0;
    return q;
}
__device__ __forceinline__ int64_t tree_ratio_up(int64_t x, int64_t y, int64_t z) { return tree_ratio(x, y, z) + (tree_ratio(x, y, z) * z < x * y); }

// Parts travel between workgroups of different dies: stores and loads that go to where all meet (fences would write back and
// drop whole caches), in order because a workgroup waits for its stores before it counts itself in.
constexpr int kTreeAux = 16;                 // scope of the device
template <int ROWS> struct TreeShared {
    __amdgpu_buffer_rsrc_t parts, sums;
    int pitch;
    __device__ __forceinline__ explicit TreeShared(const TreeWork &w) : pitch(w.pitch) {
        parts = __builtin_amdgcn_make_buffer_rsrc(w.parts, 0, 2 * w.groups * ROWS * (int)sizeof(TreePart), kRsrcFlags);
        sums = __builtin_amdgcn_make_buffer_rsrc(w.sums, 0, 2 * w.groups * ROWS * w.pitch * 4, kRsrcFlags);
    }
    __device__ __forceinline__ uint32_t sum_at(int slot, int row, int d) const { return (uint32_t)((slot * ROWS + row) * pitch + d) * 4u; }
    __device__ __forceinline__ void store(int slot, int row, int d, f32x4 x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), sums, sum_at(slot, row, d), 0, kTreeAux);
    }
    __device__ __forceinline__ void store(int slot, int row, TreePart x) const {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), parts, (uint32_t)((slot * ROWS + row) * sizeof(TreePart)), 0, kTreeAux);
    }
    __device__ __forceinline__ f32x4 sum(int slot, int row, int d) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(sums, sum_at(slot, row, d), 0, kTreeAux));
    }
    __device__ __forceinline__ TreePart part(int slot, int row) const {
        return __builtin_bit_cast(TreePart, __builtin_amdgcn_raw_buffer_load_b64(parts, (uint32_t)((slot * ROWS + row) * sizeof(TreePart)), 0, kTreeAux));
    }
};

// Dimensions d .. d + 3 of a result, as far as there are `dim`.
template <int DT> __device__ __forceinline__ void tree_store(char *row, int d, int dim, f32x4 x) {
    u16_any *const p = (u16_any *)row + d;
    if (d + 4 <= dim) {
        *(u32x2_any *)p = u32x2_any{Elem<DT>::pack2(x[0], x[1]), Elem<DT>::pack2(x[2], x[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (d + i < dim) p[i] = Elem<DT>::from_float(x[i]);
    }
}

// Row `x` of a unit: a row of q and out, and one of the query heads.
struct TreeRow {
    int node, head;                          // number within the request's rows, query head
    bool there;
};
__device__ __forceinline__ TreeRow tree_row(const PagedTreeAttentionArgs &a, const TreeWork &w, const Draft &d, int h, int64_t x) {
    TreeRow t;
    t.there = x < (int64_t)d.rows * a.group;
    const uint32_t y = t.there ? (uint32_t)x : 0u;
    t.node = (int)w.group.div(y);
    t.head = h * a.group + (int)(y - (uint32_t)t.node * w.group.d);
    return t;
}
template <int DT>
__device__ __forceinline__ void tree_result(const PagedTreeAttentionArgs &a, const Draft &d, const TreeRow &t, int dim0, f32x4 acc, float l, float v_scale) {
    if (dim0 >= a.dim) return;
    const float f = l == 0.f ? 0.f : v_scale / l;            // (rows that see nothing: zeros)
    if (l == 0.f) acc = f32x4{0.f, 0.f, 0.f, 0.f};
    tree_store<DT>(a.out + t.head * a.out_head_bytes + (int64_t)(d.row0 + t.node) * a.out_row_bytes, dim0, a.dim, acc * f);
}

// Joins the parts of a unit for its rows [row0, row1), by a whole workgroup: DC / 4 threads a row, kDeep rows of a thread and four parts of
// each on their way together (a load from where all dies meet takes some 2 us, however many there are).
template <int DT, int DC, int WR>
__device__ __forceinline__ void tree_join(const PagedTreeAttentionArgs &a, const TreeWork &w, const TreeLeft &u, int row0, int row1, float v_scale) {
    typedef TreeTile<DC, WR> T;
    constexpr int kLanes = DC / 4, kAtOnce = kTreeThreads / kLanes, kAhead = 4, kDeep = 4;
    const Draft d = draft_of<DC, WR, false>(a, u.request);
    const TreeShared<T::kRows> shared(w);
    const int dim0 = 4 * ((int)threadIdx.x % kLanes);
    const int rows = (int)min((int64_t)row1, (int64_t)d.rows * a.group - (int64_t)u.block * T::kRows);
#pragma nounroll
    for (int x0 = row0 + (int)threadIdx.x / kLanes; x0 < rows; x0 += kDeep * kAtOnce) {
        float m[kDeep], l[kDeep];
        f32x4 acc[kDeep];
#pragma unroll
        for (int z = 0; z < kDeep; ++z) {
            m[z] = -INFINITY;
            l[z] = 0.f;
            acc[z] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma nounroll
        for (int p0 = 0; p0 < u.parts; p0 += kAhead) {
            TreePart part[kDeep][kAhead];
            f32x4 sum[kDeep][kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int p = min(p0 + i, u.parts - 1), slot = 2 * (u.begins + p) + (p == 0 ? 1 : 0);
#pragma unroll
                for (int z = 0; z < kDeep; ++z) {
                    const int x = min(x0 + z * kAtOnce, rows - 1);       // (what is there already once more, and not used)
                    part[z][i] = shared.part(slot, x);
                    sum[z][i] = shared.sum(slot, x, min(dim0, w.pitch - 4));
                }
            }
#pragma unroll
            for (int z = 0; z < kDeep; ++z) {
                float top = m[z];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (p0 + i >= u.parts) part[z][i] = {-INFINITY, 0.f};
                    top = fmaxf(top, part[z][i].m);
                }
                const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m[z] - base);
                l[z] *= old;
                acc[z] *= old;
                m[z] = top;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const float f = __builtin_amdgcn_exp2f(part[z][i].m - base);
                    l[z] += f * part[z][i].l;
                    if (p0 + i < u.parts) acc[z] += f * sum[z][i];
                }
            }
        }
#pragma unroll
        for (int z = 0; z < kDeep; ++z)
            if (const int x = x0 + z * kAtOnce; x < rows) tree_result<DT>(a, d, tree_row(a, w, d, u.h, (int64_t)u.block * T::kRows + x), dim0, acc[z], l[z], v_scale);
    }
}

template <int DT> struct TreeElem;
template <> struct TreeElem<0> {
    static constexpr uint32_t kExponent = 0x7c00u;
    // Probabilities are lifted by a power of two, so that small ones stay apart from zero in fp16.  A maximum that is kept though a
    // larger one has come (by up to 2^7, see kTreeLag) leaves them below 2^13, and with scores so large that neighbouring fp32
    // numbers lie 2, 4 or 8 apart, where the difference rounds, below 2^15.
    static constexpr float kLift = 6.f;
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct TreeElem<1> {
    static constexpr uint32_t kExponent = 0x7f80u;
    static constexpr float kLift = 0.f;
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
constexpr float kTreeLag = 7.f;

// Two e4m3 values (HI: the upper two bytes) as two 16-bit numbers: exact in either type.
template <int DT, bool HI> __device__ __forceinline__ uint32_t tree_widen(uint32_t x) {
    if (DT == 0) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x, 1.f, HI));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, 1.f, HI));
}

// A 16-byte piece that was loaded from `past` bytes before its place (the row's end would have cut it off), brought into place.
__device__ __forceinline__ void tree_shift(uint32_t (&x)[4], int past) {
    const bool two = past & 8, one = past & 4;
    x[0] = two ? x[2] : x[0]; x[1] = two ? x[3] : x[1]; x[2] = two ? 0u : x[2]; x[3] = two ? 0u : x[3];
    x[0] = one ? x[1] : x[0]; x[1] = one ? x[2] : x[1]; x[2] = one ? x[3] : x[2]; x[3] = one ? 0u : x[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = past >= 16 ? 0u : __builtin_amdgcn_alignbyte(i < 3 ? x[i + 1] : 0u, x[i], past & 3);
}

// Greatest and sum over a lane and its partner, 32 lanes on.
__device__ __forceinline__ float pair_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Barrier that waits for this wavefront's LDS traffic only (loads of the next tile stay in flight).
__device__ __forceinline__ void tree_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int64_t shuffle64(int64_t v, int lane) {
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, lane), hi = (uint32_t)__shfl((int)(uint32_t)((uint64_t)v >> 32), lane);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// What a row sees of the tokens from a place on.
struct Sight {
    const int64_t *bits;                     // its row of the mask, or NULL
    int counted, chain, from;                // nodes that have bits; without a mask nodes that it sees; first token of the window
    bool there;
    // bit i: token t0 + i
    __device__ __forceinline__ uint64_t operator()(const Draft &d, int words, uint32_t t0) const {
        if (!there || t0 >= (uint32_t)d.end) return 0;
        const int j0 = (int)t0 - d.before, j = max(j0, 0);   // node of the first token; the first node
        uint64_t x = low_bits(chain - j);
        if (bits) {
            x = 0;
            if (j < counted) {
                x = (uint64_t)bits[j >> 6] >> (j & 63);
                if ((j & 63) && (j >> 6) + 1 < words) x |= (uint64_t)bits[(j >> 6) + 1] << (64 - (j & 63));
            }
        }
        const int before = j - j0;                           // tokens that lie before the draft
        x = before >= 64 ? ~0ull : x << before | low_bits(before);
        return x & low_bits(d.end - (int)t0) & ~low_bits(from - (int)t0);
    }
};
__device__ __forceinline__ Sight sight_of(const PagedTreeAttentionArgs &a, const Draft &d, const TreeRow &t, int from) {
    const int drafted = d.end - d.before;
    Sight s;
    s.bits = a.mask ? a.mask + (int64_t)(d.row0 + t.node) * a.mask_stride : nullptr;
    s.counted = a.mask ? (int)min((int64_t)drafted, 64 * (int64_t)a.words) : drafted;
    s.chain = (int)min(d.node0 + t.node + 1, (int64_t)drafted);
    s.from = from;
    s.there = t.there;
    return s;
}
// The first token that the window leaves of what a row sees.
__device__ __forceinline__ int window_from(const PagedTreeAttentionArgs &a, const Draft &d, const Sight &s) {
    int skip = s.chain - a.window, j = 0;                    // nodes that it sees no more
    if (s.bits) {
        skip = -a.window;
        for (j = 0; j < s.counted; j += 64) skip += __builtin_popcountll((uint64_t)s.bits[j >> 6] & low_bits(s.counted - j));
    }
    if (skip <= 0) return max(d.before + skip, 0);
    if (!s.bits) return d.before + skip;
    for (j = 0;; j += 64) {
        uint64_t x = (uint64_t)s.bits[j >> 6];
        const int n = __builtin_popcountll(x);
        if (n > skip) {
            for (; skip > 0; --skip) x &= x - 1;
            return d.before + j + __builtin_ctzll(x);
        }
        skip -= n;
    }
}

// What is known of the rows: whole 16-byte pieces at multiples of 16 bytes; at any address, of 16 bytes or more; shorter.
enum TreeRows { kTreePieces, kTreeAny, kTreeShort };

// DC: dimensions that the registers hold (64, 128, 256).
template <int DT, bool F8, int DC, int WR, TreeRows ROWS>
__global__ void __launch_bounds__(kTreeThreads, (TreeTile<DC, WR>::kResident)) paged_tree_attention_kernel(TreeArgs) {
    typedef TreeTile<DC, WR> T;
    typedef TreeElem<DT> E;
    constexpr int EB = F8 ? 1 : 2, kPieces = DC * EB / 16;   // bytes of an element, 16-byte pieces of a row
    constexpr int kLoaders = T::kAlone ? 64 : kTreeThreads, kAtOnce = kLoaders / kPieces, kPasses = T::kStaged / kAtOnce;
    constexpr int KS = DC / 16, DB = DC / 32, SUBS = T::kMine / 32;
    constexpr bool ANY = ROWS != kTreePieces, SHORT = ROWS == kTreeShort;
    static_assert(kLoaders % kPieces == 0 && T::kStaged % kAtOnce == 0 && T::kStaged <= 64);
    const int lane = lane_id(), l32 = lane & 31, half = lane >> 5, wave = uniform((int)threadIdx.x >> 6), wr = wave % WR, wt = wave / WR;

    extern __shared__ __attribute__((aligned(16))) char lds[];
    struct Place {
        int32_t request, unit, tile;
        int64_t at;
    };
    __shared__ Place places[2];
    __shared__ int64_t scan[2 * kTreeWaves], dealt[2];       // (dealt: tiles, workgroups that have some)
    __shared__ float wave_m[kTreeWaves][32], wave_l[kTreeWaves][32];
    __shared__ TreeLeft left[2];
    __shared__ int32_t joins[2], row_from[T::kRows], odd;    // odd: whether a part's hidden tiles have values that are not finite
    __shared__ int64_t spots[kTreeWaves][2][64];             // where the tokens that a wavefront looks after lie, of keys and values
    int unfinished = 0, group;

    {
    const PagedTreeAttentionArgs &a = tree_args().a;
    const TreeWork &w = tree_args().w;
    // ---- the share: tiles of all units in the order of requests, key heads, blocks of rows.  Thread i adds up requests [i c, (i + 1) c).
    const int c = (a.requests + kTreeThreads - 1) / kTreeThreads, r0 = (int)threadIdx.x * c, r1 = min(a.requests, r0 + c);
    int64_t mine = 0, units = 0;
    for (int r = r0; r < r1; ++r) {
        const Draft d = draft_of<DC, WR, false>(a, r);
        mine += (int64_t)a.heads * d.blocks * (d.tiles + kTreeUnit);
        units += (int64_t)a.heads * d.blocks;
    }
    int64_t upto = wave_inclusive_scan(mine);
    units = wave_inclusive_scan(units);
    if (lane == 63) { scan[wave] = upto; scan[kTreeWaves + wave] = units; }
    if (threadIdx.x == 0) odd = 0;
    __syncthreads();
    int64_t total = 0;
    units = 0;
#pragma unroll
    for (int i = 0; i < kTreeWaves; ++i) {
        if (i < wave) upto += scan[i];
        total += scan[i];
        units += scan[kTreeWaves + i];
    }
    total = uniform64(total);
    const int64_t groups = uniform64(min((int64_t)w.groups, max((total + kTreeShare - 1) / kTreeShare, units)));
    group = (int)blockIdx.x;
    if (w.left && threadIdx.x == 0) w.left[group].parts = 0;
    // rows of no request: zeros
    {
        const int64_t head = a.requests ? min(max(a.accum[0], (int64_t)0), a.tokens) : a.tokens;
        const int64_t tail = a.requests ? min(max(a.accum[a.requests], head), a.tokens) : a.tokens;
        for (int64_t i = group; i < head + a.tokens - tail; i += gridDim.x) {
            char *const out = a.out + (i < head ? i : tail + (i - head)) * a.out_row_bytes;
            for (int x = (int)threadIdx.x; x < a.heads * a.group * a.dim; x += kTreeThreads) {
                const int head_of = x / a.dim;
                *(u16_any *)(out + head_of * a.out_head_bytes + 2 * (x - head_of * a.dim)) = 0;
            }
        }
    }
    if (group >= groups) return;
    if (threadIdx.x == 0) { dealt[0] = total; dealt[1] = groups; }
#pragma nounroll
    for (int k = 0; k < 2; ++k) {
        int64_t at = tree_ratio(group + k, total, groups);
        if (at >= total) {
            if (threadIdx.x == 0) places[k] = {a.requests, 0, 0, total + kTreeUnit};
        } else if (at < upto && at >= upto - mine) {
            int64_t before = upto - mine, all;
            int r = r0 - 1;
            Draft d;
            for (all = 0;; before += all) {
                d = draft_of<DC, WR, false>(a, ++r);
                all = (int64_t)a.heads * d.blocks * (d.tiles + kTreeUnit);
                if (at < before + all) break;
            }
            // (a unit's own cost comes before its tiles: what begins within it begins with tile 0)
            int unit = (int)tree_ratio(at - before, 1, d.tiles + kTreeUnit), tile = (int)((at - before) - (int64_t)unit * (d.tiles + kTreeUnit)) - kTreeUnit;
            at += max(-tile, 0);
            tile = max(tile, 0);
            if (d.tiles <= kTreeWhole && tile) {             // short units go where most of them lies
                at -= tile;
                if (2 * tile > d.tiles) {
                    at += d.tiles + kTreeUnit;
                    if (++unit == a.heads * d.blocks) {
                        unit = 0;
                        ++r;
                    }
                }
                tile = 0;
            }
            places[k] = {r, unit, tile, at};
        }
    }
    }
    __syncthreads();
    const int64_t end = uniform64(places[1].at);

    char *const ours = lds + (T::kAlone ? wave * T::kBuffer : 0);
    const int loader = T::kAlone ? lane : (int)threadIdx.x, piece = loader % kPieces, line = loader / kPieces;
    // A unit's part that is this workgroup's: tiles [tile, last); `at`: place of the first one in the order of all.
    struct Unit {
        Draft d;
        int64_t at;
        int32_t request, unit, tile, last, h, block;
    };
    auto unit_of = [&](int request, int unit, int tile, int64_t at) {
        const PagedTreeAttentionArgs &a = tree_args().a;
        Unit u;
        u.d = draft_of<DC, WR, true>(a, request);
        while (u.d.blocks == 0) u.d = draft_of<DC, WR, true>(a, ++request);
        u.request = request; u.unit = unit; u.tile = tile; u.at = at;
        u.h = unit / u.d.blocks;
        u.block = unit - u.h * u.d.blocks;
        u.last = (int)min((int64_t)u.d.tiles, tile + (end - at));
        return u;
    };
    auto after = [&](const Unit &u) {                        // the unit behind it, whose first tile lies at ...
        const bool done = u.unit + 1 == tree_args().a.heads * u.d.blocks;
        return unit_of(u.request + (done ? 1 : 0), done ? 0 : u.unit + 1, 0, u.at + (u.last - u.tile) + kTreeUnit);
    };

    // ---- rows of keys and values.  Lane i looks after token i of what its wavefront or workgroup stages: it asks for the token's page number, two
    // tiles ahead, and leaves the place for those that load it, a tile ahead.
    const int mine_at = lane & (T::kStaged - 1);
    auto first_of = [&](const Unit &u, int i) { return (uint32_t)u.d.start + (uint32_t)i * T::kTokens + (T::kAlone ? wave * T::kMine : 0); };
    auto look_up = [&](const Unit &u, const int32_t *row, const PageDiv &page, int i) {
        const uint32_t t = first_of(u, i) + (uint32_t)mine_at;
        return i < u.last && t < (uint32_t)u.d.end ? row[page.div(t)] : -1;
    };
    auto row_of = [&](const Unit &u) {
        const PagedTreeAttentionArgs &a = tree_args().a;
        return (const int32_t *)uniform64((int64_t)(uintptr_t)(a.table + u.request * a.table_stride));
    };
    // The rows of the next tile: where they are, then one after the other.  A burst of all of them holds the wavefront up (eight loads 2400 cycles, of
    // the 7900 that a pair of tiles takes), so within a unit they go between the matrix instructions.
    uint32_t kx[kPasses][4], vx[kPasses][4];
    uint64_t missing = 0;                                    // bit i: the token that lane i looks after is not there
    // (tokens that are not there, pieces behind the row's end: anything that can be read, for 16 bytes)
    auto aim = [&](const Unit &u, int i, int32_t number) {
        const PagedTreeAttentionArgs &a = tree_args().a;
        const uint32_t t = first_of(u, i) + (uint32_t)mine_at, in = t - a.page.div(t) * a.page.d;
        const bool none = (uint32_t)number >= (uint32_t)a.pages;
        missing = __ballot(none);
        spots[wave][0][lane] = none ? -1 : (int64_t)number * a.k.page_bytes + (int64_t)in * a.k.token_bytes;
        spots[wave][1][lane] = none ? -1 : (int64_t)number * a.v.page_bytes + (int64_t)in * a.v.token_bytes;
        __builtin_amdgcn_wave_barrier();
    };
    auto aim_nowhere = [&]() {
        spots[wave][0][lane] = spots[wave][1][lane] = -1;
        __builtin_amdgcn_wave_barrier();
    };
    struct Bases {
        const char *k, *v, *readable;
        int row_bytes;
    };
    auto bases_of = [&](const Unit &u) {
        const PagedTreeAttentionArgs &a = tree_args().a;
        const int row_bytes = EB * a.dim, b = SHORT ? 0 : ANY ? min(16 * piece, row_bytes - 16) : 16 * piece;
        return Bases{a.k.base + u.h * a.k.head_bytes + b, a.v.base + u.h * a.v.head_bytes + b, a.q, row_bytes};
    };
    auto fetch = [&](uint32_t (&x)[4], const Bases &from, int which, int p) {
        const int64_t at = spots[wave][which][p * kAtOnce + line];
        const char *const q = at >= 0 && 16 * piece < from.row_bytes ? (which ? from.v : from.k) + at : from.readable;
        if (SHORT) load_part<4>(x, q, from.row_bytes);
        else load_stream<4>(x, q);
    };
    auto fetch_all = [&](const Bases &from) {
#pragma unroll
        for (int p = 0; p < kPasses; ++p) { fetch(kx[p], from, 0, p); fetch(vx[p], from, 1, p); }
    };
    // Staged tokens from t on that not all rows see: those of the draft, and where the rows' windows begin.
    auto hidden = [&](const Draft &d, int window, uint32_t t) {
        const int all_from = window ? max(d.before - window + min(d.end - d.before, window), 0) : 0;
        return t + T::kStaged > (uint32_t)d.before || t < (uint32_t)all_from;
    };

    Unit cur, next = unit_of(uniform(places[0].request), uniform(places[0].unit), uniform(places[0].tile), uniform64(places[0].at));
    bool begun_any = false, more = next.at < end;
    int32_t number = -1;
    if (more) number = look_up(next, row_of(next), tree_args().a.page, next.tile);
    f32x16 o[DB];
    float m = -INFINITY, l = 0.f;
    while (more || begun_any) {
        // ---- the next unit's first tile and queries are on their way while this one is finished
        constexpr int kQueries = T::kAlone ? 32 : T::kRows, kEach = kQueries * (DC / 8) / kLoaders;
        static_assert(kQueries * T::kPitchK <= (T::kAlone ? T::kBuffer : T::kLds) && kQueries * (DC / 8) % kLoaders == 0);
        u32x4 y[kEach];
        if (more) {
            const PagedTreeAttentionArgs &a = tree_args().a;
            const TreeWork &w = tree_args().w;
            aim(next, next.tile, number);
            fetch_all(bases_of(next));
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int x = loader + e * kLoaders, b = 16 * (x % (DC / 8));
                const TreeRow t = tree_row(a, w, next.d, next.h, (int64_t)next.block * T::kRows + x / (DC / 8));
                const char *const p = a.q + t.head * a.q_head_bytes + (int64_t)(next.d.row0 + t.node) * a.q_row_bytes;
                uint32_t z[4] = {0, 0, 0, 0};
                if (t.there && b < 2 * a.dim) {
                    if (ANY && 2 * a.dim < 16) load_part<4>(z, p, 2 * a.dim);
                    else load_stream<4>(z, p + min(b, 2 * a.dim - 16));
                }
                y[e] = u32x4{z[0], z[1], z[2], z[3]};
            }
        }
        if (begun_any) {
            // ---- the unit's end: join the wavefronts, give out the result or leave a part.  By way of LDS, so that whole rows are stored.
            const PagedTreeAttentionArgs &a = tree_args().a;
            const TreeWork &w = tree_args().w;
            const Draft &d = cur.d;
            const bool begun = cur.tile == 0, done = cur.last == d.tiles, whole = begun && done;
            const int part_slot = 2 * group + (begun ? 1 : 0);
            const float v_scale = F8 ? a.v.scale[cur.h] : 1.f;
            const TreeShared<T::kRows> shared(w);
            constexpr int kPart = T::kAlone ? T::kBuffer : T::kLds / kTreeWaves, kDims = DC < 128 ? DC : 128, kPitch = kDims + 4;       // (dimensions at a time)
            static_assert(32 * kPitch * 4 <= kPart && kPart % 16 == 0);
            float *const mineo = (float *)(lds + wave * kPart) + l32 * kPitch;
            l = pair_sum(l);
            if (half == 0) { wave_m[wave][l32] = m; wave_l[wave][l32] = l; }
            if (!T::kAlone) tree_barrier();                  // (else a wavefront's part lies where its own tokens did)
#pragma unroll
            for (int c = 0; c < DC / kDims; ++c) {
#pragma unroll
                for (int j = 0; j < kDims / 32; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *(f32x4 *)(mineo + 32 * j + 8 * g + 4 * half) =
                            f32x4{o[c * (kDims / 32) + j][4 * g], o[c * (kDims / 32) + j][4 * g + 1], o[c * (kDims / 32) + j][4 * g + 2], o[c * (kDims / 32) + j][4 * g + 3]};
                if (T::kGroups > 1) tree_barrier();
                else __builtin_amdgcn_wave_barrier();
                // kGroups > 1: all threads have the rows of all; else each wavefront has its own
                constexpr int kThreads = T::kGroups > 1 ? kTreeThreads : 64, kMany = (T::kGroups > 1 ? T::kRows : 32) * (kDims / 4);
#pragma unroll 2
                for (int e = T::kGroups > 1 ? (int)threadIdx.x : lane; e < kMany; e += kThreads) {
                    const int x = e / (kDims / 4) + (T::kGroups > 1 ? 0 : 32 * wr), dim1 = 4 * (e % (kDims / 4)), dim0 = c * kDims + dim1;
                    const TreeRow t = tree_row(a, w, d, cur.h, (int64_t)cur.block * T::kRows + x);
                    float top = -INFINITY, sum = 0.f;
                    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                    if (T::kGroups == 1) {
                        top = wave_m[wave][x % 32];
                        sum = wave_l[wave][x % 32];
                        acc = *(const f32x4 *)((const float *)(lds + wave * kPart) + (x % 32) * kPitch + dim1);
                    } else {
#pragma unroll
                        for (int i = 0; i < T::kGroups; ++i) top = fmaxf(top, wave_m[i * WR + x / 32][x % 32]);
                        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                        for (int i = 0; i < T::kGroups; ++i) {
                            const int v = i * WR + x / 32;
                            const float f = __builtin_amdgcn_exp2f(wave_m[v][x % 32] - base);
                            sum += f * wave_l[v][x % 32];
                            acc += f * *(const f32x4 *)((const float *)(lds + v * kPart) + (x % 32) * kPitch + dim1);
                        }
                    }
                    if (t.there && dim0 < a.dim) {
                        if (whole) {
                            tree_result<DT>(a, d, t, dim0, acc, sum, v_scale);
                        } else {
                            shared.store(part_slot, x, dim0, acc);
                            if (dim0 == 0) shared.store(part_slot, x, TreePart{top, sum});
                        }
                    }
                }
                if (c + 1 < DC / kDims) {
                    if (T::kGroups > 1) tree_barrier();
                    else __builtin_amdgcn_wave_barrier();
                }
            }
            tree_barrier();
            if (odd) {
                // Values that are not finite, for the rows that see them: an infinity or a NaN of whatever weight is the result's.
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                const int32_t *const row = row_of(cur);
                for (int e = (int)threadIdx.x; e < T::kRows * a.dim; e += kTreeThreads) {
                    const int x = e / a.dim, dim = e - x * a.dim;
                    const TreeRow t = tree_row(a, w, d, cur.h, (int64_t)cur.block * T::kRows + x);
                    const Sight s = sight_of(a, d, t, row_from[x]);
                    float add = 0.f;
                    const uint32_t t_end = (uint32_t)min((int64_t)d.end, (int64_t)d.start + (int64_t)cur.last * T::kTokens);
#pragma nounroll
                    for (uint32_t tok = (uint32_t)d.start + (uint32_t)cur.tile * T::kTokens; tok < t_end; ++tok) {
                        if (!hidden(d, a.window, tok & ~(uint32_t)(T::kStaged - 1)) || !(s(d, a.words, tok) & 1)) continue;
                        const uint32_t at_page = a.page.div(tok);
                        const int32_t in_page = row[at_page];
                        if ((uint32_t)in_page >= (uint32_t)a.pages) continue;
                        const char *const v = a.v.base + cur.h * a.v.head_bytes + in_page * a.v.page_bytes + (int64_t)(tok - at_page * a.page.d) * a.v.token_bytes + EB * dim;
                        const uint32_t bits = F8 ? *(const uint8_t *)v : *(const u16_any *)v;
                        if (F8 ? (bits & 0x7f) == 0x7f : (bits & E::kExponent) == E::kExponent) add += F8 ? NAN : Elem<DT>::to_float((uint16_t)bits);
                    }
                    if (t.there && add != 0.f) {
                        if (whole) ((u16_any *)(a.out + t.head * a.out_head_bytes + (int64_t)(d.row0 + t.node) * a.out_row_bytes))[dim] = Elem<DT>::from_float(add);
                        else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, add), shared.sums, shared.sum_at(part_slot, x, dim), 0, kTreeAux);
                    }
                }
                __syncthreads();
                if (threadIdx.x == 0) odd = 0;
                __syncthreads();
            }
            if (!whole) {
                const int64_t first = cur.at - cur.tile, total = uniform64(dealt[0]), groups = uniform64(dealt[1]);
                TreeLeft u = {begun ? group : (int)tree_ratio_up(first + 1, groups, total) - 1, 0, cur.request, cur.h, cur.block};
                u.parts = (int)tree_ratio_up(first + d.tiles, groups, total) - u.begins;
                if (w.left) {
                    if (begun && threadIdx.x == 0) w.left[group] = u;
                } else {
                    if (threadIdx.x == 0) left[unfinished] = u;
                    ++unfinished;                            // (the first unit of the share at most, and its last)
                }
            }
            if (!more) break;
        }
        // ---- queries by way of LDS: column l32 of the scores
        cur = next;
        begun_any = true;
        const PagedTreeAttentionArgs &a = tree_args().a;
        const Draft &d = cur.d;
        u32x4 q[KS];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int x = loader + e * kLoaders, b = 16 * (x % (DC / 8));
            uint32_t z[4] = {y[e][0], y[e][1], y[e][2], y[e][3]};
            if (ANY && 2 * a.dim >= 16) tree_shift(z, max(b - (2 * a.dim - 16), 0));
            *(u32x4 *)(ours + x / (DC / 8) * T::kPitchK + b) = u32x4{z[0], z[1], z[2], z[3]};
        }
        if (!T::kAlone) tree_barrier();
#pragma unroll
        for (int k = 0; k < KS; ++k) q[k] = *(const u32x4 *)(ours + (T::kAlone ? l32 : 32 * wr + l32) * T::kPitchK + 32 * k + 16 * half);
        if (!T::kAlone) tree_barrier();
        const int32_t *const row = row_of(cur);
        Sight sight = sight_of(a, d, tree_row(a, tree_args().w, d, cur.h, (int64_t)cur.block * T::kRows + 32 * wr + l32), 0);
        if (a.window) sight.from = window_from(a, d, sight);
        if (wt == 0 && half == 0) row_from[32 * wr + l32] = sight.from;
        const int window = uniform(a.window), words = uniform(a.words), row_bytes = uniform(EB * a.dim);
        const PageDiv page_div = {(uint32_t)uniform((int)a.page.d), (uint32_t)uniform((int)a.page.mul), (uint32_t)uniform((int)a.page.shift)};
        const bool has_piece = 16 * piece < row_bytes;
        const float to_log2 = a.scale * kLog2e * (F8 ? a.k.scale[cur.h] : 1.f);
#pragma unroll
        for (int j = 0; j < DB; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[j][i] = 0.f;
        m = -INFINITY; l = 0.f;
        more = cur.at + (cur.last - cur.tile) + kTreeUnit < end;

        const Bases from = bases_of(cur);
        number = look_up(cur, row, page_div, cur.tile + 1);
        for (int i = cur.tile; i < cur.last; ++i) {
            char *const buf = ours + (T::kAlone ? 0 : (i & 1) * T::kBuffer);
            const bool some_hidden = hidden(d, window, first_of(cur, i));
            // -- the tile's rows, which have arrived, into LDS, in 16 bits
            if (ANY && !SHORT && 16 * piece + 16 > row_bytes && has_piece) {
                const int past = 16 * piece - (row_bytes - 16);
#pragma unroll
                for (int p = 0; p < kPasses; ++p) { tree_shift(kx[p], past); tree_shift(vx[p], past); }
            }
            if (missing) {
                // Tokens that are not there, or on a page outside the cache: values of zero; keys of NaN, which is the result of a row that
                // sees them (zeros behind the row's end: the queries' zeros there would make NaN of those as well).
#pragma unroll
                for (int p = 0; p < kPasses; ++p)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int bytes = ANY ? row_bytes - 16 * piece - 4 * x : 4;
                        const uint32_t nan = (F8 ? 0x7f7f7f7fu : 0x7fff7fffu) & (bytes >= 4 ? 0xffffffffu : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1u);
                        const bool none = missing >> (p * kAtOnce + line) & 1;
                        kx[p][x] = none && has_piece ? nan : kx[p][x];
                        vx[p][x] = none ? 0u : vx[p][x];
                    }
            }
            if (some_hidden) {
                // Values that are not finite where not every row sees every token: a probability of 0 times them would be NaN.  They take part
                // as zeros, and rows that see them get them at the unit's end.
                constexpr int kWidth = F8 ? 8 : 16;
                constexpr uint32_t kTop = F8 ? 0x7fu : E::kExponent, kAll = F8 ? 0xffu : 0xffffu;
                bool found = false;
#pragma unroll
                for (int p = 0; p < kPasses; ++p)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int b = 0; b < 32; b += kWidth) {
                            const bool hit = (vx[p][x] >> b & kTop) == kTop;
                            found |= hit;
                            vx[p][x] &= hit ? ~(kAll << b) : 0xffffffffu;
                        }
                if (found && has_piece) odd = 1;
            }
            if (row_bytes < 16 * kPieces) {
#pragma unroll
                for (int p = 0; p < kPasses; ++p)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        kx[p][x] = has_piece ? kx[p][x] : 0u;
                        vx[p][x] = has_piece ? vx[p][x] : 0u;
                    }
            }
            {
                char *const kt = buf + line * T::kPitchK + (F8 ? 32 : 16) * piece, *const vt = buf + T::kStaged * T::kPitchK + line * T::kPitchV + (F8 ? 32 : 16) * piece;
                auto put = [&](char *to, const uint32_t (&x)[4]) {
                    if (F8) {
                        *(u32x4 *)to = u32x4{tree_widen<DT, false>(x[0]), tree_widen<DT, true>(x[0]), tree_widen<DT, false>(x[1]), tree_widen<DT, true>(x[1])};
                        *(u32x4 *)(to + 16) = u32x4{tree_widen<DT, false>(x[2]), tree_widen<DT, true>(x[2]), tree_widen<DT, false>(x[3]), tree_widen<DT, true>(x[3])};
                    } else {
                        *(u32x4 *)to = u32x4{x[0], x[1], x[2], x[3]};
                    }
                };
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    put(kt + p * kAtOnce * T::kPitchK, kx[p]);
                    put(vt + p * kAtOnce * T::kPitchV, vx[p]);
                }
            }
            const bool follows = i + 1 < cur.last;
            if (follows) {
                aim(cur, i + 1, number);
                if (SHORT) fetch_all(from);
                number = look_up(cur, row, page_div, i + 2);
            } else {
                aim_nowhere();
                if (more) {
                    next = after(cur);
                    number = look_up(next, row_of(next), page_div, next.tile);
                }
            }
            if (!T::kAlone) tree_barrier();

            // -- scores of tokens t0 + 32 u + 8 (x / 4) + 4 half + x % 4
            const uint32_t t0 = first_of(cur, i) + (T::kAlone ? 0 : wt * T::kMine);
            const char *const kt = buf + ((T::kAlone ? 0 : wt * T::kMine) + l32) * T::kPitchK + 16 * half;
            f32x16 s[SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
#pragma unroll
                for (int x = 0; x < 16; ++x) s[u][x] = 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    s[u] = E::mfma(*(const u32x4 *)(kt + 32 * u * T::kPitchK + 32 * k), q[k], s[u]);
                    constexpr int kEvery = SUBS * KS / kPasses;
                    if (!SHORT && (u * KS + k + 1) % kEvery == 0) fetch(kx[(u * KS + k) / kEvery], from, 0, (u * KS + k) / kEvery);
                }
            }
#pragma unroll
            for (int u = 0; u < SUBS; ++u) s[u] *= to_log2;
            if (some_hidden) {
                const uint64_t see = sight(d, words, t0) >> (4 * half);
#pragma unroll
                for (int u = 0; u < SUBS; ++u)
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[u][x] = (uint32_t)(see >> (32 * u)) >> (8 * (x / 4) + x % 4) & 1 ? s[u][x] : -INFINITY;
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int x = 0; x < 16; ++x) top = fmaxf(top, s[u][x]);
            top = pair_max(top);
            if (__any(top > m + kTreeLag)) {                 // (also the first that is seen: m is -inf)
                const float shrink = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
                l *= shrink;
#pragma unroll
                for (int j = 0; j < DB; ++j) o[j] *= shrink;
                m = top;
            }
            const float base = (m == -INFINITY ? 0.f : m) - E::kLift;
            u32x4 p[2 * SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int x = 0; x < 16; x += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(s[u][x] - base), p1 = __builtin_amdgcn_exp2f(s[u][x + 1] - base);
                    l += p0 + p1;
                    p[2 * u + x / 8][x % 8 / 2] = Elem<DT>::pack2(p0, p1);
                }
            // -- values: lane (dimension 32 j + l32, half) has tokens 16 k + 4 half + 0 .. 3 and 8 behind those
            const LdsPtr vt = (LdsPtr)(buf + T::kStaged * T::kPitchK) + ((T::kAlone ? 0 : wt * T::kMine) + 4 * half + (lane & 15) / 4) * T::kPitchV +
                              32 * (lane >> 4 & 1) + 8 * (lane & 3);
#pragma unroll
            for (int k = 0; k < 2 * SUBS; ++k)
#pragma unroll
                for (int j = 0; j < DB; ++j) {
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPiece)(vt + 16 * k * T::kPitchV + 64 * j)));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPiece)(vt + (16 * k + 8) * T::kPitchV + 64 * j)));
                    o[j] = E::mfma(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[k], o[j]);
                    constexpr int kEvery = 2 * SUBS * DB / kPasses;
                    if (!SHORT && (k * DB + j + 1) % kEvery == 0) fetch(vx[(k * DB + j) / kEvery], from, 1, (k * DB + j) / kEvery);
                }
        }
    }
    const PagedTreeAttentionArgs &a = tree_args().a;
    const TreeWork &w = tree_args().w;
    if (w.left || unfinished == 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 0; i < unfinished; ++i) {
            int32_t *const counter = w.counters + left[i].begins;
            joins[i] = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == left[i].parts - 1;
            if (joins[i]) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    __syncthreads();
#pragma nounroll
    for (int i = 0; i < unfinished; ++i)
        if (joins[i]) tree_join<DT, DC, WR>(a, w, left[i], 0, T::kRows, F8 ? a.v.scale[left[i].h] : 1.f);
}

// The joining as a kernel of its own: grid (workgroups of the other, blocks of rows).
template <int DT, int DC, int WR> __global__ void __launch_bounds__(kTreeThreads) paged_tree_join_kernel(TreeArgs args, int rows) {
    const PagedTreeAttentionArgs &a = args.a;
    const TreeWork &w = args.w;
    const TreeLeft u = w.left[blockIdx.x];
    const int row0 = (int)blockIdx.y * rows;
    if (u.parts) tree_join<DT, DC, WR>(a, w, u, row0, row0 + rows, a.v.scale ? a.v.scale[u.h] : 1.f);
}

// ------------------------------------------------------------------ host
// Which build takes a call: dimensions that its registers hold, wavefronts side by side over the rows.
static inline int tree_dims(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
static inline int tree_waves(int64_t tokens, int64_t requests, int64_t group) { return tokens * group <= 32 * std::max<int64_t>(1, requests) ? 1 : 4; }

template <int DT, bool F8, int DC, int WR, TreeRows ROWS> static int launch_tree_build(const PagedTreeAttentionArgs &a, const TreeWork &w, hipStream_t stream) {
    typedef TreeTile<DC, WR> T;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_tree_attention_kernel<DT, F8, DC, WR, ROWS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (attr != hipSuccess) return BA_ERR_LAUNCH;
    paged_tree_attention_kernel<DT, F8, DC, WR, ROWS><<<w.groups, kTreeThreads, T::kLds, stream>>>(TreeArgs{a, w});
    if (w.left) {
        constexpr int kRows = std::min(T::kRows, 4 * kTreeThreads / (DC / 4));      // (a round of its threads)
        paged_tree_join_kernel<DT, DC, WR><<<dim3((unsigned)w.groups, T::kRows / kRows), kTreeThreads, 0, stream>>>(TreeArgs{a, w}, kRows);
    }
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

template <int DT, bool F8, int DC, int WR> static int launch_tree_rows(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, hipStream_t stream) {
    if constexpr (DC == 64)
        if (rows == kTreeShort) return launch_tree_build<DT, F8, DC, WR, kTreeShort>(a, w, stream);
    return rows == kTreePieces ? launch_tree_build<DT, F8, DC, WR, kTreePieces>(a, w, stream) : launch_tree_build<DT, F8, DC, WR, kTreeAny>(a, w, stream);
}
template <int DT, bool F8, int DC> static int launch_tree_dims(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream) {
    return waves == 1 ? launch_tree_rows<DT, F8, DC, 1>(a, w, rows, stream) : launch_tree_rows<DT, F8, DC, 4>(a, w, rows, stream);
}
template <int DT, bool F8> int launch_tree_types(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream) {
    switch (tree_dims(a.dim)) {
        case 64: return launch_tree_dims<DT, F8, 64>(a, w, rows, waves, stream);
        case 128: return launch_tree_dims<DT, F8, 128>(a, w, rows, waves, stream);
        default: return launch_tree_dims<DT, F8, 256>(a, w, rows, waves, stream);
    }
}

}  // namespace ba
