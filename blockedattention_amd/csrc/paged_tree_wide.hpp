// Attention of drafted tokens for many rows a key head (units of 64 or 128; tree_rows).
//
// A unit is 128 rows, 32 a wavefront, or (64 dimensions) 64, of which two wavefronts have the same and half of the tile's tokens each.  All four wavefronts bring a tile
// of 64 tokens (32 for 128 rows of more than 128 dimensions) into LDS together, in 16 bits, by way of registers; two tiles lie there in turn.
//   Scores, S[token][row] = K Q^T on the 32 x 32 x 16 matrix instruction, so that a lane has sixteen tokens of one row: maxima and sums cost one
//   exchange between the halves, and the probabilities are, packed to 16 bits, the second product's operand as they are, if that runs over the
//   tokens in the order in which the lanes have them.
//   Values, O[d][row] = V^T P: the transposing LDS read gives four tokens of a dimension.
// A row's maximum is only moved when a larger one comes by more than 2^7, so accumulators are scaled seldom.  Probabilities are as exact as in the kernel for
// few rows, since which of the two answers a request depends on the other requests: two 16-bit terms (paged_attention_kernel.hpp), or, for bf16 queries
// over an 8-bit cache, one of fp16, whose error is an eighth of the result's own rounding; e4m3 values are exact in fp16.  One term of the result's type
// would add its own rounding's error once more (1.3 times the whole error); two cost the second product again (64 requests of 4000 tokens, 128 rows of 128
// dimensions 240 -> 286 us, 512 rows 215 -> 265; a batch of 32 drafts 94.6 -> 97.5).
// What bounds it: a wavefront's chain of LDS, products, exponentials, LDS, products, of which two to a SIMD hide half (two requests of 32768 to 65536
// tokens in 8 bits, 512 rows a key head, 240 GFLOP: 340 to 352 us, 680 to 705 TFLOP/s with the matrix unit busy 33 % of the time, vector instructions
// 37 %, LDS 37 %).  32 requests of up to 4096 tokens and 32 nodes (281 MB) take 92 to 97 us by the card.
#pragma once
#include "paged_tree_attention.hpp"

namespace ba {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char *LdsBytes;
typedef __attribute__((address_space(3))) s16x4 *LdsPiece;

// WR: wavefronts side by side over the rows, 2 or 4.
template <int DC_, int WR> struct TreeWide {
    static constexpr int DC = DC_, kRows = 32 * WR, kGroups = kTreeWaves / WR, kWaveRows = kGroups > 1 ? kRows : 32;
    static constexpr int kTokens = DC < 256 ? 64 : 32, kStaged = kTokens, kMine = kTokens / kGroups;      // kMine: of a wavefront
    // Bytes between rows in LDS: keys 16 more than whole lines of banks, so that sixteen rows' pieces lie side by side; values 64 more, so
    // that four rows' 64 bytes do.
    static constexpr int kPitchK = 2 * DC + 16, kPitchV = 2 * DC + 64, kBuffer = kTokens * (kPitchK + kPitchV), kLds = 2 * kBuffer;
    static constexpr int kDims = DC < 128 ? DC : 128, kPitch = kDims + 4, kPart = kWaveRows * kPitch * 4;
    static constexpr int kResident = DC == 64 ? 3 : DC == 128 ? 2 : 1;    // by LDS and registers
    static_assert((kGroups > 1 ? kGroups : kTreeWaves) * kPart <= kLds && kRows * kPitchK <= kLds);
};

template <int DT> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == 0) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Probabilities are lifted by a power of two, so that small ones stay apart from zero in fp16.  A maximum that is kept though a
// larger one has come (by up to 2^7) leaves them at 2^15 at most.
template <int PT> constexpr float kTreeLift = PT == 0 ? 8.f : 0.f;
constexpr float kTreeLag = 7.f;
constexpr int kMatrix = 0x8, kDsRead = 0x100;                // kinds of instructions, for the scheduler

// Greatest and sum over a lane and its partner, 32 lanes on.
__device__ __forceinline__ float pair_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// A sum and both fp16 halves of a dword: of probabilities of one term as they are after rounding, which the values are weighed with.
__device__ __forceinline__ float add_both(uint32_t x, float sum) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
}

// DC: dimensions that the registers hold (64, 128, 256).
template <int DT, bool F8, int DC, int WR, TreeRows ROWS>
__global__ void __launch_bounds__(kTreeThreads, (TreeWide<DC, WR>::kResident)) paged_tree_wide_kernel(TreeArgs) {
    typedef TreeWide<DC, WR> T;
    constexpr bool ANY = ROWS != kTreePieces, SHORT = ROWS == kTreeShort;
    constexpr int EB = F8 ? 1 : 2, kPieces = DC * EB / 16;   // bytes of an element, 16-byte pieces of a row
    constexpr int kAtOnce = kTreeThreads / kPieces, kPasses = T::kTokens / kAtOnce;      // rows of a load, loads of a tile
    constexpr int KS = DC / 16, DB = DC / 32, SUBS = T::kMine / 32;
    constexpr int PT = F8 ? 0 : DT;          // type of probabilities and values in the second product (8 bits: exact in fp16)
    constexpr bool TWO = !(F8 && DT == 1);   // probabilities have two terms
    static_assert(kTreeThreads % kPieces == 0 && T::kTokens % kAtOnce == 0);
    const int lane = lane_id(), l32 = lane & 31, half = lane >> 5, wave = uniform((int)threadIdx.x >> 6), wr = wave % WR, wt = wave / WR;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ TreeLds<T> sh;
    int unfinished = 0;
    TreeUnit cur, next;
    int group;
    const int64_t end = tree_deal<T>(sh, next, group);
    if (end < 0) return;

    const int piece = (int)threadIdx.x % kPieces, line = (int)threadIdx.x / kPieces, mine_at = lane & (T::kTokens - 1);
    // The rows of the next tile: where they are, then one after the other.  A burst of all of them holds the wavefront up (eight loads 2400 cycles, of
    // the 7900 that a pair of tiles took), so within a unit they go between the matrix instructions.
    uint32_t kx[kPasses][4], vx[kPasses][4];
    Missing missing = {};                                    // of the tile
    auto first_of = [&](const TreeUnit &u, int i) { return (uint32_t)u.d.start + (uint32_t)i * T::kTokens; };
    // (pieces behind the row's end: its last bytes)
    auto fetch = [&](uint32_t (&x)[4], const TreeBases &from, int which, int p) {
        const int b = SHORT ? 0 : min(16 * piece, from.row_bytes - 16);
        const char *const q = (which ? from.v : from.k) + b + sh.spots[wave][which][p * kAtOnce + line];
        if (SHORT) load_part<4>(x, q, from.row_bytes);
        else load_stream<4>(x, q);
    };
    auto fetch_all = [&](const TreeBases &from) {
#pragma unroll
        for (int p = 0; p < kPasses; ++p) { fetch(kx[p], from, 0, p); fetch(vx[p], from, 1, p); }
    };

    bool any = false, more = true;
    int32_t number = look_up(next, table_row(next), tree_args().a.page, true, first_of(next, next.tile) + mine_at);
    f32x16 o[DB];
    float m = -INFINITY, l = 0.f, base = kTreeLift<PT>;      // base: what is added to scores in the exponent
    for (;;) {
        // ---- the next unit's first tile and queries are on their way while this one is finished
        constexpr int kEach = T::kRows * (DC / 8) / kTreeThreads;
        u32x4 y[kEach];
        if (more) {
            const PagedTreeAttentionArgs &a = tree_args().a;
            const TreeWork &w = tree_args().w;
            const TreeBases from = tree_bases<EB>(next);
            missing = tree_aim<T>(sh.spots[wave], mine_at, tree_steps(), from, next, first_of(next, next.tile) + mine_at, number);
            fetch_all(from);
            const int me = opaque((int)threadIdx.x);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int x = me + e * kTreeThreads, b = 16 * (x % (DC / 8));
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
        if (any) {
            const int me = opaque((int)threadIdx.x), my32 = me & 31;
            // (kGroups > 1: the rows of all wavefronts with the same tokens are one part)
            const int part = T::kGroups > 1 ? wt : wave, mine = T::kGroups > 1 ? 32 * wr + my32 : my32;
            float *const mineo = (float *)(lds + part * T::kPart) + mine * T::kPitch + 4 * (me >> 5 & 1);
            const float v_scale = F8 ? tree_args().a.v.scale[cur.h] : 1.f;
            l = pair_sum(l);
            if ((me & 32) == 0) { sh.m[part][mine] = m == -INFINITY ? m : -base; sh.l[part][mine] = l; }
            lds_barrier();
#pragma unroll
            for (int c = 0; c < DC; c += T::kDims) {
#pragma unroll
                for (int j = 0; j < T::kDims / 32; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x16 &x = o[c / 32 + j];
                        *(f32x4 *)(mineo + 32 * j + 8 * g) = f32x4{x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
                    }
                lds_barrier();
                tree_store<DT, T>(sh, group, lds, cur, me, c, v_scale);
                if (c + T::kDims < DC) lds_barrier();
            }
            const bool odd = uniform(sh.odd) != 0;
            lds_barrier();
            tree_end<DT, F8, T>(sh, group, cur, me, odd, unfinished);
            if (!more) break;
        }
        // ---- queries by way of LDS: column l32 of the scores
        cur = next;
        any = true;
        const PagedTreeAttentionArgs &a = tree_args().a;
        const Draft &d = cur.d;
        u32x4 q[KS];
        // Scores are scaled within the exponent, by a factor above 0: the sign goes to the queries, 0 becomes the smallest number, and a scale that is no number
        // makes the queries such, so that a row is NaN if it sees a token.
        const float scale = a.scale * kLog2e * (F8 ? a.k.scale[cur.h] : 1.f);
        const bool is_number = scale == scale;
        const float to_log2 = is_number ? fmaxf(fabsf(scale), 0x1p-149f) : 1.f, lag = fminf(kTreeLag / to_log2, 0x1.fffffep127f);
        const uint32_t turn = scale < 0.f ? 0x80008000u : 0u, nan = is_number ? 0u : 0x7fff7fffu;
        const int me = opaque((int)threadIdx.x);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int x = me + e * kTreeThreads, b = 16 * (x % (DC / 8));
            uint32_t z[4] = {y[e][0], y[e][1], y[e][2], y[e][3]};
            if (ANY && 2 * a.dim >= 16) shift_down<4>(z, max(b - (2 * a.dim - 16), 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = (z[i] ^ turn) | nan;
            *(u32x4 *)(lds + x / (DC / 8) * T::kPitchK + b) = u32x4{z[0], z[1], z[2], z[3]};
        }
        lds_barrier();
#pragma unroll
        for (int k = 0; k < KS; ++k) q[k] = *(const u32x4 *)(lds + (32 * wr + (me & 31)) * T::kPitchK + 32 * k + 16 * (me >> 5 & 1));
        lds_barrier();
        const TableRow row = table_row(cur);
        Sight sight = sight_of(a, d, tree_row(a, tree_args().w, d, cur.h, (int64_t)cur.block * T::kRows + 32 * wr + (me & 31)), 0);
        if (a.window) sight.from = window_from(a, d, sight);
        if (wt == 0 && (me & 32) == 0) sh.row_from[32 * wr + (me & 31)] = sight.from;
        const int window = uniform(a.window), words = uniform(a.words), row_bytes = uniform(EB * a.dim);
        const TreeSteps by = tree_steps();
        const TreeBases from = tree_bases<EB>(cur);
        const bool has_piece = 16 * piece < row_bytes;
#pragma unroll
        for (int j = 0; j < DB; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[j][i] = 0.f;
        m = -INFINITY; l = 0.f; base = kTreeLift<PT>;
        more = tree_next(cur) < end;

        number = look_up(cur, row, by.page, cur.tile + 1 < cur.last, first_of(cur, cur.tile + 1) + mine_at);
        for (int i = cur.tile; i < cur.last; ++i) {
            char *const buf = lds + (i & 1) * T::kBuffer;
            const bool some_hidden = hidden<T>(d, window, first_of(cur, i));
            // -- the tile's rows, which have arrived, into LDS, in 16 bits
            if (ANY && !SHORT && 16 * piece + 16 > row_bytes && has_piece) {
                const int past = 16 * piece - (row_bytes - 16);
#pragma unroll
                for (int p = 0; p < kPasses; ++p) { shift_down<4>(kx[p], past); shift_down<4>(vx[p], past); }
            }
            // Tokens that are not there: values of zero.  On a page outside the cache: keys of NaN as well, which is the result of a row that sees them
            // (zeros behind the row's end: the queries' zeros there would make NaN of those too).
            if (missing.any) {
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    const bool none = missing.any >> (p * kAtOnce + line) & 1;
#pragma unroll
                    for (int x = 0; x < 4; ++x) vx[p][x] = none ? 0u : vx[p][x];
                }
                if (missing.bad)
#pragma unroll
                    for (int p = 0; p < kPasses; ++p)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int bytes = ANY ? row_bytes - 16 * piece - 4 * x : 4;
                            const uint32_t nan = (F8 ? 0x7f7f7f7fu : 0x7fff7fffu) & (bytes >= 4 ? 0xffffffffu : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1u);
                            kx[p][x] = missing.bad >> (p * kAtOnce + line) & 1 ? nan : kx[p][x];
                        }
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
            if (some_hidden) {
                uint32_t mark = 0;
#pragma unroll
                for (int p = 0; p < kPasses; ++p) watch<DT, F8>(mark, vx[p]);
                if (__any(seen_odd<DT, F8>(mark))) {
#pragma unroll
                    for (int p = 0; p < kPasses; ++p) take_out<DT, F8>(vx[p]);
                    sh.odd = 1;
                }
            }
            {
                char *const kt = buf + line * T::kPitchK + (F8 ? 32 : 16) * piece, *const vt = buf + T::kTokens * T::kPitchK + line * T::kPitchV + (F8 ? 32 : 16) * piece;
                auto put = [&](auto type, char *to, const uint32_t (&x)[4]) {
                    constexpr int To = decltype(type)::value;
                    if (F8) {
                        *(u32x4 *)to = u32x4{widen<To, false>(x[0]), widen<To, true>(x[0]), widen<To, false>(x[1]), widen<To, true>(x[1])};
                        *(u32x4 *)(to + 16) = u32x4{widen<To, false>(x[2]), widen<To, true>(x[2]), widen<To, false>(x[3]), widen<To, true>(x[3])};
                    } else {
                        *(u32x4 *)to = u32x4{x[0], x[1], x[2], x[3]};
                    }
                };
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    put(std::integral_constant<int, DT>(), kt + p * kAtOnce * T::kPitchK, kx[p]);
                    put(std::integral_constant<int, PT>(), vt + p * kAtOnce * T::kPitchV, vx[p]);
                }
            }
            if (i + 1 < cur.last) {
                missing = tree_aim<T>(sh.spots[wave], mine_at, by, from, cur, first_of(cur, i + 1) + mine_at, number);
                if (SHORT) fetch_all(from);
                number = look_up(cur, row, by.page, i + 2 < cur.last, first_of(cur, i + 2) + mine_at);
            } else {
                sh.spots[wave][0][mine_at] = from.k_none;
                sh.spots[wave][1][mine_at] = from.v_none;
                __builtin_amdgcn_wave_barrier();
                if (more) {
                    next = unit_after<T>(cur, end);
                    number = look_up(next, table_row(next), by.page, true, first_of(next, next.tile) + mine_at);
                }
            }
            lds_barrier();

            // -- scores of tokens t0 + 32 u + 8 (x / 4) + 4 half + x % 4
            const uint32_t t0 = first_of(cur, i) + wt * T::kMine;
            const char *const kt = buf + (wt * T::kMine + l32) * T::kPitchK + 16 * half;
            f32x16 s[SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
#pragma unroll
                for (int x = 0; x < 16; ++x) s[u][x] = 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    s[u] = mfma32<DT>(*(const u32x4 *)(kt + 32 * u * T::kPitchK + 32 * k), q[k], s[u]);
                    constexpr int kEvery = SUBS * KS / kPasses;
                    if (!SHORT && (u * KS + k + 1) % kEvery == 0) fetch(kx[(u * KS + k) / kEvery], from, 0, (u * KS + k) / kEvery);
                }
            }
            // (four operands on their way from LDS ahead of the products)
            __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
#pragma unroll
            for (int n = 0; n < SUBS * KS; ++n) {
                __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
            }
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
            if (__any(top - m > lag)) {                      // (also the first that is seen: m is -inf)
                const float to = kTreeLift<PT> - (top == -INFINITY ? 0.f : top * to_log2);
                const float shrink = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(to - base);
                l *= shrink;
#pragma unroll
                for (int j = 0; j < DB; ++j) o[j] *= shrink;
                m = top;
                base = to;
            }
            // Scores so large that `base` is rounded by more than 2^-8: the maximum is taken off before.
            float add = base;
            if (__any(fabsf(base) > 0x1p16f)) {
#pragma unroll
                for (int u = 0; u < SUBS; ++u) s[u] -= m == -INFINITY ? 0.f : m;
                add = kTreeLift<PT>;
            }
            u32x4 p[2 * SUBS], rest[TWO ? 2 * SUBS : 1];
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int x = 0; x < 16; x += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][x], to_log2, add)), p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][x + 1], to_log2, add));
                    if constexpr (TWO) {
                        const uint32_t first = first_term<PT>(p0, p1);
                        p[2 * u + x / 8][x % 8 / 2] = first;
                        rest[2 * u + x / 8][x % 8 / 2] = Elem<PT>::pack2(second_term<PT, F8>(p0, Elem<PT>::to_float((uint16_t)first)),
                                                                         second_term<PT, F8>(p1, Elem<PT>::to_float((uint16_t)(first >> 16))));
                        l += p0;
                        l += p1;
                    } else {
                        p[2 * u + x / 8][x % 8 / 2] = Elem<PT>::pack2(p0, p1);
                        l = add_both(p[2 * u + x / 8][x % 8 / 2], l);
                    }
                }
            // -- values: lane (dimension 32 j + l32, half) has tokens 16 k + 4 half + 0 .. 3 and 8 behind those
            const LdsBytes vt = (LdsBytes)(buf + T::kTokens * T::kPitchK) + (wt * T::kMine + 4 * half + (lane & 15) / 4) * T::kPitchV + 32 * (lane >> 4 & 1) + 8 * (lane & 3);
#pragma unroll
            for (int k = 0; k < 2 * SUBS; ++k)
#pragma unroll
                for (int j = 0; j < DB; ++j) {
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPiece)(vt + 16 * k * T::kPitchV + 64 * j)));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPiece)(vt + (16 * k + 8) * T::kPitchV + 64 * j)));
                    const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
                    o[j] = mfma32<PT>(v, p[k], o[j]);
                    if constexpr (TWO) o[j] = mfma32<PT>(v, rest[k], o[j]);
                    constexpr int kEvery = 2 * SUBS * DB / kPasses;
                    if (!SHORT && (k * DB + j + 1) % kEvery == 0) fetch(vx[(k * DB + j) / kEvery], from, 1, (k * DB + j) / kEvery);
                }
            __builtin_amdgcn_sched_group_barrier(kDsRead, 8, 1);
#pragma unroll
            for (int n = 0; n < 2 * SUBS * DB; ++n) {
                __builtin_amdgcn_sched_group_barrier(kMatrix, TWO ? 2 : 1, 1);
                __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 1);
            }
        }
    }
    tree_count_in<DT, F8, DC, T>(sh, unfinished);
}

// ------------------------------------------------------------------ host
template <int DT, bool F8, int DC, int WR, TreeRows ROWS> static int launch_wide_rows(const PagedTreeAttentionArgs &a, const TreeWork &w, hipStream_t stream) {
    typedef TreeWide<DC, WR> T;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_tree_wide_kernel<DT, F8, DC, WR, ROWS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (attr != hipSuccess) return BA_ERR_LAUNCH;
    return tree_launch<DT, DC, T>(paged_tree_wide_kernel<DT, F8, DC, WR, ROWS>, a, w, stream);
}
template <int DT, bool F8, int DC, int WR> static int launch_wide_waves(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, hipStream_t stream) {
    if constexpr (DC == 64)
        if (rows == kTreeShort) return launch_wide_rows<DT, F8, DC, WR, kTreeShort>(a, w, stream);
    return rows == kTreePieces ? launch_wide_rows<DT, F8, DC, WR, kTreePieces>(a, w, stream) : launch_wide_rows<DT, F8, DC, WR, kTreeAny>(a, w, stream);
}
template <int DT, bool F8, int DC> static int launch_wide_dims(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream) {
    if constexpr (DC == 64)
        if (waves == 2) return launch_wide_waves<DT, F8, DC, 2>(a, w, rows, stream);
    return launch_wide_waves<DT, F8, DC, 4>(a, w, rows, stream);
}
template <int DT, bool F8> int launch_tree_wide(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream) {
    switch (dim_class(a.dim)) {
        case 64: return launch_wide_dims<DT, F8, 64>(a, w, rows, waves, stream);
        case 128: return launch_wide_dims<DT, F8, 128>(a, w, rows, waves, stream);
        default: return launch_wide_dims<DT, F8, 256>(a, w, rows, waves, stream);
    }
}

}  // namespace ba
