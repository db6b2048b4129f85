// Attention of drafted tokens for few rows a key head (units of 16 or 32; tree_rows).
//
// Every key and value is read once, so memory traffic is the floor, as for one query per request (paged_attention_kernel.hpp), and the tile is worked
// on in the same way: nothing of the cache passes through LDS, the four wavefronts take 32 tokens each, scores are K Q^T on the
// 16 x 16 x 32 matrix instruction with tokens as rows and one or two sets of 16 columns, which are rows of the queries here; a lane turns
// the small matrix of its eight tokens' values in registers; probabilities enter the second product as two 16-bit terms.  A token's place is
// worked out by one lane and handed to those that load it through LDS, whatever the pages are.
// What bounds it: memory where requests are long (64 requests of 4000 tokens, 8 key heads of 128, 1.05 GB: 16 rows a key head 168 us, 6.3 TB/s; 32 rows
// 176; in 8 bits, 0.52 GB, 96 and 158); where they are short a unit's beginning and end, some 6 us, and the sums over all requests before (492 units of 1000 tokens, 80 dimensions
// 43.5 us, 3.0 TB/s; one request of 500 tokens 14.5).
#pragma once
#include "paged_tree_attention.hpp"

namespace ba {

template <int DC_, int SETS> struct TreeFew {
    static constexpr int DC = DC_, kRows = 16 * SETS, kGroups = kTreeWaves, kWaveRows = kRows;
    static constexpr int kTokens = 32 * kTreeWaves, kStaged = 32;
    static constexpr int kDims = DC < 128 ? DC : 128, kPitch = kDims + 4, kPart = kRows * kPitch * 4, kLds = kTreeWaves * kPart;
    // Workgroups of a compute unit, by registers (128 dimensions: two sets with two workgroups, and registers in memory, 233 us for 64 requests of
    // 4000 tokens and 32 rows a key head, with one 181; one set with three 579 for 500 of 1000, with two 384).
    static constexpr int kResident = DC == 64 ? (SETS == 2 ? 2 : 3) : DC == 128 && SETS == 1 ? 2 : 1;
};

// DC: dimensions that the registers hold (64, 128, 256: with one set).
template <int DT, bool F8, int DC, int SETS, TreeRows ROWS>
__global__ void __launch_bounds__(kTreeThreads, (TreeFew<DC, SETS>::kResident)) paged_tree_few_kernel(TreeArgs) {
    typedef TreeFew<DC, SETS> T;
    constexpr bool ANY = ROWS != kTreePieces, SHORT = ROWS == kTreeShort;
    constexpr int EB = F8 ? 1 : 2;           // bytes of an element
    constexpr int PW = DC / 16;              // dimensions of a value's row that a lane holds
    constexpr int E = PW * EB < 16 ? PW : 16 / EB, N = E * EB / 4;      // those of one load, its dwords
    constexpr int L = PW / E;                // loads; load k of lane x of a row: dimensions 16 E k + E x ..
    constexpr int KL = DC * EB / 64, QK = DC / 32;           // loads of a key's row, 16 bytes a lane; operands of the queries
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4, wave = uniform((int)threadIdx.x >> 6);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ TreeLds<T> sh;
    int unfinished = 0;
    TreeUnit cur, next;
    int group;
    const int64_t end = tree_deal<T>(sh, next, group);
    if (end < 0) return;

    const int mine_at = lane & 31;
    uint32_t kx[2][KL][4], vx[8][L][N];
    Missing missing = {};                                    // of the wavefront's tile
    u32x4 q[SETS][QK];
    auto first_of = [&](const TreeUnit &u, int i) { return (uint32_t)u.d.start + (uint32_t)i * T::kTokens + 32 * wave; };
    // The rows of a tile: a lane has 16-byte pieces of tokens l16 and 16 + l16 of the keys, E dimensions at a time of tokens 16 i + 4 g + j of the values.
    // (Pieces behind a row's end: the row's last bytes.)
    auto load_keys = [&](const TreeBases &from) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const char *const p = from.k + sh.spots[wave][0][16 * i + l16];
#pragma unroll
            for (int k = 0; k < KL; ++k) {
                const int b = 64 * k + 16 * g;
                if (SHORT) load_part<4>(kx[i][k], p + b, from.row_bytes - b);
                else load_stream<4>(kx[i][k], p + (!ANY && DC > 64 && 64 * (k + 1) <= DC / 2 * EB ? b : min(b, from.row_bytes - 16)));      // (dim > DC / 2)
            }
        }
    };
    auto load_values = [&](const TreeBases &from) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const char *const p = from.v + sh.spots[wave][1][16 * (i / 4) + 4 * g + i % 4];
#pragma unroll
            for (int k = 0; k < L; ++k) {
                const int b = EB * E * (16 * k + l16);
                if (SHORT) load_part<N>(vx[i][k], p + b, from.row_bytes - b);
                else load_stream<N>(vx[i][k], p + min(b, from.row_bytes - 4 * N));
            }
        }
    };
    // Pieces that the rows' end cuts off, or that lie behind it, once they are there.
    auto settle = [&](auto &x, int past) {
        constexpr int M = sizeof(x) / 4;
        if constexpr (ANY) shift_down<M>(x, max(past, 0));
        else
#pragma unroll
            for (int i = 0; i < M; ++i) x[i] = past > 0 ? 0u : x[i];
    };
    auto settle_keys = [&](int row_bytes) {
        if (SHORT) return;
#pragma unroll
        for (int k = 0; k < KL; ++k)
            if (64 * (k + 1) > row_bytes)
#pragma unroll
                for (int i = 0; i < 2; ++i) settle(kx[i][k], 64 * k + 16 * g - (row_bytes - 16));
    };
    auto settle_values = [&](int row_bytes) {
        if (SHORT) return;
#pragma unroll
        for (int k = 0; k < L; ++k)
            if (16 * EB * E * (k + 1) > row_bytes)
#pragma unroll
                for (int i = 0; i < 8; ++i) settle(vx[i][k], EB * E * (16 * k + l16) - (row_bytes - 4 * N));
    };

    bool any = false, more = true;
    int32_t number = look_up(next, table_row(next), tree_args().a.page, true, first_of(next, next.tile) + mine_at);
    f32x4 o[SETS][PW];
    float m[SETS], l[SETS];
    for (;;) {
        // ---- the next unit's first tile and queries are on their way while this one is finished
        if (more) {
            const PagedTreeAttentionArgs &a = tree_args().a;
            const TreeBases from = tree_bases<EB>(next);
            missing = tree_aim<T>(sh.spots[wave], mine_at, tree_steps(), from, next, first_of(next, next.tile) + mine_at, number);
            load_keys(from);
            load_values(from);
            const int me = opaque(lane);
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                const TreeRow t = tree_row(a, tree_args().w, next.d, next.h, (int64_t)next.block * T::kRows + 16 * z + (me & 15));
                const char *const p = a.q + t.head * a.q_head_bytes + (int64_t)(next.d.row0 + t.node) * a.q_row_bytes;
#pragma unroll
                for (int k = 0; k < QK; ++k) {
                    const int d0 = F8 ? 64 * (k / 2) + 16 * (me >> 4) + 8 * (k % 2) : 32 * k + 8 * (me >> 4);      // (the order in which the keys arrive)
                    uint32_t x[4] = {0, 0, 0, 0};
                    if (t.there && d0 < a.dim) {
                        if (ANY) load_part<4>(x, p + 2 * d0, 2 * (a.dim - d0));
                        else load_stream<4>(x, p + 2 * d0);
                    }
                    q[z][k] = u32x4{x[0], x[1], x[2], x[3]};
                }
            }
        }
        if (any) {
            const int me = opaque((int)threadIdx.x), my16 = me & 15, my_g = me >> 4 & 3;
            const float v_scale = F8 ? tree_args().a.v.scale[cur.h] : 1.f;
            bool odd = false;
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
                l[z] = quad_column_sum(l[z]);
                if (my_g == 0) { sh.m[wave][16 * z + my16] = m[z]; sh.l[wave][16 * z + my16] = l[z]; }
            }
#pragma unroll
            for (int c = 0; c < DC; c += T::kDims) {
                // lane (g, l16) has dimensions 16 E k + E (4 g + i) + x of rows l16 and 16 + l16, j = E k + x
#pragma unroll
                for (int z = 0; z < SETS; ++z) {
                    float *const mineo = (float *)(lds + wave * T::kPart) + (16 * z + my16) * T::kPitch;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < PW; j += 4) {
                            const int dim = 16 * E * (j / E) + E * (4 * my_g + i) + j % E;
                            if (DC == T::kDims || dim / T::kDims == c / T::kDims)
                                *(f32x4 *)(mineo + dim - c) = f32x4{o[z][j][i], o[z][j + 1][i], o[z][j + 2][i], o[z][j + 3][i]};
                        }
                }
                lds_barrier();
                odd = uniform(sh.odd) != 0;
                tree_store<DT, T>(sh, group, lds, cur, me, c, v_scale);
                lds_barrier();
            }
            tree_end<DT, F8, T>(sh, group, cur, me, odd, unfinished);
            if (!more) break;
        }
        cur = next;
        any = true;
        const PagedTreeAttentionArgs &a = tree_args().a;
        const Draft &d = cur.d;
        const TableRow row = table_row(cur);
        Sight sight[SETS];
        const int me = opaque(lane);
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            sight[z] = sight_of(a, d, tree_row(a, tree_args().w, d, cur.h, (int64_t)cur.block * T::kRows + 16 * z + (me & 15)), 0);
            if (a.window) sight[z].from = window_from(a, d, sight[z]);
            if (wave == 0 && me < 16) sh.row_from[16 * z + me] = sight[z].from;
        }
        const int window = uniform(a.window), words = uniform(a.words), row_bytes = uniform(EB * a.dim);
        const TreeSteps by = tree_steps();
        const TreeBases from = tree_bases<EB>(cur);
        const float to_log2 = a.scale * kLog2e * (F8 ? a.k.scale[cur.h] : 1.f);
#pragma unroll
        for (int z = 0; z < SETS; ++z) {
            m[z] = -INFINITY; l[z] = 0.f;
#pragma unroll
            for (int j = 0; j < PW; ++j) o[z][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        more = tree_next(cur) < end;
        number = look_up(cur, row, by.page, cur.tile + 1 < cur.last, first_of(cur, cur.tile + 1) + mine_at);
        for (int i = cur.tile; i < cur.last; ++i) {
            const uint32_t t0 = first_of(cur, i);
            const bool some_hidden = hidden<T>(d, window, t0), follows = i + 1 < cur.last;
            settle_keys(row_bytes);
            settle_values(row_bytes);
            // Tokens that are not there: values of zero.  On a page outside the cache: keys of NaN as well, which is the result of a row that sees them
            // (zeros behind the row's end: the queries' zeros there would make NaN of those too).
            if (missing.any) {
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    const bool none = (uint32_t)missing.any >> (16 * (y / 4) + 4 * g + y % 4) & 1;
#pragma unroll
                    for (int k = 0; k < L; ++k)
#pragma unroll
                        for (int x = 0; x < N; ++x) vx[y][k][x] = none ? 0u : vx[y][k][x];
                }
                if (missing.bad)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int k = 0; k < KL; ++k)
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const int bytes = row_bytes - 64 * k - 16 * g - 4 * x;
                                const uint32_t nan = (F8 ? 0x7f7f7f7fu : 0x7fff7fffu) & (bytes >= 4 ? 0xffffffffu : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1u);
                                kx[y][k][x] = (uint32_t)missing.bad >> (16 * y + l16) & 1 ? nan : kx[y][k][x];
                            }
            }
            if (some_hidden) {
                uint32_t mark = 0;
#pragma unroll
                for (int y = 0; y < 8; ++y)
#pragma unroll
                    for (int k = 0; k < L; ++k) watch<DT, F8>(mark, vx[y][k]);
                if (__any(seen_odd<DT, F8>(mark))) {
#pragma unroll
                    for (int y = 0; y < 8; ++y)
#pragma unroll
                        for (int k = 0; k < L; ++k) take_out<DT, F8>(vx[y][k]);
                    sh.odd = 1;
                }
            }
            // -- scores of tokens t0 + 16 y + 4 g + j
            f32x4 sc[SETS][2];
#pragma unroll
            for (int z = 0; z < SETS; ++z)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < QK; ++k) s = product<DT, F8, F8 ? 16 : 8>(kx[y][F8 ? k / 2 : k], F8 ? k % 2 : 0, q[z][k], s);
                    sc[z][y] = s * to_log2;
                }
            // the next tile's keys are asked for as soon as the scores have used this one's, its values behind the second product
            if (follows) {
                missing = tree_aim<T>(sh.spots[wave], mine_at, by, from, cur, first_of(cur, i + 1) + mine_at, number);
                load_keys(from);
                number = look_up(cur, row, by.page, i + 2 < cur.last, first_of(cur, i + 2) + mine_at);
            } else if (more) {
                next = unit_after<T>(cur, end);
                number = look_up(next, table_row(next), by.page, true, first_of(next, next.tile) + mine_at);
            }
            if (some_hidden) {
#pragma unroll
                for (int z = 0; z < SETS; ++z) {
                    const uint32_t see = (uint32_t)sight[z](d, words, t0) >> (4 * g);
#pragma unroll
                    for (int x = 0; x < 8; ++x) sc[z][x / 4][x % 4] = see >> (16 * (x / 4) + x % 4) & 1 ? sc[z][x / 4][x % 4] : -INFINITY;
                }
            }
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
                for (int x = 0; x < 8; ++x) {
                    p[x] = __builtin_amdgcn_exp2f(sc[z][x / 4][x % 4] - base);
                    l[z] += p[x];
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    hi[z][x] = first_term<DT>(p[2 * x], p[2 * x + 1]);
                    lo[z][x] = Elem<DT>::pack2(second_term<DT, F8>(p[2 * x], Elem<DT>::to_float((uint16_t)hi[z][x])),
                                               second_term<DT, F8>(p[2 * x + 1], Elem<DT>::to_float((uint16_t)(hi[z][x] >> 16))));
                }
            }
            // -- values
#pragma unroll
            for (int j = 0; j < PW; ++j) {
                uint32_t f[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int k = j / E, x = j % E;
                    if (F8) {
                        // byte x of both rows next to each other, then widened together
                        const uint32_t both = __builtin_amdgcn_perm(vx[2 * y + 1][k][x / 4], vx[2 * y][k][x / 4], 0x0c0c0400u + (uint32_t)(x % 4) * 0x0101u);
                        f[y] = widen<DT, false>(both);
                    } else {
                        f[y] = __builtin_amdgcn_perm(vx[2 * y + 1][k][x / 2], vx[2 * y][k][x / 2], x % 2 ? 0x07060302u : 0x05040100u);
                    }
                }
                const u32x4 v = {f[0], f[1], f[2], f[3]};
#pragma unroll
                for (int z = 0; z < SETS; ++z) {
                    o[z][j] = Elem<DT>::mfma(v, hi[z], o[z][j]);
                    o[z][j] = Elem<DT>::mfma(v, lo[z], o[z][j]);
                }
            }
            if (follows) load_values(from);
        }
    }
    tree_count_in<DT, F8, DC, T>(sh, unfinished);
}

// ------------------------------------------------------------------ host
template <int DT, bool F8, int DC, int SETS, TreeRows ROWS> static int launch_few_rows(const PagedTreeAttentionArgs &a, const TreeWork &w, hipStream_t stream) {
    typedef TreeFew<DC, SETS> T;
    if constexpr (T::kLds > 65536) {
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_tree_few_kernel<DT, F8, DC, SETS, ROWS>),
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
        if (attr != hipSuccess) return BA_ERR_LAUNCH;
    }
    return tree_launch<DT, DC, T>(paged_tree_few_kernel<DT, F8, DC, SETS, ROWS>, a, w, stream);
}
template <int DT, bool F8, int DC, int SETS> static int launch_few_dims(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, hipStream_t stream) {
    if constexpr (DC == 64)
        if (rows == kTreeShort) return launch_few_rows<DT, F8, 64, SETS, kTreeShort>(a, w, stream);
    return rows == kTreePieces ? launch_few_rows<DT, F8, DC, SETS, kTreePieces>(a, w, stream) : launch_few_rows<DT, F8, DC, SETS, kTreeAny>(a, w, stream);
}
template <int DT, bool F8, int DC> static int launch_few_sets(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int sets, hipStream_t stream) {
    if constexpr (DC <= 128)
        if (sets == 2) return launch_few_dims<DT, F8, DC, 2>(a, w, rows, stream);
    return launch_few_dims<DT, F8, DC, 1>(a, w, rows, stream);
}
template <int DT, bool F8> int launch_tree_few(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int sets, hipStream_t stream) {
    switch (dim_class(a.dim)) {
        case 64: return launch_few_sets<DT, F8, 64>(a, w, rows, sets, stream);
        case 128: return launch_few_sets<DT, F8, 128>(a, w, rows, sets, stream);
        default: return launch_few_sets<DT, F8, 256>(a, w, rows, sets, stream);
    }
}

}  // namespace ba
