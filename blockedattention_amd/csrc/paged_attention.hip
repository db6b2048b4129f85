// Attention of one new query per request over a paged key-value cache.
//
// out[h][r] = sum_t softmax_t(scale q[h][r] . K[t]) V[t] over the request's tokens t.  Every key and value is read once and
// takes part in 4 x group operations a byte pair, so memory traffic is the floor; what the kernel is built for is bytes in
// flight on every compute unit, whatever the lengths are.
//
// Split.  A unit is a request and up to 16 query heads that share a key head.  Its tokens are cut into tiles of 32, and
// the tiles of all units, in order, are dealt out to the workgroups in equal shares (the lengths are on the GPU only, so
// every workgroup adds them up itself).  A workgroup goes through its share unit by unit, its four wavefronts taking every
// fourth tile each; at the end of a unit their results are joined in LDS.  A unit that lies in one share is done
// then; for others each workgroup leaves its maximum, sum and fp32 accumulators, and a second small kernel joins them.
//
// One tile.  Scores: S[token][head] = K Q^T with 16 tokens as the rows of a 16 x 16 x 32 matrix instruction; a lane's
// operand is 16 bytes of one key, loaded straight from the cache.  A lane then holds the scores of tokens 4g..4g+3 of both
// halves of the tile for one head (g = lane / 16): packed to 16 bits these are, as they are, its operand of the second
// product if the reduction runs over the tokens in the order (half, g, i) -- no lane exchanges a probability.  Values: O[d][head]
// = V^T P.  A lane loads 2 or more adjacent dimensions of its eight tokens (16 lanes cover a row: whole lines) and turns
// the small matrix in registers: the operand of dimension j is made of the j-th halves of its eight rows.  Nothing of the cache
// passes through LDS.
#include <algorithm>
#include <type_traits>

#include "ba_device.hpp"
#include "ba_host.hpp"
#include "paged.hpp"

namespace ba {

constexpr int kPagedWaves = 4;
constexpr int kPagedThreads = 64 * kPagedWaves;
constexpr int kPagedTile = 32;               // tokens
constexpr int kPagedHeads = 16;              // query heads of a unit at most
constexpr int kPagedShare = kPagedWaves;     // tiles of a workgroup at least
constexpr int kPagedWhole = 8;               // units of up to so many tiles are not split between workgroups

// Probabilities are scaled by a power of two that keeps those of 2^-39 (and not 2^-24) of the largest apart from
// zero in fp16; it is in the sums as well and drops out.
template <int DT> constexpr float kLift = DT == 0 ? 14.f : 0.f;

struct PagedPart {                           // what a workgroup leaves for a unit that others work on too
    float m, l;
};
// Units of which a workgroup does the first tiles and not the last ones: who has to join what.
struct PagedJoin {
    int32_t request, unit, first, parts;     // parts 0: nothing to join; first: workgroup
};

struct PagedWork {
    PagedJoin *joins;                        // one entry a unit, or a workgroup where there are fewer of those
    PagedPart *parts;                        // [2 * groups][kPagedHeads]
    float *sums;                             // [2 * groups][rows][pitch]
    int32_t groups, by_unit, tiles_a_head, rows, pitch;   // tiles_a_head: units of a key head; rows: query heads of the largest unit
};

// Two e4m3 values (HI: the upper two bytes) as two 16-bit numbers: exact in either type.
template <int DT, bool HI> __device__ __forceinline__ uint32_t widen(uint32_t x) {
    if (DT == 0) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x, 1.f, HI));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)x, 1.f, HI));
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

// What is known of the head dimension: it fills the registers (64, 128, 256), it is whole pieces (16 bytes of a key), or neither.
enum Shape { kFull, kPieces, kAny };
// What is known of the pages: whole halves of tiles, whole groups of four tokens, nothing.
enum Pages { kHalves, kFours, kTokens };

struct Visible {
    int first, len;                          // tokens first .. len - 1 are seen
    __device__ __forceinline__ int start() const { return first & ~(kPagedTile - 1); }
    // a request without tokens has one tile: its zeros are written by whoever gets it
    __device__ __forceinline__ int tiles() const { return len > first ? (len - start() + kPagedTile - 1) / kPagedTile : 1; }
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

// DC: dimensions that the registers hold (64, 128, 256).
template <int DT, bool F8, int DC, Shape SHAPE, Pages PAGES>
__global__ void __launch_bounds__(kPagedThreads, DC == 64 ? 4 : DC == 128 ? 3 : 2)
paged_attention_kernel(PagedAttentionArgs a, PagedWork w) {
    constexpr int EB = F8 ? 1 : 2;           // bytes of an element
    constexpr int KK = DC / 32;              // matrix instructions of a half's scores
    constexpr int KL = KK * EB / 2;          // 16-byte pieces of a key that a lane holds
    constexpr int PW = DC / 16;              // dimensions of a value that a lane holds
    constexpr int VN = PW * EB / 4 > 4 ? 4 : PW * EB / 4;      // dwords of one load of them
    constexpr int VL = PW * EB / 4 / VN;     // loads
    const int lane = lane_id(), l16 = lane & 15, g = lane >> 4, wave = uniform((int)threadIdx.x >> 6);
    const int units = a.heads * w.tiles_a_head;

    extern __shared__ __attribute__((aligned(16))) float lds[];           // [waves][rows][DC + 4]
    __shared__ int64_t scan[kPagedWaves];
    __shared__ Place places[2];
    __shared__ float wave_m[kPagedWaves][kPagedHeads], wave_l[kPagedWaves][kPagedHeads];

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
    const int64_t groups = min((int64_t)w.groups, (total + kPagedShare - 1) / kPagedShare);
    const int64_t group = blockIdx.x;
    if (group >= groups) {
        if (!w.by_unit && threadIdx.x == 0) w.joins[group].parts = 0;
        return;
    }
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
    int request = uniform(places[0].request), unit = uniform(places[0].unit), tile = uniform(places[0].tile);
    int64_t at = uniform64(places[0].at);
    const int64_t end = uniform64(places[1].at);
    Visible see = {uniform(places[0].see.first), uniform(places[0].see.len)};
    PagedJoin join = {0, 0, 0, 0};

    while (at < end) {
        const int first = see.first, len = see.len, n = see.tiles(), start = see.start();
        const int last = (int)min((int64_t)n, tile + (end - at));      // tiles of this unit in this share: [tile, last)
        const int h = unit / w.tiles_a_head, q0 = h * a.group + (unit - h * w.tiles_a_head) * w.rows;
        const int rows = min(w.rows, (h + 1) * a.group - q0);
        const char *const kh = a.k.base + h * a.k.head_bytes, *const vh = a.v.base + h * a.v.head_bytes;
        typedef const __attribute__((address_space(4))) int32_t *Row;
        const Row row = (Row)(uintptr_t)(a.table + request * a.table_stride);

        // queries: head l16 in the order of dimensions in which the keys arrive
        u32x4 qf[KK];
#pragma unroll
        for (int i = 0; i < KK; ++i) {
            const int d = F8 ? 64 * (i / 2) + 16 * g + 8 * (i % 2) : 32 * i + 8 * g;
            uint32_t x[4] = {0, 0, 0, 0};
            const char *const p = a.q + (q0 + l16) * a.q_head_bytes + request * a.q_row_bytes + 2 * d;
            if (l16 < rows) {
                if (SHAPE == kAny) load_part<4>(x, p, 2 * (a.dim - d));
                else if (SHAPE == kFull || d < a.dim) load_stream<4>(x, p);
            }
            qf[i] = u32x4{x[0], x[1], x[2], x[3]};
        }
        const float to_log2 = a.scale * kLog2e * (F8 ? a.k.scale[h] : 1.f);

        f32x4 o[PW];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int j = 0; j < PW; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};

        // Pages and lines of a tile.  Tokens that are not seen may have no page (any more): a half, a group of four or a token
        // without any that is seen borrows the place of one with.  Page numbers outside the cache become page 0 and poison
        // the result.
        constexpr int NK = 2, NV = PAGES == kHalves ? 0 : PAGES == kFours ? 2 : 8;
        int32_t page[NK + NV], line[NK + NV];
        bool poison = a.pages == 0;
        auto look_up = [&](int t0) {
            if (PAGES == kHalves) {
                int t[2] = {t0, t0 + 16};
                if (t[1] >= len) t[1] = t[0];
                if (t[0] + 16 <= first) t[0] = t[1];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t c = a.page.div((uint32_t)t[i]);
                    page[i] = row[c];
                    line[i] = t[i] - (int)(c * a.page.d);
                }
            } else {
                constexpr int four = PAGES == kFours ? 3 : 0;
#pragma unroll
                for (int i = 0; i < NK + NV; ++i) {
                    const int mine = i < NK ? t0 + 16 * i + l16
                                     : PAGES == kFours ? t0 + 16 * (i - NK) + 4 * g
                                                       : t0 + 16 * ((i - NK) / 4) + 4 * g + (i - NK) % 4;
                    const int t = min(max(mine & ~four, first & ~four), (len - 1) & ~four) + (mine & four);
                    const uint32_t c = a.page.div((uint32_t)t);
                    page[i] = a.table[request * a.table_stride + c];
                    line[i] = t - (int)(c * a.page.d);
                }
            }
        };
        auto checked = [&](int i) {
            const int32_t p = PAGES == kHalves ? uniform(page[i]) : page[i];
            const bool bad = (uint32_t)p >= (uint32_t)a.pages;
            poison |= bad;
            return bad ? 0 : p;
        };
        // Pieces that are not there (kPieces) are loaded from the row's front: those of a key count as zeros, those of a value
        // make results that nobody stores.
        uint32_t kx[2][KL][4], vx[8][VL][VN];
        auto load_keys = [&] {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int32_t p = checked(i), ln = PAGES == kHalves ? uniform(line[i]) : line[i];
                const char *const base = kh + p * a.k.page_bytes + (int64_t)ln * a.k.token_bytes;
                const uint32_t mine = PAGES == kHalves ? (uint32_t)(l16 * a.k.token_bytes) : 0u;
#pragma unroll
                for (int k = 0; k < KL; ++k) {
                    const uint32_t b = 64 * k + 16 * g;
                    if (SHAPE == kAny) load_part<4>(kx[i][k], base + (mine + b), EB * a.dim - (int)b);
                    else if (SHAPE == kPieces) load_stream<4>(kx[i][k], base + (mine + ((int)b < EB * a.dim ? b : 0u)));
                    else load_stream<4>(kx[i][k], base + (mine + 16u * g) + 64 * k);
                }
            }
        };
        auto load_values = [&] {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int from = PAGES == kHalves ? i / 4 : PAGES == kFours ? NK + i / 4 : NK + i;
                const int32_t p = checked(from), ln = PAGES == kHalves ? uniform(line[from]) : line[from];
                const char *const base = vh + p * a.v.page_bytes + (int64_t)ln * a.v.token_bytes;
                const uint32_t mine = PAGES == kHalves ? (uint32_t)((4 * g + i % 4) * a.v.token_bytes) : PAGES == kFours ? (uint32_t)(i % 4 * a.v.token_bytes) : 0u;
#pragma unroll
                for (int k = 0; k < VL; ++k) {
                    const uint32_t b = EB * PW * l16 + 16 * k;
                    if (SHAPE == kAny) load_part<VN>(vx[i][k], base + (mine + b), EB * a.dim - (int)b);
                    else if (SHAPE == kPieces) load_stream<VN>(vx[i][k], base + (mine + ((int)b < EB * a.dim ? b : 0u)));
                    else load_stream<VN>(vx[i][k], base + (mine + (uint32_t)(EB * PW * l16)) + 16 * k);
                }
            }
        };
        // The tile that begins with token t0; MORE: the wavefront's next one follows, whose keys are asked for as soon as the
        // scores have used this one's, and its values likewise.
        auto attend = [&](auto more, int t0) {
            constexpr bool MORE = decltype(more)::value;
            if (SHAPE == kPieces) {
#pragma unroll
                for (int k = 0; k < KL; ++k)
                    if (64 * k + 64 > EB * a.dim) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int x = 0; x < 4; ++x) kx[i][k][x] = 64 * k + 16 * g < EB * a.dim ? kx[i][k][x] : 0u;
                    }
            }
            // ---- scores of tokens t0 + 16 i + 4 g + e
            f32x4 sc[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KL; ++k) {
                    if (F8) {
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t x = kx[i][k][2 * half], y = kx[i][k][2 * half + 1];
                            sc[i] = Elem<DT>::mfma(u32x4{widen<DT, false>(x), widen<DT, true>(x), widen<DT, false>(y), widen<DT, true>(y)},
                                                   qf[(2 * k + half) % KK], sc[i]);
                        }
                    } else {
                        sc[i] = Elem<DT>::mfma(u32x4{kx[i][k][0], kx[i][k][1], kx[i][k][2], kx[i][k][3]}, qf[k % KK], sc[i]);
                    }
                }
                sc[i] *= to_log2;
            }
            if (MORE) load_keys();
            if (t0 < first || t0 + kPagedTile > len) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
                    const bool seen = t >= first && t < len;
                    sc[i / 4][i % 4] = seen ? sc[i / 4][i % 4] : -INFINITY;
#pragma unroll
                    for (int k = 0; k < VL; ++k)
#pragma unroll
                        for (int x = 0; x < VN; ++x) vx[i][k][x] = seen ? vx[i][k][x] : 0u;    // (a probability of 0 times what lies there may be NaN)
                }
            }
            float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                              fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
            top = fmaxf(m, quad_column_max(top));
            const float base = (top == -INFINITY ? 0.f : top) - kLift<DT>;
            if (__any(top != m)) {
                const float shrink = __builtin_amdgcn_exp2f(m - kLift<DT> - base);
                l *= shrink;
#pragma unroll
                for (int j = 0; j < PW; ++j) o[j] *= shrink;
                m = top;
            }
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = __builtin_amdgcn_exp2f(sc[i / 4][i % 4] - base);
                l += p[i];
            }
            // Probabilities in two 16-bit terms: one alone would cost as much accuracy as the rounding of the result, and the
            // matrix unit has time to spare.
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hi[i] = Elem<DT>::pack2(p[2 * i], p[2 * i + 1]);
                lo[i] = Elem<DT>::pack2(p[2 * i] - Elem<DT>::to_float((uint16_t)hi[i]), p[2 * i + 1] - Elem<DT>::to_float((uint16_t)(hi[i] >> 16)));
            }
            // ---- values
#pragma unroll
            for (int j = 0; j < PW; ++j) {
                uint32_t f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (F8) {
                        // byte j of both rows next to each other, then widened together
                        const uint32_t both = __builtin_amdgcn_perm(vx[2 * i + 1][j / 4 / VN][j / 4 % VN], vx[2 * i][j / 4 / VN][j / 4 % VN],
                                                                    0x0c0c0400u + (uint32_t)(j % 4) * 0x0101u);
                        f[i] = widen<DT, false>(both);
                    } else {
                        f[i] = __builtin_amdgcn_perm(vx[2 * i + 1][j / 2 / VN][j / 2 % VN], vx[2 * i][j / 2 / VN][j / 2 % VN],
                                                     j % 2 ? 0x07060302u : 0x05040100u);
                    }
                }
                const u32x4 v = {f[0], f[1], f[2], f[3]};
                o[j] = Elem<DT>::mfma(v, u32x4{hi[0], hi[1], hi[2], hi[3]}, o[j]);
                o[j] = Elem<DT>::mfma(v, u32x4{lo[0], lo[1], lo[2], lo[3]}, o[j]);
            }
            if (MORE) load_values();
        };
        int s = tile + wave;
        if (s < last && len > first && a.pages > 0) {
            constexpr int kStep = kPagedWaves * kPagedTile;
            int t0 = start + s * kPagedTile;
            look_up(t0);
            load_keys();
            load_values();
            for (; s + kPagedWaves < last; s += kPagedWaves, t0 += kStep) {
                look_up(t0 + kStep);
                attend(std::true_type{}, t0);
            }
            attend(std::false_type{}, t0);
        }
        if (__any(poison)) l = NAN;

        // ---- join the wavefronts: lane (g, l16) has dimensions PW (4 g + i) + j of head l16
        constexpr int pitch = DC + 4;
        const int busy = min(last - tile, kPagedWaves);
        l = quad_column_sum(l);
        if (wave < busy) {
            if (g == 0) { wave_m[wave][l16] = m; wave_l[wave][l16] = l; }
            if (l16 < rows) {
                float *const mineo = lds + (wave * w.rows + l16) * pitch;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < PW; j += 4) {
                        const int d = PW * (4 * g + i) + j;
                        if (SHAPE == kFull || d < a.dim) *(f32x4 *)(mineo + d) = f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]};
                    }
            }
        }
        __syncthreads();
        const bool begun = tile == 0, done = last == n, whole = begun && done;
        const int slot = 2 * (int)group + (begun ? 1 : 0);
        for (int x = 4 * (int)threadIdx.x; x < rows * DC; x += 4 * kPagedThreads) {
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
                const float f = len > first ? (F8 ? a.v.scale[h] : 1.f) / sum : 0.f;
                if (len <= first) acc = f32x4{0.f, 0.f, 0.f, 0.f};
                store_result<DT>(a.out + (q0 + hd) * a.out_head_bytes + request * a.out_row_bytes, d, a.dim, acc * f);
            } else {
                *(f32x4 *)(w.sums + ((int64_t)slot * w.rows + hd) * w.pitch + d) = acc;
                if (d == 0) w.parts[slot * kPagedHeads + hd] = {top, sum};
            }
        }
        if (begun) {
            // who has the unit's last tile
            const int parts = done ? 0 : (int)(scaled(at - tile + n, groups, total) + (scaled(at - tile + n, groups, total) * total < (at - tile + n) * groups) - group);
            join = {request, unit, (int)group, parts};
            if (w.by_unit && threadIdx.x == 0) w.joins[(int64_t)request * units + unit] = join;
        }
        at += last - tile;
        tile = 0;
        if (++unit == units) {
            unit = 0;
            if (++request < a.requests) {
                const Visible v = visible(a, request);
                see = {uniform(v.first), uniform(v.len)};
            }
        }
        __syncthreads();
    }
    if (!w.by_unit && threadIdx.x == 0) w.joins[group] = join;
}

// Joins units that were split: grid (entries of the list, query heads / `heads`).  DC / 4 threads read a row of
// partial sums; the rest of a workgroup's threads take other heads, or every so manieth part of the same ones.
template <int DT, int DC> __global__ void __launch_bounds__(kPagedThreads) paged_join_kernel(PagedAttentionArgs a, PagedWork w, int heads) {
    constexpr int kLanes = DC / 4, kRows = kPagedThreads / kLanes, kAhead = 4;
    const PagedJoin join = w.joins[blockIdx.x];
    if (join.parts == 0) return;
    __shared__ float rest_m[kRows], rest_l[kRows];
    __shared__ f32x4 rest_acc[kRows][kLanes];
    const int mine = (int)threadIdx.x / kLanes, d = 4 * ((int)threadIdx.x % kLanes), deep = kRows / heads;
    const int hd = (int)blockIdx.y * heads + mine % heads, sub = mine / heads;
    const int h = join.unit / w.tiles_a_head, q = h * a.group + (join.unit - h * w.tiles_a_head) * w.rows + hd;
    const bool there = hd < w.rows && q < (h + 1) * a.group && d < a.dim;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (there)
        for (int p0 = sub; p0 < join.parts; p0 += kAhead * deep) {
            PagedPart x[kAhead];
            f32x4 y[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int p = p0 + i * deep;
                x[i] = {-INFINITY, 0.f};
                y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (p < join.parts) {
                    const int64_t slot = 2 * (int64_t)(join.first + p) + (p == 0 ? 1 : 0);
                    x[i] = w.parts[slot * kPagedHeads + hd];
                    y[i] = *(const f32x4 *)(w.sums + (slot * w.rows + hd) * w.pitch + d);
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
        if (sub) return;
        float top = m;
        for (int i = 1; i < deep; ++i) top = fmaxf(top, rest_m[mine + i * heads]);
        const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m - base);
        l *= old;
        acc *= old;
        for (int i = 1; i < deep; ++i) {
            const float f = __builtin_amdgcn_exp2f(rest_m[mine + i * heads] - base);
            l += f * rest_l[mine + i * heads];
            acc += f * rest_acc[mine + i * heads][d / 4];
        }
    }
    if (there) store_result<DT>(a.out + q * a.out_head_bytes + join.request * a.out_row_bytes, d, a.dim, acc * ((a.v.scale ? a.v.scale[h] : 1.f) / l));
}

// ------------------------------------------------------------------ host
static int dim_class(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Workgroups: as many as are resident, or fewer where the longest possible requests would not give each its least share.
static PagedWork work_of(int64_t heads, int64_t group, int64_t dim, int64_t requests, int64_t width, int64_t page, void *workspace, size_t *bytes) {
    PagedWork w{};
    w.tiles_a_head = (int32_t)((group + kPagedHeads - 1) / kPagedHeads);
    w.rows = (int32_t)((group + w.tiles_a_head - 1) / w.tiles_a_head);
    const int64_t resident = (int64_t)device_cu_count() * (dim_class(dim) == 64 ? 4 : dim_class(dim) == 128 ? 3 : 2);
    const int64_t units = requests * heads * w.tiles_a_head;
    const double tiles = (double)units * ((double)width * page / kPagedTile + 1);
    w.groups = (int32_t)std::max<int64_t>(1, (int64_t)std::min<double>((double)resident, tiles / kPagedShare + 1));
    w.by_unit = units <= w.groups;
    const size_t entries = (size_t)(w.by_unit ? units : w.groups);
    const size_t joins = (entries * sizeof(PagedJoin) + 255) & ~size_t(255);
    const size_t parts = (2 * (size_t)w.groups * kPagedHeads * sizeof(PagedPart) + 255) & ~size_t(255);
    w.pitch = (int32_t)((dim + 3) & ~int64_t(3));
    const size_t sums = 2 * (size_t)w.groups * w.rows * w.pitch * sizeof(float);
    if (bytes) *bytes = joins + parts + sums;
    if (workspace) {
        w.joins = (PagedJoin *)workspace;
        w.parts = (PagedPart *)((char *)workspace + joins);
        w.sums = (float *)((char *)workspace + joins + parts);
    }
    return w;
}

size_t paged_attention_workspace(int64_t heads, int64_t group, int64_t dim, int64_t requests, int64_t width, int64_t page) {
    size_t bytes = 0;
    work_of(heads, group, dim, requests, width, page, nullptr, &bytes);
    return bytes;
}

template <int DT, bool F8, int DC, Shape SHAPE, Pages PAGES>
static int launch_split(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream) {
    constexpr int kMostLds = kPagedWaves * kPagedHeads * (DC + 4) * (int)sizeof(float);
    if constexpr (kMostLds > 65536) {
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&paged_attention_kernel<DT, F8, DC, SHAPE, PAGES>),
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
        if (attr != hipSuccess) return BA_ERR_LAUNCH;
    }
    const size_t lds = (size_t)kPagedWaves * w.rows * (DC + 4) * sizeof(float);
    paged_attention_kernel<DT, F8, DC, SHAPE, PAGES><<<w.groups, kPagedThreads, lds, stream>>>(a, w);
    // Few units have many parts each, and a workgroup joins one head of one; of many units most were not split, and a
    // workgroup takes as many heads as it has threads for.
    const int most = kPagedThreads / (DC / 4);
    int heads = 1;
    while (!w.by_unit && heads < most && heads < w.rows) heads *= 2;
    const dim3 grid((unsigned)(w.by_unit ? a.requests * a.heads * w.tiles_a_head : w.groups), (unsigned)((w.rows + heads - 1) / heads));
    paged_join_kernel<DT, DC><<<grid, kPagedThreads, 0, stream>>>(a, w, heads);
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

// Pages of 16, 32, ... tokens and those of 4, 8, 12, 20, ... have builds of their own where rows are whole pieces; all else
// runs through the build that takes every token and byte by itself.
template <int DT, bool F8, int DC> static int launch_class(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream) {
    if (a.page.d % 4 || a.dim % (F8 ? 16 : 8)) return launch_split<DT, F8, DC, kAny, kTokens>(a, w, stream);
    if (a.page.d % 16) return a.dim == DC ? launch_split<DT, F8, DC, kFull, kFours>(a, w, stream) : launch_split<DT, F8, DC, kPieces, kFours>(a, w, stream);
    return a.dim == DC ? launch_split<DT, F8, DC, kFull, kHalves>(a, w, stream) : launch_split<DT, F8, DC, kPieces, kHalves>(a, w, stream);
}

template <int DT, bool F8> static int launch_dtype(const PagedAttentionArgs &a, const PagedWork &w, hipStream_t stream) {
    switch (dim_class(a.dim)) {
        case 64: return launch_class<DT, F8, 64>(a, w, stream);
        case 128: return launch_class<DT, F8, 128>(a, w, stream);
        default: return launch_class<DT, F8, 256>(a, w, stream);
    }
}

int launch_paged_attention(const PagedAttentionArgs &a, int dtype, int cache_dtype, void *workspace, hipStream_t stream) {
    const PagedWork w = work_of(a.heads, a.group, a.dim, a.requests, a.width, a.page.d, workspace, nullptr);
    const bool f8 = cache_dtype == BA_F8_E4M3;
    if (dtype == BA_F16) return f8 ? launch_dtype<0, true>(a, w, stream) : launch_dtype<0, false>(a, w, stream);
    return f8 ? launch_dtype<1, true>(a, w, stream) : launch_dtype<1, false>(a, w, stream);
}

}  // namespace ba
