// Attention of the drafted tokens of each request over a paged key-value cache: what its two kernels share (paged_tree_few.hpp,
// paged_tree_wide.hpp).
//
// out[h][i] = sum_t softmax_t(scale q[h][i] . K[t]) V[t] over the tokens t that row i sees: those before the draft, of the draft
// those with a bit in the row's mask, of these the last `window`.  A key takes part in one product for every row and query head that
// shares it, n x group of them.
//
// Split.  A unit is a block of rows (nodes and the query heads that share a key head, heads fastest) of a request and key head.  Its tokens are
// cut into tiles, and the tiles of all units, in the order of requests, key heads and blocks, are dealt out to the workgroups in equal
// shares, with a constant for what a unit costs besides; sums and lengths are on the GPU only, so every workgroup adds them up itself.
// (Where there are about as many units as workgroups, each gets a unit.)  A unit that lies in one share is done then; for others each workgroup leaves
// maxima, sums and fp32 accumulators in memory.  Where units have few parts, each counts itself in and the last one joins them all, in the order of the tokens whoever it is; else a
// second kernel does.
//
// Tiles that not all rows see all of -- the draft's own, and where windows begin -- hide scores by the rows' bits.  Values there that are not
// finite become zeros, since a probability of 0 times them would be NaN; rows that see them get them at the unit's end.
#pragma once
#include "paged_attention_kernel.hpp"

namespace ba {

constexpr int kTreeThreads = kPagedThreads, kTreeWaves = kPagedWaves;
constexpr int kTreeUnit = 3;                 // what a unit costs besides its tiles, in tiles: queries, first loads, joining, results
constexpr int kTreeShare = kTreeUnit + 1;    // of both, what a workgroup has at least: a unit of one tile
// Where each unit can have a workgroup, it gets one, unless the longest has more than so many tiles above an equal share.  (60 requests of 1000 tokens,
// 8 key heads, 480 units of 15 tiles for 512 workgroups: 95 us, 112 when split evenly.  28 requests of up to 1000, 12 key heads: 38.7 split, 43.4 whole;
// there it is 4 tiles above a share of 7.)
constexpr int kTreeSplit = 4;
constexpr int kTreeWhole = 4;                // units of up to so many tiles are not split between workgroups
constexpr int kTreeFewParts = 8;             // parts of a unit, on the average, up to which the kernel itself joins them
constexpr int kTreeJoinAhead = 8;            // parts on their way together in that kernel

// A unit of which several workgroups did a part each: the one that has its first tile, how many they are (0: not split).
struct TreeLeft {
    int32_t begins, parts, request, h, block;
};
struct TreeWork {
    int32_t *counters;                       // [groups]: how many have left their part of the unit begun by a workgroup; 0 between calls
    TreeLeft *left;                          // not NULL: instead of counting, an entry a workgroup for the joining kernel
    PagedPart *parts;                        // [2 * groups][rows of a unit]
    float *sums;                             // [2 * groups][rows of a unit][pitch]
    PageDiv group;                           // query heads of a key head
    int32_t groups, pitch;
};
struct TreeArgs {
    PagedTreeAttentionArgs a;
    TreeWork w;
};
// The kernel's arguments, fetched again.  Held in scalar registers from the start they, and what is derived from them, are twice what there is; the
// compiler then moves whole groups of them to and from vector registers within the loop over tiles (that loop's loads took 2300 cycles, not 700).
__device__ __forceinline__ const TreeArgs &tree_args() {
    auto p = (const __attribute__((address_space(4))) TreeArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const TreeArgs *)p;
}
// The same number, of which the compiler knows nothing: what is worked out from it for a unit's beginning and end is then worked out there, and not
// kept in vector registers throughout the tiles.
__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Tiles of a kernel, T:  kRows rows of a unit; kTokens tokens of a tile; kStaged of them are loaded together; kGroups wavefronts with the same rows;
// kDims dimensions that are joined and stored at a time, rows kPitch floats apart, kPart bytes of LDS a wavefront; kResident workgroups a compute unit.

// A request's draft.
struct Draft {
    int64_t node0;                           // number of the node of its first row
    int32_t row0, rows;                      // rows of q and out
    int32_t before, end;                     // tokens before the draft, tokens; as far as the table's row holds them
    int32_t blocks, start, tiles;            // of kRows rows; first token of the first tile that may be seen, tiles
};
// UNIFORM: r is the same in all lanes (scalar loads).
template <class T, bool UNIFORM> __device__ __forceinline__ Draft draft_of(const PagedTreeAttentionArgs &a, int r) {
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
__device__ __forceinline__ int64_t tree_ratio_up(int64_t x, int64_t y, int64_t z) {
    const int64_t q = tree_ratio(x, y, z);
    return q + (q * z < x * y);
}

// Parts in memory, as in paged_attention_kernel.hpp.
template <class T> __device__ __forceinline__ Shared tree_shared(const TreeWork &w) {
    return {__builtin_amdgcn_make_buffer_rsrc(w.parts, 0, 2 * w.groups * T::kRows * (int)sizeof(PagedPart), kRsrcFlags),
            __builtin_amdgcn_make_buffer_rsrc(w.sums, 0, 2 * w.groups * T::kRows * w.pitch * 4, kRsrcFlags), T::kRows, w.pitch};
}

// Row `x` of a request's rows and query heads of a key head: a row of q and out, and one of the heads.
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
__device__ __forceinline__ char *tree_out(const PagedTreeAttentionArgs &a, const Draft &d, const TreeRow &t) {
    return a.out + t.head * a.out_head_bytes + (int64_t)(d.row0 + t.node) * a.out_row_bytes;
}
// What accumulators are multiplied with: 0 for rows that see nothing.  (The reciprocal is off by 2^-23 at most, of results of 16 bits.)
__device__ __forceinline__ float tree_factor(float l, float v_scale) { return l == 0.f ? 0.f : v_scale * __builtin_amdgcn_rcpf(l); }

// A part's accumulators by its weight.  CAREFUL: the weight may be 0, where another part's scores are far larger; an infinity among them, of a value that the
// row sees, stays one.
template <bool CAREFUL> __device__ __forceinline__ f32x4 weighed(float f, f32x4 x) {
    f32x4 y = f * x;
    if (CAREFUL)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = f == 0.f && y[i] != y[i] ? x[i] : y[i];
    return y;
}

// Joins the parts of a unit for its rows [row0, row1), by a whole workgroup: DC / 4 threads a row, kDeep rows of a thread and kAhead parts of
// each on their way together (a load from where all dies meet takes some 2 us, however many there are).
template <int DT, int DC, class T, int kDeep, int kAhead>
__device__ __forceinline__ void tree_join(const PagedTreeAttentionArgs &a, const TreeWork &w, const TreeLeft &u, int row0, int row1, float v_scale) {
    constexpr int kLanes = DC / 4, kAtOnce = kTreeThreads / kLanes;
    const Draft d = draft_of<T, false>(a, u.request);
    const Shared shared = tree_shared<T>(w);
    const int dim0 = 4 * ((int)threadIdx.x % kLanes);
    const int rows = (int)min((int64_t)row1, (int64_t)d.rows * a.group - (int64_t)u.block * T::kRows);
#pragma nounroll
    for (int x0 = row0 + (int)threadIdx.x / kLanes; x0 < rows; x0 += kDeep * kAtOnce) {
        float m[kDeep], l[kDeep];
        f32x4 acc[kDeep];
        auto add_up = [&](auto careful) {
            constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
            for (int z = 0; z < kDeep; ++z) {
                m[z] = -INFINITY;
                l[z] = 0.f;
                acc[z] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma nounroll
            for (int p0 = 0; p0 < u.parts; p0 += kAhead) {
                PagedPart part[kDeep][kAhead];
                f32x4 sum[kDeep][kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int p = p0 + i, slot = 2 * (u.begins + p) + (p == 0 ? 1 : 0);
#pragma unroll
                    for (int z = 0; z < kDeep; ++z) {
                        part[z][i] = {-INFINITY, 0.f};
                        sum[z][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                        if (p < u.parts) {
                            const int x = min(x0 + z * kAtOnce, rows - 1);   // (what is there already once more, and not used)
                            part[z][i] = shared.part(slot, x);
                            sum[z][i] = shared.sum(slot, x, min(dim0, w.pitch - 4));
                        }
                    }
                }
#pragma unroll
                for (int z = 0; z < kDeep; ++z) {
                    float top = m[z];
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) top = fmaxf(top, part[z][i].m);
                    const float base = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m[z] - base);
                    l[z] *= old;
                    acc[z] = weighed<CAREFUL>(old, acc[z]);
                    m[z] = top;
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        const float f = __builtin_amdgcn_exp2f(part[z][i].m - base);
                        l[z] += f * part[z][i].l;
                        acc[z] += weighed<CAREFUL>(f, sum[z][i]);
                    }
                }
            }
        };
        add_up(std::false_type());
        // (once more where something is NaN: with the care for all of them the batch of drafts takes 99.7 us, 97.4 so)
        bool again = false;
#pragma unroll
        for (int z = 0; z < kDeep; ++z)
#pragma unroll
            for (int i = 0; i < 4; ++i) again |= acc[z][i] != acc[z][i];
        if (again) add_up(std::true_type());
#pragma unroll
        for (int z = 0; z < kDeep; ++z)
            if (const int x = x0 + z * kAtOnce; x < rows && dim0 < a.dim) {
                if (l[z] == 0.f) acc[z] = f32x4{0.f, 0.f, 0.f, 0.f};
                store_result<DT>(tree_out(a, d, tree_row(a, w, d, u.h, (int64_t)u.block * T::kRows + x)), dim0, a.dim, acc[z] * tree_factor(l[z], v_scale));
            }
    }
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// What a row sees of the tokens from a place on.
struct Sight {
    const int64_t *bits;                     // its row of the mask, or NULL
    uint64_t word0;                          // the first word there
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
                x = (j < 64 ? word0 : (uint64_t)bits[j >> 6]) >> (j & 63);
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
    s.word0 = a.mask ? (uint64_t)s.bits[0] : 0;
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
// Staged tokens from t on that not all rows see: those of the draft, and where the rows' windows begin.
__device__ __forceinline__ uint32_t all_see_from(const Draft &d, int window) {
    return window ? (uint32_t)max(d.before - window + min(d.end - d.before, window), 0) : 0u;
}
template <class T> __device__ __forceinline__ bool hidden(const Draft &d, int window, uint32_t t) {
    return t + T::kStaged > (uint32_t)d.before || t < all_see_from(d, window);
}

// A workgroup's LDS besides its tiles.
template <class T> struct TreeLds {
    struct Place {
        int32_t request, unit, tile;
        int64_t at;
        Draft d;
    };
    Place places[2];
    int64_t scan[kTreeWaves], dealt[2];                      // (dealt: tiles, workgroups that have some)
    int32_t units[kTreeWaves], longest[kTreeWaves];
    int64_t spots[kTreeWaves][2][T::kStaged];                // where the tokens that a wavefront looks after lie, of keys and values
    float m[kTreeWaves][T::kWaveRows], l[kTreeWaves][T::kWaveRows];
    TreeLeft left[2];
    int32_t joins[2], row_from[T::kRows], odd;               // odd: whether a part's hidden tiles have values that are not finite
};

// A unit's part that is a workgroup's: tiles [tile, last); `at`: place of the first one in the order of all.
struct TreeUnit {
    Draft d;
    int64_t at;
    int32_t request, unit, tile, last, h, block;
};
__device__ __forceinline__ TreeUnit unit_of(const Draft &d, int request, int unit, int tile, int64_t at, int64_t end) {
    TreeUnit u;
    u.d = d; u.request = request; u.unit = unit; u.tile = tile; u.at = at;
    u.h = unit / u.d.blocks;
    u.block = unit - u.h * u.d.blocks;
    u.last = (int)min((int64_t)u.d.tiles, tile + (end - at));
    return u;
}
// The unit behind it, if the share goes on.
__device__ __forceinline__ int64_t tree_next(const TreeUnit &u) { return u.at + (u.last - u.tile) + kTreeUnit; }
template <class T> __device__ __forceinline__ TreeUnit unit_after(const TreeUnit &u, int64_t end) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    if (u.unit + 1 < a.heads * u.d.blocks) return unit_of(u.d, u.request, u.unit + 1, 0, tree_next(u), end);
    int request = u.request + 1;
    Draft d = draft_of<T, true>(a, request);
    while (d.blocks == 0) d = draft_of<T, true>(a, ++request);
    return unit_of(d, request, 0, 0, tree_next(u), end);
}

// The workgroup's share.  The first half of the threads finds where it begins, the other where it ends: thread i of each adds up requests
// [i c, (i + 1) c).  Rows of no request get their zeros here.  Returns where the share ends, or -1
// if there is none; `group`: its number in the order of shares.
template <class T> __device__ __forceinline__ int64_t tree_deal(TreeLds<T> &sh, TreeUnit &first, int &group) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    const TreeWork &w = tree_args().w;
    group = (int)blockIdx.x;
    const int lane = lane_id(), wave = uniform((int)threadIdx.x >> 6);
    constexpr int kHalf = kTreeThreads / 2, kHalfWaves = kTreeWaves / 2;
    const int k = wave / kHalfWaves, me = (int)threadIdx.x % kHalf, c = (a.requests + kHalf - 1) / kHalf, r0 = me * c, r1 = min(a.requests, r0 + c);
    const int64_t head = a.requests ? min(max(a.accum[0], (int64_t)0), a.tokens) : a.tokens;         // rows of no request: before, from `tail` on
    const int64_t tail = a.requests ? min(max(a.accum[a.requests], head), a.tokens) : a.tokens;
    int64_t mine = 0;
    int units = 0, longest = 0;                              // (tiles)
    Draft front = {};
    for (int r = r0; r < r1; ++r) {
        const Draft d = draft_of<T, false>(a, r);
        if (r == r0) front = d;
        mine += (int64_t)a.heads * d.blocks * (d.tiles + kTreeUnit);
        units = (int)min(units + (int64_t)a.heads * d.blocks, (int64_t)1 << 23);
        longest = d.blocks ? max(longest, d.tiles) : longest;
    }
    int64_t upto = wave_inclusive_scan(mine);
    int units_upto = wave_inclusive_scan(units);
    longest = wave_max_nonneg(longest);
    if (lane == 63) { sh.scan[wave] = upto; sh.units[wave] = units_upto; sh.longest[wave] = longest; }
    if (threadIdx.x == 0) sh.odd = 0;
    __syncthreads();
    int64_t total = 0;
    int all_units = 0;
#pragma unroll
    for (int i = 0; i < kHalfWaves; ++i) {
        if (i < wave % kHalfWaves) { upto += sh.scan[i]; units_upto += sh.units[i]; }
        total += sh.scan[i];
        all_units += sh.units[i];
        longest = max(longest, sh.longest[i]);
    }
    total = uniform64(total);
    int64_t groups = uniform64(min((int64_t)w.groups, (total + kTreeShare - 1) / kTreeShare));
    const bool whole = uniform(all_units) <= groups && (uniform(longest) + kTreeUnit - kTreeSplit) * groups <= total;
    if (whole) groups = uniform(all_units);
    for (int64_t i = group; i < head + a.tokens - tail; i += gridDim.x) {
        char *const out = a.out + (i < head ? i : tail + (i - head)) * a.out_row_bytes;
        for (int x = (int)threadIdx.x; x < a.heads * a.group * a.dim; x += kTreeThreads) {
            const int head_of = x / a.dim;
            *(u16_any *)(out + head_of * a.out_head_bytes + 2 * (x - head_of * a.dim)) = 0;
        }
    }
    // Dies take workgroups in turn.  A die's workgroups get shares next to each other, so that blocks of rows of the same keys and values meet in its cache (16
    // requests of 4000 tokens, 512 rows: 331 us, 293 so; batch of drafts 100, 97).  Small units only where most of them are such blocks: else it makes dies unequal
    // (64 requests of 4000 tokens, 16 rows: 168 us, 170 so).
    if (group < groups && (T::kRows >= 64 || uniform(all_units) >= 2 * (int64_t)a.heads * a.requests)) {
        const int each = (int)groups / 8, rest = (int)groups % 8, die = group % 8;
        group = die * each + min(die, rest) + group / 8;
    }
    if (w.left && threadIdx.x == 0) w.left[group].parts = 0;
    if (group >= groups) return -1;
    if (threadIdx.x == 0) { sh.dealt[0] = total; sh.dealt[1] = groups; }
    const int number = group + k;
    int64_t at = whole ? 0 : tree_ratio(number, total, groups);
    if (number >= groups) {
        if (me == 0) sh.places[k] = {a.requests, 0, 0, total + kTreeUnit, front};
    } else if (whole ? number < units_upto && number >= units_upto - units : at < upto && at >= upto - mine) {
        int64_t before = upto - mine;
        int r = r0, passed = units_upto - units;
        Draft d = front;
        for (int64_t all; all = (int64_t)a.heads * d.blocks * (d.tiles + kTreeUnit), whole ? number >= passed + a.heads * d.blocks : at >= before + all; before += all) {
            passed += a.heads * d.blocks;
            d = draft_of<T, false>(a, ++r);
        }
        if (whole) at = before + (int64_t)(number - passed) * (d.tiles + kTreeUnit);
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
                    do {
                        if (++r < a.requests) d = draft_of<T, false>(a, r);
                    } while (r < a.requests && d.blocks == 0);
                }
            }
            tile = 0;
        }
        sh.places[k] = {r, unit, tile, at, d};
    }
    __syncthreads();
    const int64_t end = uniform64(sh.places[1].at);
    at = uniform64(sh.places[0].at);
    if (at >= end) return -1;
    const Draft &d = sh.places[0].d;
    first = unit_of({uniform64(d.node0), uniform(d.row0), uniform(d.rows), uniform(d.before), uniform(d.end), uniform(d.blocks), uniform(d.start), uniform(d.tiles)},
                    uniform(sh.places[0].request), uniform(sh.places[0].unit), uniform(sh.places[0].tile), at, end);
    return end;
}

// ---- rows of keys and values.  Lane i of a wavefront looks after token i of those that are staged: it asks for the token's page number, two tiles ahead,
// and leaves the token's place for the lanes that load it.
typedef const __attribute__((address_space(1))) int32_t *TableRow;       // (loads through a generic pointer would wait for LDS too)
__device__ __forceinline__ TableRow table_row(const TreeUnit &u) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    return (TableRow)(uintptr_t)uniform64((int64_t)(uintptr_t)(a.table + u.request * a.table_stride));
}
struct TreeSteps {                           // of pages and tokens, each in registers of its own
    int64_t k_page, v_page;
    int k_token, v_token, pages;
    PageDiv page;
};
__device__ __forceinline__ TreeSteps tree_steps() {
    const PagedTreeAttentionArgs &a = tree_args().a;
    return {uniform64(a.k.page_bytes), uniform64(a.v.page_bytes), uniform(a.k.token_bytes), uniform(a.v.token_bytes), uniform(a.pages),
            {(uint32_t)uniform((int)a.page.d), (uint32_t)uniform((int)a.page.mul), (uint32_t)uniform((int)a.page.shift)}};
}
__device__ __forceinline__ int32_t look_up(const TreeUnit &u, TableRow row, const PageDiv &page, bool has, uint32_t t) {
    return has && t < (uint32_t)u.d.end ? row[page.div(t)] : -1;
}
// Where a unit's rows lie.  The place of a token that is not there is that of the first bytes of the queries, which are as long as a row: whatever
// is read is there, without a comparison at every load.
struct TreeBases {
    const char *k, *v;
    int64_t k_none, v_none;
    int row_bytes;
};
template <int EB> __device__ __forceinline__ TreeBases tree_bases(const TreeUnit &u) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    TreeBases b = {a.k.base + u.h * a.k.head_bytes, a.v.base + u.h * a.v.head_bytes, 0, 0, uniform(EB * a.dim)};
    b.k_none = uniform64((int64_t)((uintptr_t)a.q - (uintptr_t)b.k));
    b.v_none = uniform64((int64_t)((uintptr_t)a.q - (uintptr_t)b.v));
    return b;
}
// Places of tokens t of page `number`; the bits of those that are not there or on a page outside the cache, and of the latter alone.
struct Missing {
    uint64_t any, bad;
};
template <class T>
__device__ __forceinline__ Missing tree_aim(int64_t (&spots)[2][T::kStaged], int i, const TreeSteps &by, const TreeBases &from, const TreeUnit &u, uint32_t t, int32_t number) {
    const uint32_t in = t - by.page.div(t) * by.page.d;
    const bool none = (uint32_t)number >= (uint32_t)by.pages;
    auto wide = [](uint32_t x, int64_t y) { return (int64_t)((uint64_t)x * (uint32_t)y + ((uint64_t)(x * (uint32_t)((uint64_t)y >> 32)) << 32)); };
    spots[0][i] = none ? from.k_none : wide((uint32_t)number, by.k_page) + (int64_t)((uint64_t)in * (uint32_t)by.k_token);
    spots[1][i] = none ? from.v_none : wide((uint32_t)number, by.v_page) + (int64_t)((uint64_t)in * (uint32_t)by.v_token);
    __builtin_amdgcn_wave_barrier();
    return {__ballot(none), __ballot(none && t < (uint32_t)u.d.end)};
}

// Values that are not finite: `mark` is not 0 behind every dword that has one or more (its halves, for 16 bits, are above the type's exponent).
template <int DT, bool F8> constexpr uint32_t kNotFinite = F8 ? 0x7fu : DT == 0 ? 0x7c00u : 0x7f80u;
template <int DT, bool F8, int N> __device__ __forceinline__ void watch(uint32_t &mark, const uint32_t (&x)[N]) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (F8) mark |= ((x[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        else mark = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, mark), __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu)));
    }
}
template <int DT, bool F8> __device__ __forceinline__ bool seen_odd(uint32_t mark) {
    return F8 ? mark != 0 : (mark & 0xffffu) >= kNotFinite<DT, F8> || mark >> 16 >= kNotFinite<DT, F8>;
}
template <int DT, bool F8, int N> __device__ __forceinline__ void take_out(uint32_t (&x)[N]) {
    constexpr int kWidth = F8 ? 8 : 16;
    constexpr uint32_t kAll = F8 ? 0xffu : 0xffffu;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int b = 0; b < 32; b += kWidth) x[i] &= (x[i] >> b & kNotFinite<DT, F8>) == kNotFinite<DT, F8> ? ~(kAll << b) : 0xffffffffu;
}

// ---- the end of a unit, whose wavefronts have their maxima and sums in sh.m and sh.l.  Dimensions c .. c + kDims of the accumulators lie in LDS, rows
// kPitch floats apart, kPart bytes a wavefront: they are joined, and given out or left as a part.  By way of LDS so that whole rows are stored.
template <int DT, class T>
__device__ __forceinline__ void tree_store(const TreeLds<T> &sh, int group, const char *lds, const TreeUnit &u, int me, int c, float v_scale) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    const TreeWork &w = tree_args().w;
    const bool begun = u.tile == 0, whole = begun && u.last == u.d.tiles;
    const int slot = 2 * group + (begun ? 1 : 0);
    const Shared shared = tree_shared<T>(w);
    // all threads have the rows of all that are there; kGroups == 1: part x / 32 has rows 32 (x / 32) ..
    constexpr int kLanes = T::kDims / 4;
    const int dim1 = 4 * (me % kLanes), dim0 = c + dim1;
    const int many = uniform((int)min((int64_t)T::kRows, (int64_t)u.d.rows * a.group - (int64_t)u.block * T::kRows) * kLanes);
#pragma unroll 4
    for (int e = me; e < many; e += kTreeThreads) {
        const int x = e / kLanes;
        const TreeRow t = tree_row(a, w, u.d, u.h, (int64_t)u.block * T::kRows + x);
        float top = -INFINITY, sum = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (T::kGroups == 1) {
            top = sh.m[x / 32][x % 32];
            sum = sh.l[x / 32][x % 32];
            acc = *(const f32x4 *)((const float *)(lds + x / 32 * T::kPart) + x % 32 * T::kPitch + dim1);
        } else {
#pragma unroll
            for (int i = 0; i < T::kGroups; ++i) top = fmaxf(top, sh.m[i][x]);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int i = 0; i < T::kGroups; ++i) {
                const float f = __builtin_amdgcn_exp2f(sh.m[i][x] - base);
                sum += f * sh.l[i][x];
                acc += f * *(const f32x4 *)((const float *)(lds + i * T::kPart) + x * T::kPitch + dim1);
            }
        }
        if (dim0 < a.dim) {
            if (whole) {
                if (sum == 0.f) acc = f32x4{0.f, 0.f, 0.f, 0.f};
                store_result<DT>(tree_out(a, u.d, t), dim0, a.dim, acc * tree_factor(sum, v_scale));
            } else {
                shared.store(slot, x, dim0, acc);
                if (dim0 == 0) shared.store(slot, x, PagedPart{top, sum});
            }
        }
    }
}
// Values that are not finite, for the rows that see them (an infinity or a NaN of whatever weight is the result's), and what is said of a part.
// `odd`: sh.odd, read by every wavefront before the barrier that comes before this.  Behind that barrier a wavefront may be at the next unit's tiles, where
// it sets sh.odd, while another is still here.
template <int DT, bool F8, class T> __device__ __forceinline__ void tree_end(TreeLds<T> &sh, int group, const TreeUnit &u, int me, bool odd, int &unfinished) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    const TreeWork &w = tree_args().w;
    const Draft &d = u.d;
    const bool begun = u.tile == 0, whole = begun && u.last == d.tiles;
    const int slot = 2 * group + (begun ? 1 : 0);
    if (odd) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const TableRow row = table_row(u);
        const Shared shared = tree_shared<T>(w);
        // the part's tokens [t_first, t_end) that are hidden from some: those before `head` and from `tail` on (32 requests of 4000 tokens and 10 nodes, 40 rows a key
        // head, one NaN in a draft: 660 us, 9200 by way of all tokens, 144 without the NaN; eight at a time 490, but drafts without any then take 104 us for 97)
        const uint32_t t_first = (uint32_t)d.start + (uint32_t)u.tile * T::kTokens, t_end = (uint32_t)min((int64_t)d.end, (int64_t)d.start + (int64_t)u.last * T::kTokens);
        const uint32_t head = (all_see_from(d, a.window) + T::kStaged - 1) & ~(uint32_t)(T::kStaged - 1), tail = (uint32_t)d.before & ~(uint32_t)(T::kStaged - 1);
        for (int e = me; e < T::kRows * a.dim; e += kTreeThreads) {
            const int x = e / a.dim, dim = e - x * a.dim;
            const TreeRow t = tree_row(a, w, d, u.h, (int64_t)u.block * T::kRows + x);
            const Sight s = sight_of(a, d, t, sh.row_from[x]);
            float add = 0.f;
#pragma nounroll
            for (uint32_t tok = t_first; tok < t_end; ++tok) {
                if (tok >= head && tok < tail) tok = tail;
                if (tok >= t_end) break;
                if (!(s(d, a.words, tok) & 1)) continue;
                const uint32_t at_page = a.page.div(tok);
                const int32_t in_page = row[at_page];
                if ((uint32_t)in_page >= (uint32_t)a.pages) continue;
                const char *const v = a.v.base + u.h * a.v.head_bytes + in_page * a.v.page_bytes + (int64_t)(tok - at_page * a.page.d) * a.v.token_bytes + (F8 ? 1 : 2) * dim;
                const uint32_t bits = F8 ? *(const uint8_t *)v : *(const u16_any *)v;
                if ((bits & kNotFinite<DT, F8>) == kNotFinite<DT, F8>) add += F8 ? NAN : Elem<DT>::to_float((uint16_t)bits);
            }
            if (t.there && add != 0.f) {
                if (whole) ((u16_any *)tree_out(a, d, t))[dim] = Elem<DT>::from_float(add);
                else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, add), shared.sums, shared.sum_at(slot, x, dim), 0, kSharedAux);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) sh.odd = 0;
        __syncthreads();
    }
    if (!whole) {
        const int64_t first = u.at - u.tile, total = uniform64(sh.dealt[0]), groups = uniform64(sh.dealt[1]);
        TreeLeft left = {begun ? group : (int)tree_ratio_up(first + 1, groups, total) - 1, 0, u.request, u.h, u.block};
        left.parts = (int)tree_ratio_up(first + d.tiles, groups, total) - left.begins;
        if (w.left) {
            if (begun && threadIdx.x == 0) w.left[group] = left;
        } else {
            if (threadIdx.x == 0) sh.left[unfinished] = left;
            ++unfinished;                                    // (the first unit of the share at most, and its last)
        }
    }
}
// The end of a workgroup: the last one that has left its part of a unit joins them.
template <int DT, bool F8, int DC, class T> __device__ __forceinline__ void tree_count_in(TreeLds<T> &sh, int unfinished) {
    const PagedTreeAttentionArgs &a = tree_args().a;
    const TreeWork &w = tree_args().w;
    if (w.left || unfinished == 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 0; i < unfinished; ++i) {
            int32_t *const counter = w.counters + sh.left[i].begins;
            sh.joins[i] = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == sh.left[i].parts - 1;
            if (sh.joins[i]) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    __syncthreads();
#pragma nounroll
    for (int i = 0; i < unfinished; ++i)
        if (sh.joins[i]) tree_join<DT, DC, T, 4, 4>(a, w, sh.left[i], 0, T::kRows, F8 ? a.v.scale[sh.left[i].h] : 1.f);
}

// The joining as a kernel of its own: grid (blocks of rows, workgroups of the other), one row a thread, so that many workgroups share
// the loads (32 parts of 32 rows 9 us; with four rows a thread 19).  Units often begin with every 32nd workgroup or so, which would all be on one XCD,
// dies taking workgroups in turn (16 units of 32 parts of 128 rows 65 us): the number's low bits are mixed with those above.
template <int DT, int DC, class T> __global__ void __launch_bounds__(kTreeThreads) paged_tree_join_kernel(TreeArgs args, int rows) {
    const int group = (int)blockIdx.y ^ ((int)(blockIdx.y >> 3) & 7) ^ ((int)(blockIdx.y >> 6) & 7);
    if (group >= args.w.groups) return;
    const TreeLeft u = args.w.left[group];
    const int row0 = (int)blockIdx.x * rows;
    if (u.parts) tree_join<DT, DC, T, 1, kTreeJoinAhead>(args.a, args.w, u, row0, row0 + rows, args.a.v.scale ? args.a.v.scale[u.h] : 1.f);
}

// What is known of the rows: whole 16-byte pieces at multiples of 16 bytes; at any address, of 16 bytes or more; shorter.
enum TreeRows { kTreePieces, kTreeAny, kTreeShort };

// ------------------------------------------------------------------ host
template <int DT, int DC, class T, typename K> int tree_launch(K kernel, const PagedTreeAttentionArgs &a, const TreeWork &w, hipStream_t stream) {
    kernel<<<w.groups, kTreeThreads, T::kLds, stream>>>(TreeArgs{a, w});
    if (w.left) {
        constexpr int kRows = std::min(T::kRows, kTreeThreads / (DC / 4));           // (a round of its threads)
        paged_tree_join_kernel<DT, DC, T><<<dim3(T::kRows / kRows, (unsigned)(w.groups + 7) / 8 * 8), kTreeThreads, 0, stream>>>(TreeArgs{a, w}, kRows);
    }
    return hipGetLastError() == hipSuccess ? BA_OK : BA_ERR_LAUNCH;
}

// Rows of a unit, and with them the kernel, by the rows that a request and key head have on the average: a unit's time hardly depends on how many of its
// rows are there (64 requests of 4000 tokens, 8 key heads of 128: 16 rows 167 us, with units of 128 273; 32 rows 175 and 243; 64 rows of 128
// dimensions 271 with units of 64 and 294 with 128, but over 1000 tokens, 60 requests, 86 and 80, and 261 and 232 of 80 dimensions; of 64 dimensions 140 and 170).
// Small units also where requests are brief and their small units no more than there are compute units, which then share the rows (4 requests of 100
// tokens, 128 rows: 14.7 us, with units of 128 25; 8 of 1000 30 and 42; but 24 of 200 35 and 30, 2 of 20000 93 and 73); a few of the smallest for 32
// rows (500 tokens 14.8 us, with units of 32 19.1; 4 requests of 1000 17.6 and 21.4).
// More than 128 dimensions have units of 16 or 128 rows, for want of registers (8 key heads, 64 requests, 32 rows, 60 tokens: 43 us and 43; 4000 tokens 652 and
// 594; 2 requests, 128 rows, 60 / 400 / 1200 tokens: 15 / 22 / 34 and 30 / 32 / 38).
constexpr int64_t kTreeBrief = 2048;
static inline int tree_rows(int64_t heads, int64_t tokens, int64_t requests, int64_t group, int64_t dim, int64_t longest) {
    const int64_t rows = tokens * group, many = std::max<int64_t>(1, requests);
    const bool brief = longest <= kTreeBrief;
    if (dim > 128) return rows <= (brief ? 32 : 24) * many || (brief && heads * rows <= 16 * (int64_t)device_cu_count()) ? 16 : 128;
    if (rows <= 16 * many || (brief && rows <= 32 * many && heads * rows <= 16 * 64)) return 16;
    if (rows <= 32 * many || (brief && heads * rows <= 32 * (int64_t)device_cu_count())) return 32;
    return rows <= 64 * many && dim <= 64 ? 64 : 128;
}
template <int DT, bool F8> int launch_tree_few(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int sets, hipStream_t stream);
template <int DT, bool F8> int launch_tree_wide(const PagedTreeAttentionArgs &a, const TreeWork &w, TreeRows rows, int waves, hipStream_t stream);

}  // namespace ba
