// Attention backward under score rules: tiles on the f16 matrix core, no atomics.
//   P = 2^(x - lse), dP = dO V^T, ds = P (dP - delta) slope, delta = sum dO O
//   dQ = scale ds K (k_attn_dq, a tile of queries over the keys that it sees), dK = scale ds^T Q and dV = P^T dO (k_attn_dkv, a tile of keys over the rows that see
//   it, of all query heads that share it).  Scores and dP are formed by both: seven products a pair where five would do, for sums in a fixed order.
// Operands are cut into f16 terms as in the forward pass (f16x2.h).  ds and P have no scale of their own: a running exponent for each row (or key) keeps the largest so
// far, times the factors of what it is multiplied by, at 2^10 to 2^15, and the sum is rescaled when it moves, as an online softmax does.
//
// A wave owns 16 rows (or keys): two operands of them and two sums are half as many registers as for 32, so two waves share a SIMD at every head size, and one's vector
// instructions run beside the other's products.  (32 rows a wave had one wave a SIMD from heads of 96 on, its matrix core idle two thirds of the time; what 16 cost is twice the reads from LDS
// for a product.)  A lane owns row (l & 15) of the wave in the tiles of 32 keys: its eight values are keys 16 t + 4 (l / 16) + 0..3, t = 0, 1.  In
// k_attn_dkv the key is on the lane side and the eight are rows, and what these need (lse, delta, end, document) lies in LDS beside the block.  Blocks are double in
// LDS and staged by the two waves of a SIMD at different times, as in the forward pass.  Where there are few tiles, what each runs over is shared out to several workgroups, which
// meet in memory (plan_of, met).  Rows (keys) whose sums are not finite are formed again with fp32 instructions.
//
// What bounds it: as in the forward pass the matrix core and the vector instructions in turn, which two waves overlap in part; the matrix core is busy 46 % of the time with heads of
// 128, 36 % with heads of 64 (32 rows by 16 keys: 96 matrix and 309 vector instructions, 48 and 247).  2 x 16 heads, 8 of keys, [2048, 128] without a mask take 700 us,
// 245 TFLOP/s counted as five products, 343 of the seven that are formed; causal and under a cap 443 to 474; 4 x 16 of [2048, 64] 838 and 470.
#include <algorithm>
#include <cmath>

#include "attn_launch.h"
#include "attn_tiles.h"

namespace {
using namespace axhip;

constexpr int WAVES = 8;
typedef float Eight[8];

template <int N>
__device__ __forceinline__ void times(v4f (&acc)[N], float by) {
#pragma unroll
    for (int n = 0; n < N; n++) acc[n] *= by;
}

// Scores of a lane (products already scaled) after cap and distance; `slope` the cap's derivative
template <typename Distance>
__device__ __forceinline__ void score_tile(const AttnArgs &a, Eight &s, Eight &slope, Distance distance) {
    if (a.cap > 0.0f) {
        float big = 0.0f;
#pragma unroll
        for (int v = 0; v < 8; v++) big = fmaxf(big, __builtin_fabsf(s[v]));
        if (__builtin_amdgcn_ballot_w64(!(big < a.cap_near)))
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const Capped c = capped(a, s[v]);
                s[v] = c.score;
                slope[v] = c.slope;
            }
        else
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const Capped c = capped_near(a, s[v]);
                s[v] = c.score;
                slope[v] = c.slope;
            }
    }
    if (a.slopes)
#pragma unroll
        for (int v = 0; v < 8; v++) s[v] -= distance(v);
}

// The next block of TILES tiles from `blk` on, below n, of which some tile's documents meet [low, high]: 64 blocks at a time, a lane each
template <int TILES>
struct Blocks {
    const DocRange *ranges;                      // NULL: every block
    int n, tiles, low, high, at;
    uint64_t window;
    __device__ Blocks(const DocRange *r, int blocks, int range_tiles, int from, int to) : ranges(r), n(blocks), tiles(range_tiles), low(from), high(to), at(-64), window(0) {}
    __device__ __forceinline__ int next(int blk, int lane) {
        if (!ranges) return blk < n ? blk : n;
        while (blk < n) {
            if (blk < at || blk - at >= 64) {
                at = blk & ~63;
                const int mine = at + lane;
                bool meets = false;
                if (mine < n) {
#pragma unroll
                    for (int i = 0; i < TILES; i++)
                        if (TILES * mine + i < tiles) meets |= ranges[TILES * mine + i].meets(low, high);
                }
                window = __builtin_amdgcn_ballot_w64(meets);
            }
            const uint64_t ahead = window >> (blk - at);
            if (ahead) {
                const int found = blk + __builtin_ctzll(ahead);
                return found < n ? found : n;
            }
            blk = at + 64;
        }
        return n;
    }
};

// Workgroups go to the eight XCDs in turn: a unit's tiles (a head's, a group of heads') to one, eight units at a time, or, causal, the longest tile of every unit first
struct Work {
    int64_t lin;                                 // the tile of the launch
    int split;
};
__device__ __forceinline__ Work work_of(const AttnArgs &a, const BwdGrid &grid, int64_t &unit, int &tile) {
    const int64_t at = grid.first + blockIdx.x, lin = at / grid.splits, group = lin / (8 * (int64_t)grid.tiles), r8 = lin - group * 8 * grid.tiles;
    const int64_t left = grid.units - group * 8, width = left < 8 ? left : 8;
    unit = a.causal ? lin % grid.units : group * 8 + r8 % width;
    tile = (int)(a.causal ? lin / grid.units : r8 / width);
    return {lin, (int)(at - lin * grid.splits)};
}

// The splits of a tile meet in memory: each leaves the sums of its `mine` waves (wave w, `part` floats a split), the last to arrive adds them, in order, and true is
// what it gets.  Parts, counter and reads are device-scope accesses (the workgroups run on XCDs with an L2 each); the wait completes a thread's stores before the
// barrier, the barrier orders them before thread 0's increment.  `flag`: a word of LDS that is no longer read.
template <int N>
__device__ __forceinline__ bool met(const BwdGrid &grid, const Work &work, int part, bool mine, int w, int lane, int *flag, v4f *(&&sums)[N], int each) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    const int64_t of_tile = work.lin * grid.splits * part;
    const int at = w * N * each * 256 + lane * 4;
    if (mine) {
        float *to = grid.parts + of_tile + (int64_t)work.split * part + at;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int i = 0; i < each; i++) {
                const v4f v = sums[n][i];
                int64_t *there = reinterpret_cast<int64_t *>(to + (n * each + i) * 256);
                __hip_atomic_store(there, __builtin_bit_cast(int64_t, v2f{v[0], v[1]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(there + 1, __builtin_bit_cast(int64_t, v2f{v[2], v[3]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                sums[n][i] = v4f{0.f, 0.f, 0.f, 0.f};
            }
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) *flag = __hip_atomic_fetch_add(grid.arrivals + work.lin, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == grid.splits - 1;
    __syncthreads();
    if (!*flag) return false;
    if (mine)
        for (int s = 0; s < grid.splits; s++) {
            const float *from = grid.parts + of_tile + (int64_t)s * part + at;
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < each; i++) {
                    const int64_t *there = reinterpret_cast<const int64_t *>(from + (n * each + i) * 256);
                    const v2f x = __builtin_bit_cast(v2f, __hip_atomic_load(there, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                    const v2f y = __builtin_bit_cast(v2f, __hip_atomic_load(there + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                    sums[n][i] += v4f{x[0], x[1], y[0], y[1]};
                }
        }
    if (threadIdx.x == 0) __hip_atomic_store(grid.arrivals + work.lin, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);       // ready for the next launch
    return true;
}

// SETS waves side by side, 16 rows (or keys) each; where those are half of the waves, the others take the other tiles of each block
template <int DK, int SETS>
struct BwdGeom {
    static constexpr int ROWS = DK <= 64 ? 128 : 64, TILES = ROWS / 32, SHARES = WAVES / SETS;
    using B = Block<DK, ROWS>;
};

template <int DK, int SETS>
struct DqGeom : BwdGeom<DK, SETS> {
    using Base = BwdGeom<DK, SETS>;
    static constexpr int FACTORS_AT = 2 * Base::B::BYTES;        // of each key row, then of each value row
    static constexpr int DOCS_AT = FACTORS_AT + Base::ROWS * 8;  // documents of the keys, then the ranges of their tiles
    static constexpr int STAGE = (DOCS_AT + Base::ROWS * 4 + Base::TILES * 8 + 255) / 256 * 256;
    static constexpr int META_AT = 2 * STAGE;
    static constexpr int JOIN = DK / 16 * 1024;                  // the other share's sums: [DK / 16][64 lanes] v4f a wave
    static constexpr int SMEM = META_AT + 16 * WAVES;
    static_assert(SMEM <= 160 * 1024 && SETS * JOIN <= META_AT, "LDS");
};

template <int DK, int SETS, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, 2) k_attn_dq(AttnArgs a, BwdGrid grid) {
    using G = DqGeom<DK, SETS>;
    using B = typename G::B;
    constexpr int KS = DK / 32, NT = DK / 16, ROWS = G::ROWS, TILES = G::TILES;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, part = lane >> 4;
    int64_t unit;
    int tile;
    const Work work = work_of(a, grid, unit, tile);
    if (a.causal) tile = grid.tiles - 1 - tile;
    const int b = (int)(unit / a.H), head = (int)(unit - (int64_t)b * a.H), hk = head / a.G;
    const int r = tile * 16 * SETS + wave % SETS * 16 + col, i = r < a.Sq ? r : a.Sq - 1;
    const bool valid = r < a.Sq;
    AttnRow row = attn_row(a, b, head, i);
    if (!valid) row.end = 0;
    const bool live = row.end > 0, docs = a.doc_q != nullptr;
    const RowsSeen mine = same_for_wave(rows_seen(row));
    const int last = mine.last, sure = mine.sure, d_low = mine.low, d_high = mine.high;
    int *meta = reinterpret_cast<int *>(lds + G::META_AT);
    if (lane == 0) *reinterpret_cast<v4i *>(meta + 4 * wave) = v4i{last, 0, d_low, d_high};
    __syncthreads();
    int wg_last = 0, wg_low = 0x7fffffff, wg_high = -1;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const v4i m = *reinterpret_cast<const v4i *>(meta + 4 * w);
        wg_last = max(wg_last, m[0]);
        wg_low = min(wg_low, m[2]);
        wg_high = max(wg_high, m[3]);
    }
    wg_last = __builtin_amdgcn_readfirstlane(wg_last);
    wg_low = __builtin_amdgcn_readfirstlane(wg_low);
    wg_high = __builtin_amdgcn_readfirstlane(wg_high);
    const DocRange *ranges = docs ? grid.key_ranges + (int64_t)b * grid.key_tiles : nullptr;
    const int64_t all_blocks = (wg_last + ROWS - 1) / ROWS;
    Blocks<TILES> blocks(ranges, (int)(all_blocks * (work.split + 1) / grid.splits), grid.key_tiles, wg_low, wg_high);

    const float *Kb = a.K + (int64_t)b * a.kv_rows * a.ldk + (int64_t)hk * a.dk, *Vb = a.V + (int64_t)b * a.kv_rows * a.ldv + (int64_t)hk * a.dk;
    using S = Stage<DK, ROWS, WAVES, PAD>;
    S ks, vs;
    const unsigned base = lds_address(lds);
    int doc_here = -1;
    DocRange range_here = {0, 0};
    auto load = [&](int blk) {
        const int64_t k0 = (int64_t)blk * ROWS;
        const int end = wg_last - 1 - (int)k0, l = (int)afresh(lane);        // (places of lanes are formed anew: registers are dearer)
        ks.load(Kb + k0 * a.ldk, a.ldk, end, S::place(wave, l, a.ldk), l, a.dk);
        vs.load(Vb + k0 * a.ldv, a.ldv, end, S::place(wave, l, a.ldv), l, a.dk);
        if (docs && threadIdx.x < ROWS) doc_here = (int)threadIdx.x <= end ? a.doc_k[(int64_t)b * a.Sk + k0 + threadIdx.x] : -1;
        if (docs && threadIdx.x < TILES) range_here = TILES * blk + (int)threadIdx.x < grid.key_tiles ? ranges[TILES * blk + threadIdx.x] : DocRange{0x7fffffff, -1};
    };
    auto stage = [&](unsigned cur) {
        unsigned char *at = lds + cur;
        const int l = (int)afresh(lane);
        const typename S::Place place = S::place(wave, l, 0);
        ks.put(base + cur, base + cur + G::FACTORS_AT, place, l, 1.0f, a.dk);
        vs.put(base + cur + B::BYTES, base + cur + G::FACTORS_AT + 4 * ROWS, place, l, 1.0f, a.dk);
        if (docs && threadIdx.x < ROWS) reinterpret_cast<int *>(at + G::DOCS_AT)[threadIdx.x] = doc_here;
        if (docs && threadIdx.x < TILES) reinterpret_cast<DocRange *>(at + G::DOCS_AT + ROWS * 4)[threadIdx.x] = range_here;
    };

    int blk = blocks.next((int)(all_blocks * work.split / grid.splits), lane), ahead = blocks.n;
    if (blk < blocks.n) load(blk);
    // ---- the row: query, gradient, delta ----
    const int64_t at = ((int64_t)b * a.H + head) * a.Sq + i;
    v4i qf[KS][2], of[KS][2];
    float q_down, o_down, delta = 0.0f;
    {
        float x[KS][8], y[KS][8];
        load_row<PAD, 4>(x, a.Oin + ((int64_t)b * a.Sq + i) * a.ldo + (int64_t)head * a.dk, live, part, a.dk);
        load_row<PAD, 4>(y, a.dO + ((int64_t)b * a.Sq + i) * a.lddo + (int64_t)head * a.dk, live, part, a.dk);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) delta = __builtin_fmaf(x[s][e], y[s][e], delta);
        delta = over_parts(delta, [](float p, float q) { return p + q; });
        o_down = cut_row(y, most_of_parts(most_of(y)), of);
        load_row<PAD, 4>(x, a.Q + ((int64_t)b * a.Sq + i) * a.ldq + (int64_t)head * a.dk, live, part, a.dk);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] *= a.q_up;
        q_down = cut_row(x, most_of_parts(most_of(x)), qf);
    }
    if (valid && part == 0 && wave < SETS && work.split == 0) a.delta[at] = delta;
    // probabilities come times 2^BIAS
    float lse2 = live ? __builtin_fmaf(a.Lin[at], LOG2E, -(float)BIAS) : INFINITY;
    if (lse2 == -INFINITY) lse2 = INFINITY;          // a row that saw nothing: no probability
    if (blk < blocks.n) {
        stage(0);
        ahead = blocks.next(blk + 1, lane);
        if (ahead < blocks.n) load(ahead);
    }
    __syncthreads();

    v4f acc[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) acc[n] = v4f{0.f, 0.f, 0.f, 0.f};
    // acc is 2^(BIAS + d_up) times the sum: the running exponent of ds times its key row's factor, which starts where products of dO and delta are floats
    int d_up = MOST_UP - max(0, max(__builtin_amdgcn_frexp_expf(o_down), __builtin_amdgcn_frexp_expf(delta)));
    float o_times = __builtin_ldexpf(o_down, d_up), delta_times = __builtin_ldexpf(delta, d_up);
    const float one = hidden_one();
    // what is left to a score: q_down, where more is done to it before, in the exponential's multiply-add otherwise
    const bool plain = a.cap == 0.0f && !a.slopes;
    const float down = plain ? q_down : 1.0f;

    const unsigned row_at = B::row_place16(lane) + base, column_at = B::column_place16(lane) + base;
    auto attend = [&](int blk, unsigned cur) {
        const unsigned char *here = lds + cur;
#pragma unroll 1
        for (int kt = wave / SETS; kt < TILES; kt += G::SHARES) {
            const int kt0 = blk * ROWS + 32 * kt;
            if (kt0 >= last) break;
            bool partly = kt0 + 32 > sure;
            if (docs) {
                const v2i32 range = *reinterpret_cast<const v2i32 *>(here + G::DOCS_AT + ROWS * 4 + 8 * kt);
                const DocRange of_keys = {__builtin_amdgcn_readfirstlane(range[0]), __builtin_amdgcn_readfirstlane(range[1])};
                if (!of_keys.meets(d_low, d_high)) continue;
                partly |= of_keys.low != of_keys.high || of_keys.low != d_low || d_low != d_high;
            }
            const unsigned tile_at = cur + 32 * kt * B::PITCH, row_place = afresh(row_at) + tile_at, column_place = afresh(column_at) + tile_at;
            v4f of_k[2], of_v[2];                    // factors of keys 16 t + 4 part + 0..3 of the tile and of their values
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const v4f *from = reinterpret_cast<const v4f *>(here + G::FACTORS_AT + 4 * (32 * kt + 16 * t + 4 * part));
                of_k[t] = from[0];
                of_v[t] = from[ROWS / 4];
            }
            v4f sc[2], pr[2];
            sc[0] = sc[1] = pr[0] = pr[1] = v4f{0.f, 0.f, 0.f, 0.f};
            products<4 * KS>(                        // scores of both halves of the keys, then their dP
                [&](int n, v4i (&f)[2]) {
                    const unsigned from = row_place + n / (2 * KS) * B::BYTES;
                    f[1] = B::rows16(from, 16 * (n & 1), n / 2 % KS, 1);
                    f[0] = B::rows16(from, 16 * (n & 1), n / 2 % KS, 0);
                },
                [&](int n, const v4i (&f)[2]) {
                    if (n < 2 * KS) sc[n & 1] = mfma_cut16(f, qf[n / 2 % KS], sc[n & 1]);
                    else pr[n & 1] = mfma_cut16(f, of[n / 2 % KS], pr[n & 1]);
                });
            Eight s, slope;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const v4f f = of_k[t];
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * t + e] = sc[t][e] * f[e];
            }
            if (!plain)
#pragma unroll
                for (int v = 0; v < 8; v++) s[v] *= q_down;
            const float from = (float)(row.p - kt0 - 4 * part);
            score_tile(a, s, slope, [&](int v) { return row.slope2 * __builtin_fabsf(from - (float)(16 * (v >> 2) + (v & 3))); });
            if (partly) {
                const int end = row.end - kt0 - 4 * part;
#pragma unroll
                for (int v = 0; v < 8; v++)
                    if (16 * (v >> 2) + (v & 3) >= end) s[v] = -INFINITY;
                if (docs)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const v4i d = *reinterpret_cast<const v4i *>(here + G::DOCS_AT + 4 * (32 * kt + 16 * t + 4 * part));
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (d[e] != row.doc) s[4 * t + e] = -INFINITY;
                    }
            }
            // ds times its key row's factor and 2^d_up, which is in o_times and delta_times
            Eight x;
            float most;
            auto form = [&]() {
                most = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const v4f kf = of_k[t], vf = of_v[t];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int v = 4 * t + e;
                        x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], down, -lse2)) * __builtin_fmaf(pr[t][e] * vf[e], o_times, -delta_times);
                        if (a.cap > 0.0f) x[v] *= slope[v];
                        x[v] *= kf[e];
                        most = fmaxf(most, __builtin_fabsf(x[v]));
                    }
                }
            };
            form();
            if (__builtin_amdgcn_ballot_w64(most > ROOM)) {      // (always for the first that are not zero)
                const int before = d_up;
                auto take = [&]() {
                    o_times = __builtin_ldexpf(o_down, d_up);
                    delta_times = __builtin_ldexpf(delta, d_up);
                    // A scale at which the products of dO and V have no float left, or that its inverse could not undo: from here on the row is formed again.
                    if (o_times == 0.0f || d_up < -126) o_down = o_times = NAN;
                };
                most = most_of_parts(most);
                const bool over = most > ROOM, past = most == INFINITY;
                if (past) {                                      // no float at the scale so far: by what they are at one where they are
                    d_up -= MOST_UP;
                    take();
                }
                if (__builtin_amdgcn_ballot_w64(past)) {         // (the other rows come out as they were)
                    form();
                    most = most_of_parts(most);
                }
                if (over) {
                    d_up = min(d_up + LARGEST - __builtin_amdgcn_frexp_expf(most), before);
                    take();
                }
                times(acc, two_to(d_up - before));
                form();
            }
            v4i df[2];
            cut_scaled(x, one, df);
            products<NT>(
                [&](int n, v4i (&f)[2]) {
                    f[1] = B::columns16(column_place, n, 1);
                    f[0] = B::columns16(column_place, n, 0);
                },
                [&](int n, const v4i (&f)[2]) { acc[n] = mfma_cut16(f, df, acc[n]); });
        }
    };
    unsigned cur = 0;
    while (blk < blocks.n) {
        const bool more = ahead < blocks.n;
        int after = blocks.n;
        auto bring = [&]() {
            stage(cur ^ G::STAGE);
            after = blocks.next(ahead + 1, lane);
            if (after < blocks.n) load(after);
        };
        if (more && wave >= 4) bring();
        attend(blk, cur);
        if (more && wave < 4) bring();
        __syncthreads();
        blk = ahead;
        ahead = after;
        cur ^= G::STAGE;
    }

    times(acc, two_to(-d_up - BIAS));
    if constexpr (G::SHARES == 2) {                  // the other share's keys (the last barrier has passed: no block is read any more)
        v4f *sums = reinterpret_cast<v4f *>(lds + wave % SETS * G::JOIN) + lane;
        if (wave >= SETS)
#pragma unroll
            for (int n = 0; n < NT; n++) sums[64 * n] = acc[n];
        __syncthreads();
        if (wave < SETS)
#pragma unroll
            for (int n = 0; n < NT; n++) acc[n] += sums[64 * n];
    }
    if (grid.splits > 1 && !met(grid, work, SETS * NT * 256, wave < SETS, wave, lane, reinterpret_cast<int *>(lds), {acc}, NT)) return;
    if (wave >= SETS) return;
    float seen = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen = __builtin_fmaf(acc[n][e], 0.0f, seen);
    uint64_t again = __builtin_amdgcn_ballot_w64(live && !(seen == 0.0f));
    again |= again >> 32;
    again = (again | again >> 16) & 0xffff;
    if (valid && !((again >> col) & 1)) {
        float *dq = a.dQ + ((int64_t)b * a.Sq + i) * a.lddq + (int64_t)head * a.dk;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int c = 16 * n + 4 * part;
            if (!PAD || c < a.dk) *reinterpret_cast<v4f *>(dq + c) = live ? acc[n] * a.scale : v4f{0.f, 0.f, 0.f, 0.f};
        }
    }
    for (unsigned rest = (unsigned)again; rest; rest &= rest - 1) {
        const int n = __builtin_ctz(rest);
        attn_dq_row(a, b, head, __builtin_amdgcn_readlane(i, n), (int)afresh(lane));
    }
}

template <int DK, int SETS>
struct DkvGeom : BwdGeom<DK, SETS> {
    using Base = BwdGeom<DK, SETS>;
    static constexpr int ROW_AT = 2 * Base::B::BYTES;            // of each row: factors of Q and dO, lse, delta, slope (floats), end, position, document (ints)
    static constexpr int TILE_AT = ROW_AT + Base::ROWS * 32;     // of each 32 rows: last end, first end, range of documents
    static constexpr int STAGE = (TILE_AT + Base::TILES * 16 + 255) / 256 * 256;
    static constexpr int JOIN = DK / 16 * 2048;                  // the other share's sums, of both gradients
    static constexpr int SMEM = 2 * STAGE;
    static_assert(SMEM <= 160 * 1024 && SETS * JOIN <= SMEM, "LDS");
};

template <int DK, int SETS, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, 2) k_attn_dkv(AttnArgs a, BwdGrid grid) {
    using G = DkvGeom<DK, SETS>;
    using B = typename G::B;
    constexpr int KS = DK / 32, NT = DK / 16, ROWS = G::ROWS, TILES = G::TILES;
    constexpr bool EARLY = DK <= 96;                // registers for what rows need before the products are formed
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, part = lane >> 4;
    int64_t unit;
    int tile;                                        // (causal: the first keys are those that most rows see)
    const Work work = work_of(a, grid, unit, tile);
    const int b = (int)(unit / a.Hkv), hk = (int)(unit - (int64_t)b * a.Hkv);
    const int k0 = tile * 16 * SETS, kw0 = k0 + wave % SETS * 16, key = kw0 + col;
    const AttnSeq seq = attn_seq(a, b);
    const int len = seq.len, start = seq.start;
    const bool valid = key < a.Sk, live = key < len, docs = a.doc_q != nullptr;
    int doc = 0, d_low = 0, d_high = 0, wg_low = 0, wg_high = 0;
    if (docs) {
        doc = live ? a.doc_k[(int64_t)b * a.Sk + key] : -1;
        // the ranges of the wave's keys and of the workgroup's, from those of 32
        const DocRange *ranges = grid.key_ranges + (int64_t)b * grid.key_tiles;
        d_low = wg_low = 0x7fffffff;
        d_high = wg_high = -1;
#pragma unroll
        for (int w = 0; w < SETS / 2; w++)
            if (k0 / 32 + w < grid.key_tiles) {
                const DocRange range = ranges[k0 / 32 + w];
                const int low = range.low < 0 ? ~range.low : range.low;
                wg_low = min(wg_low, low);
                wg_high = max(wg_high, range.high);
                if (w == wave % SETS / 2) {
                    d_low = low;
                    d_high = range.high;
                }
            }
        d_low = __builtin_amdgcn_readfirstlane(d_low);
        d_high = __builtin_amdgcn_readfirstlane(d_high);
        wg_low = __builtin_amdgcn_readfirstlane(wg_low);
        wg_high = __builtin_amdgcn_readfirstlane(wg_high);
    }
    // rows of a head that may see the workgroup's keys
    int first = 0, rows_end = a.Sq;
    if (a.causal) {
        if (seq.prefix <= k0) first = k0 - start > 0 ? k0 - start : 0;
        if (len - start < rows_end) rows_end = len - start;
    }
    if (k0 >= len || first >= rows_end) rows_end = 0;
    first = __builtin_amdgcn_readfirstlane(first);
    rows_end = __builtin_amdgcn_readfirstlane(rows_end);
    const DocRange *row_ranges = docs ? grid.row_ranges + (int64_t)b * grid.row_tiles : nullptr;
    Blocks<TILES> blocks(row_ranges, rows_end > 0 ? (rows_end + ROWS - 1) / ROWS : 0, grid.row_tiles, wg_low, wg_high);

    // head `g` of the group, block `blk` of it: the place of the work
    struct Place {
        int g, blk;
    };
    const int first_blk = first / ROWS, of_head = blocks.n > 0 ? blocks.n - first_blk : 0;
    const int64_t stop = (int64_t)a.G * of_head * (work.split + 1) / grid.splits;
    auto settle = [&](Place p) -> Place {            // the first place from p on with work
        while (p.g < a.G) {
            p.blk = blocks.next(p.blk, lane);
            if (p.blk < blocks.n) break;
            p.g++;
            p.blk = first_blk;
        }
        if ((int64_t)p.g * of_head + p.blk - first_blk >= stop) p.g = a.G;
        return p;
    };
    using S = Stage<DK, ROWS, WAVES, PAD>;
    S qs, os;
    const unsigned base = lds_address(lds);
    float r_lse = 0.0f, r_delta = 0.0f;
    int r_doc = 0;
    auto load = [&](Place p) {
        const int head = hk * a.G + p.g, i0 = p.blk * ROWS, end = rows_end - 1 - i0, l = (int)afresh(lane);
        qs.load(a.Q + ((int64_t)b * a.Sq + i0) * a.ldq + (int64_t)head * a.dk, a.ldq, end, S::place(wave, l, a.ldq), l, a.dk);
        os.load(a.dO + ((int64_t)b * a.Sq + i0) * a.lddo + (int64_t)head * a.dk, a.lddo, end, S::place(wave, l, a.lddo), l, a.dk);
        if (threadIdx.x < ROWS) {
            const int i = min(i0 + (int)threadIdx.x, rows_end - 1);
            const int64_t at = ((int64_t)b * a.H + head) * a.Sq + i;
            r_lse = a.Lin[at];
            r_delta = a.delta[at];
            if (docs) r_doc = a.doc_q[(int64_t)b * a.Sq + i];
        }
    };
    auto stage = [&](Place p, unsigned cur) {
        const int l = (int)afresh(lane);
        const typename S::Place place = S::place(wave, l, 0);
        qs.put(base + cur, base + cur + G::ROW_AT, place, l, a.q_up, a.dk);
        os.put(base + cur + B::BYTES, base + cur + G::ROW_AT + 4 * ROWS, place, l, 1.0f, a.dk);
        if (threadIdx.x < ROWS) {
            const int i = p.blk * ROWS + threadIdx.x;
            AttnRow row = attn_row(a, seq, i, r_doc, a.slopes ? a.slopes[hk * a.G + p.g] : 0.0f);
            if (i >= rows_end) row.end = 0;
            float *at = reinterpret_cast<float *>(lds + cur + G::ROW_AT) + threadIdx.x;
            int *ints = reinterpret_cast<int *>(at);
            at[2 * ROWS] = r_lse == -INFINITY ? INFINITY : __builtin_fmaf(r_lse, LOG2E, -(float)BIAS);        // a row that saw nothing: no probability
            at[3 * ROWS] = row.end > 0 ? r_delta : 0.0f;
            at[4 * ROWS] = row.slope2;
            ints[5 * ROWS] = row.end;
            ints[6 * ROWS] = row.p;
            ints[7 * ROWS] = row.doc;
            RowsSeen seen = rows_seen(row);
            if (of_half_wave(row.end, [](int x, int y) { return min(x, y); }) == 0) seen.sure = 0;
            if ((lane & 31) == 0) *reinterpret_cast<v4i *>(lds + cur + G::TILE_AT + 16 * (threadIdx.x >> 5)) = v4i{seen.last, seen.sure, seen.low, seen.high};
        }
    };

    Place at = {a.G, 0}, ahead = at;
    if (of_head > 0) {
        const int64_t from = (int64_t)a.G * of_head * work.split / grid.splits;
        at = settle({(int)(from / of_head), first_blk + (int)(from % of_head)});
    }
    if (at.g < a.G) load(at);
    v4i kf[KS][2], vf[KS][2];                        // this lane's key and value rows
    float k_down, v_down;
    {
        float x[KS][8];
        load_row<PAD, 4>(x, a.K + ((int64_t)b * a.kv_rows + key) * a.ldk + (int64_t)hk * a.dk, live, part, a.dk);
        k_down = cut_row(x, most_of_parts(most_of(x)), kf);
        load_row<PAD, 4>(x, a.V + ((int64_t)b * a.kv_rows + key) * a.ldv + (int64_t)hk * a.dk, live, part, a.dk);
        v_down = cut_row(x, most_of_parts(most_of(x)), vf);
    }
    if (at.g < a.G) {
        stage(at, 0);
        ahead = settle({at.g, at.blk + 1});
        if (ahead.g < a.G) load(ahead);
    }
    __syncthreads();

    v4f acc_k[NT], acc_v[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) acc_k[n] = acc_v[n] = v4f{0.f, 0.f, 0.f, 0.f};
    // acc_k is 2^BIAS d_scale times the sum of ds q, acc_v 2^BIAS p_scale times that of P dO: running scales of ds and P times their rows' factors
    float d_scale = two_to(MOST_UP), p_scale = d_scale;
    const bool plain = a.cap == 0.0f && !a.slopes;  // (as for the rows' gradient)
    const float down = plain ? k_down : 1.0f;

    const unsigned row_at = B::row_place16(lane) + base, column_at = B::column_place16(lane) + base;
    auto attend = [&](int qt, unsigned cur) {
        const v4i whole = *reinterpret_cast<const v4i *>(lds + cur + G::TILE_AT + 16 * qt);
        const int t_last = __builtin_amdgcn_readfirstlane(whole[0]), t_sure = __builtin_amdgcn_readfirstlane(whole[1]);
        if (t_last <= kw0) return;
        bool partly = t_sure < kw0 + 16;
        if (docs) {
            const int t_low = __builtin_amdgcn_readfirstlane(whole[2]), t_high = __builtin_amdgcn_readfirstlane(whole[3]);
            if (t_high < d_low || t_low > d_high) return;
            partly = true;
        }
        const unsigned tile_at = cur + 32 * qt * B::PITCH, row_place = afresh(row_at) + tile_at, column_place = afresh(column_at) + tile_at;
        const unsigned char *of_tile = lds + cur + G::ROW_AT + 4 * (32 * qt + 4 * part);     // rows 16 t + 0..3 from here: 16 bytes at 64 t
        auto of_rows = [&](int what, int t) { return *reinterpret_cast<const v4i *>(of_tile + what * ROWS * 4 + 64 * t); };
        auto floats = [&](int what, int t) { return __builtin_bit_cast(v4f, of_rows(what, t)); };
        v4f ahead[4][2];
        if (EARLY)
#pragma unroll
            for (int n = 0; n < 8; n++) ahead[n / 2][n % 2] = floats(n / 2, n % 2);
        auto of_q = [&](int t) { return EARLY ? ahead[0][t] : floats(0, t); };
        v4f sc[2], pr[2];
        sc[0] = sc[1] = pr[0] = pr[1] = v4f{0.f, 0.f, 0.f, 0.f};
        products<4 * KS>(
            [&](int n, v4i (&f)[2]) {
                const unsigned from = row_place + n / (2 * KS) * B::BYTES;
                f[1] = B::rows16(from, 16 * (n & 1), n / 2 % KS, 1);
                f[0] = B::rows16(from, 16 * (n & 1), n / 2 % KS, 0);
            },
            [&](int n, const v4i (&f)[2]) {
                if (n < 2 * KS) sc[n & 1] = mfma_cut16(f, kf[n / 2 % KS], sc[n & 1]);
                else pr[n & 1] = mfma_cut16(f, vf[n / 2 % KS], pr[n & 1]);
            });
        Eight s, dp, slope;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const v4f f = of_q(t);
#pragma unroll
            for (int e = 0; e < 4; e++) s[4 * t + e] = sc[t][e] * f[e];
        }
        if (!plain)
#pragma unroll
            for (int v = 0; v < 8; v++) s[v] *= k_down;
        if (a.cap > 0.0f || a.slopes) {
            Eight far;
            if (a.slopes)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const v4f sl = floats(4, t);
                    const v4i p = of_rows(6, t);
#pragma unroll
                    for (int e = 0; e < 4; e++) far[4 * t + e] = sl[e] * __builtin_fabsf((float)(p[e] - key));
                }
            score_tile(a, s, slope, [&](int v) { return far[v]; });
        }
        if (partly)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const v4i end = of_rows(5, t);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (key >= end[e]) s[4 * t + e] = -INFINITY;
                if (docs) {
                    const v4i d = of_rows(7, t);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (d[e] != doc) s[4 * t + e] = -INFINITY;
                }
            }
        float most_d = 0.0f, most_p = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const v4f qf = of_q(t), of = EARLY ? ahead[1][t] : floats(1, t), lse = EARLY ? ahead[2][t] : floats(2, t), delta = EARLY ? ahead[3][t] : floats(3, t);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int v = 4 * t + e;
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], down, -lse[e]));
                dp[v] = p * __builtin_fmaf(pr[t][e] * of[e], v_down, -delta[e]);
                if (a.cap > 0.0f) dp[v] *= slope[v];
                dp[v] *= qf[e];
                s[v] = p * of[e];
                most_p = fmaxf(most_p, s[v]);
                most_d = fmaxf(most_d, __builtin_fabsf(dp[v]));
            }
        }
        if (__builtin_amdgcn_ballot_w64(most_d * d_scale > ROOM || most_p * p_scale > ROOM)) {
            const float d_next = regrown(most_of_parts(most_d), d_scale), p_next = regrown(most_of_parts(most_p), p_scale);
            times(acc_k, d_next / d_scale);
            times(acc_v, p_next / p_scale);
            d_scale = d_next;
            p_scale = p_next;
        }
        v4i pf[2], df[2];
        cut_halves(s, p_scale, pf);
        cut_halves(dp, d_scale, df);
        products<2 * NT>(
            [&](int n, v4i (&f)[2]) {
                const unsigned from = column_place + (n < NT ? B::BYTES : 0);
                f[1] = B::columns16(from, n % NT, 1);
                f[0] = B::columns16(from, n % NT, 0);
            },
            [&](int n, const v4i (&f)[2]) {
                if (n < NT) acc_v[n % NT] = mfma_cut16(f, pf, acc_v[n % NT]);
                else acc_k[n % NT] = mfma_cut16(f, df, acc_k[n % NT]);
            });
    };
    unsigned cur = 0;
    while (at.g < a.G) {
        const bool more = ahead.g < a.G;
        Place after = {a.G, 0};
        auto bring = [&]() {
            stage(ahead, cur ^ G::STAGE);
            after = settle({ahead.g, ahead.blk + 1});
            if (after.g < a.G) load(after);
        };
        if (more && wave >= 4) bring();
#pragma unroll 1
        for (int qt = wave / SETS; qt < TILES; qt += G::SHARES) attend(qt, cur);
        if (more && wave < 4) bring();
        __syncthreads();
        at = ahead;
        ahead = after;
        cur ^= G::STAGE;
    }

    times(acc_k, two_to(-BIAS) / d_scale * LN2);                // (scale over what the rows of Q were taken times)
    times(acc_v, two_to(-BIAS) / p_scale);
    if constexpr (G::SHARES == 2) {
        v4f *sums = reinterpret_cast<v4f *>(lds + wave % SETS * G::JOIN) + lane;
        if (wave >= SETS)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                sums[128 * n] = acc_k[n];
                sums[128 * n + 64] = acc_v[n];
            }
        __syncthreads();
        if (wave < SETS)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                acc_k[n] += sums[128 * n];
                acc_v[n] += sums[128 * n + 64];
            }
    }
    if (grid.splits > 1 && !met(grid, work, SETS * NT * 512, wave < SETS, wave, lane, reinterpret_cast<int *>(lds), {acc_k, acc_v}, NT)) return;
    if (wave >= SETS) return;
    float seen = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen = __builtin_fmaf(acc_v[n][e], 0.0f, __builtin_fmaf(acc_k[n][e], 0.0f, seen));
    uint64_t again = __builtin_amdgcn_ballot_w64(live && !(seen == 0.0f));
    again |= again >> 32;
    again = (again | again >> 16) & 0xffff;
    if (valid && !((again >> col) & 1)) {
        const int64_t row = (int64_t)b * a.kv_rows + key;
        float *dk = a.dK + row * a.lddk + (int64_t)hk * a.dk, *dv = a.dV + row * a.lddv + (int64_t)hk * a.dk;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int c = 16 * n + 4 * part;
            if (!PAD || c < a.dk) {
                *reinterpret_cast<v4f *>(dk + c) = live ? acc_k[n] : v4f{0.f, 0.f, 0.f, 0.f};
                *reinterpret_cast<v4f *>(dv + c) = live ? acc_v[n] : v4f{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    for (unsigned rest = (unsigned)again; rest; rest &= rest - 1) attn_dkv_row(a, b, hk, kw0 + __builtin_ctz(rest), (int)afresh(lane));
}

template <auto KERNEL>
int launch_tiles(int smem, const AttnArgs &a, BwdGrid grid, const char *what) {
    static bool attr_set = false;
    if (!attr_set) {
        AXHIP_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, smem), "hipFuncSetAttribute");
        attr_set = true;
    }
    const int64_t all = grid.units * grid.tiles * grid.splits;
    for (grid.first = 0; grid.first < all; grid.first += GRID_MOST) {
        const int64_t left = all - grid.first;
        hipLaunchKernelGGL(KERNEL, dim3((unsigned)(left < GRID_MOST ? left : GRID_MOST)), dim3(64 * WAVES), smem, kStream, a, grid);
        if (int rc = check_launch(what)) return rc;
    }
    return AXHIP_OK;
}

// How the `length` rows (or keys) of each unit are shared out, each tile over `blocks` blocks of the other side: tiles of 128, or of 64 with two shares, and what a tile runs over whole
// or split to several workgroups.  The least time by a model, in blocks of a tile of 64 (of 128: WIDE each): a workgroup's start and end are START of them, and splits cost MEET and
// PART each for the last one to add; rounds of workgroups over the CUs, or, causal, the longest, the pairs that fall on one CU, or all of them evenly.  (us:
//   tiles of 64 -> 128: 64 heads of [2048, 64] 1038 -> 836, 32 of [1000, 128] 243 -> 188, 32 causal ones of [2048, 128] 491 -> 388, but 32 of [600, 128] 84 -> 113, 16 of [2048, 64] 154 -> 204;
//   whole -> split: causal, 8 heads, 2 of keys, of [500, 64] 96 -> 43, 16, 4 of keys, of [1000, 128] 281 -> 129, 4 heads of [2048, 128] without a mask 218 -> 141, but with splits for two rounds 182;
//   64 -> 128 and split in two: causal, 2 x 16, 8 of keys, of [2048, 128] under a cap 457 -> 444, of [1500, 96] 254 -> 225.)
struct Plan {
    bool wide;
    int64_t units;
    int tiles, splits;
    size_t part;                                     // floats that a split leaves, for each column of a sum
};
Plan plan_of(const AttnArgs &a, int64_t units, int64_t length, int64_t blocks) {
    Plan p = {false, units, 0, 1, 0};
    if (units == 0 || length == 0) return p;
    constexpr double START = 8.0, WIDE = 1.75, MEET = 1.0, PART[] = {0.1, 0.6};
    const int64_t cus = cu_count();
    double best = INFINITY;
    for (int wide = 0; wide < 2; wide++) {
        const int64_t tiles = wide ? (length + 127) / 128 : (length + 63) / 64, work = units * tiles;
        for (int64_t s = 1; s == 1 || (work < 2 * cus && s <= std::min<int64_t>(blocks, 32)); s++) {
            const double each = (wide ? WIDE : 1.0) * (double)blocks / (double)s, start = START + (s > 1 ? MEET + PART[wide] * (double)s : 0.0);
            const double rounds = (double)(work * s) / (double)cus;
            double time = start + each;
            if (!a.causal) time *= std::ceil(rounds);
            else if (rounds > 2.0) time = std::max(time, rounds * (start + 0.5 * each));
            else if (rounds > 1.0) time = std::max(time, 2.0 * (start + (1.0 - 1.0 / rounds) * each));
            if (time < 0.98 * best) {
                best = time;
                p.wide = wide != 0;
                p.tiles = (int)tiles;
                p.splits = (int)s;
            }
        }
    }
    const int64_t work = units * p.tiles, rows = p.wide ? 128 : 64;
    if (p.splits > 1) p.part = (size_t)work * p.splits * rows;
    return p;
}

template <int DK, bool PAD>
int launch_bwd(const AttnArgs &a, BwdGrid grid, const Plan &of_rows, const Plan &of_keys) {
    auto set = [&](const Plan &p) {
        grid.units = p.units;
        grid.tiles = p.tiles;
        grid.splits = p.splits;
    };
    if (a.Sq > 0) {
        set(of_rows);
        if (int rc = of_rows.wide ? launch_tiles<k_attn_dq<DK, 8, PAD>>(DqGeom<DK, 8>::SMEM, a, grid, "attn_bwd queries")
                                  : launch_tiles<k_attn_dq<DK, 4, PAD>>(DqGeom<DK, 4>::SMEM, a, grid, "attn_bwd queries"))
            return rc;
    }
    set(of_keys);
    return of_keys.wide ? launch_tiles<k_attn_dkv<DK, 8, PAD>>(DkvGeom<DK, 8>::SMEM, a, grid, "attn_bwd keys")
                        : launch_tiles<k_attn_dkv<DK, 4, PAD>>(DkvGeom<DK, 4>::SMEM, a, grid, "attn_bwd keys");
}

}  // namespace

namespace axhip {

int attn_bwd_tiles(AttnArgs &a) {
    BwdGrid grid = {};
    const size_t deltas = ((size_t)a.B * a.H * a.Sq * sizeof(float) + 15) & ~size_t(15);
    size_t bytes = deltas;
    if (a.doc_k) {
        grid.key_tiles = (int)(((int64_t)a.Sk + 31) / 32);
        grid.row_tiles = (int)(((int64_t)a.Sq + 31) / 32);
        bytes += (size_t)a.B * (grid.key_tiles + grid.row_tiles) * 8;
    }
    const int width = (a.dk + 31) / 32 * 32;
    const int64_t rows = width <= 64 ? 128 : 64;     // of a block
    const Plan of_rows = plan_of(a, (int64_t)a.B * a.H, a.Sq, (a.Sk + rows - 1) / rows), of_keys = plan_of(a, (int64_t)a.B * a.Hkv, a.Sk, a.G * ((a.Sq + rows - 1) / rows));
    const size_t parts_at = (bytes + 15) & ~size_t(15), parts = std::max(of_rows.part, 2 * of_keys.part) * width * sizeof(float);
    if (parts) {
        bytes = parts_at + parts;
        auto tiles = [](const Plan &p) { return p.splits > 1 ? p.units * p.tiles : 0; };
        grid.arrivals = strip_counters((size_t)std::max(tiles(of_rows), tiles(of_keys)));
        if (!grid.arrivals) return AXHIP_ERR_ALLOC;
    }
    char *ws = static_cast<char *>(workspace(bytes));
    if (!ws) return AXHIP_ERR_ALLOC;
    a.delta = reinterpret_cast<float *>(ws);
    grid.parts = reinterpret_cast<float *>(ws + parts_at);
    if (a.doc_k) {
        grid.key_ranges = reinterpret_cast<DocRange *>(ws + deltas);
        grid.row_ranges = reinterpret_cast<DocRange *>(ws + deltas + (size_t)a.B * grid.key_tiles * 8);
        if (int rc = doc_ranges(a.doc_k, a.B, a.Sk, ws + deltas)) return rc;
        if (int rc = doc_ranges(a.doc_q, a.B, a.Sq, ws + deltas + (size_t)a.B * grid.key_tiles * 8)) return rc;
    }
    note_kernel("attn_grad_tiles");
    auto run = [&](auto width) {
        constexpr int DK = decltype(width)::value;
        return a.dk < DK ? launch_bwd<DK, true>(a, grid, of_rows, of_keys) : launch_bwd<DK, false>(a, grid, of_rows, of_keys);
    };
    if (a.dk <= 32) return run(std::integral_constant<int, 32>());
    if (a.dk <= 64) return run(std::integral_constant<int, 64>());
    if (a.dk <= 96) return run(std::integral_constant<int, 96>());
    return run(std::integral_constant<int, 128>());
}

}  // namespace axhip
