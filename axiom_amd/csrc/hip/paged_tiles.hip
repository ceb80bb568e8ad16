// Attention over a paged cache: tiles of queries on the f16 matrix core.
//
// A workgroup of eight waves owns 256 rows of queries (the new tokens of a sequence for all query heads that share keys, token by token), a wave 32 of them, or 128, two waves 32 of them and
// half of the keys each.  Keys and values come from their pages in blocks of 64 (128 of heads up to 64) and stand in LDS as f16, twice, so that the numbers of the cache are converted once for
// all rows; they are f16 exactly, so a product of fp32 is two of f16 terms, the query's or the probability's (f16x2.h).  The tiles of scores and outputs, the online softmax and its
// running reference are those of attn_fwd.hip.
// What rows see goes up with their positions: blocks before the window of a workgroup's first row, but for the first tokens that stay visible, and behind its last row's position are not
// fetched, 32-key tiles that no row of a wave sees not computed, and only tiles that some row sees in part pay for the mask.
// Where tiles would leave CUs idle, ranges of their keys go to workgroups of their own, as many as a tile's blocks ask for, and a second launch adds what they leave, in order.
//
// Bound by vector instructions (some 150 for a tile of 32 x 32 and, of the block's conversion, 25 to 75) and products (32 for heads of 128, 16 for 64), one kind after the other in a wave, of which the two
// waves of a SIMD overlap little.  Two chunks of 2048 and 1564 tokens over up to 4096 int8 keys, 32 heads, 8 of keys, of 128 take 307 to 319 us, 504 to 486 TFLOP/s of fp32 products (two f16 products each: a large library product
// in f16 does 1175); f16 317 to 331; four prompts of 2636 to 4096 in windows of 1024, 16 heads of 64, 4 bits 191, of which conversion is 11 %, barriers 6 and the scores' products 22; 64 tokens over 8192 int8 keys, 32 heads, 8 of keys 29 to 31 and 9
// for the sums of 32 ranges (with 128 rows 33 and 7: level; the ranges leave 34 MB, twice the cache that is read).
#include <algorithm>

#include "attn_launch.h"
#include "attn_tiles.h"
#include "paged.h"
#include "paged_share.h"

namespace {
using namespace axhip;

constexpr int WAVES = 8, SPLITS_MOST = PAGED_SPLITS;

template <int DK, int SETS>
struct TileGeom {
    static constexpr int BQ = 32 * SETS, BKV = DK <= 64 ? 128 : 64, SHIFT = DK <= 64 ? 7 : 6, SHARES = WAVES / SETS, PIECES = DK / 8;
    using B = Block<DK, BKV>;
    static constexpr int V_AT = B::PLANE, FACTORS_AT = 2 * B::PLANE;   // factors of each key row, then of each value row
    static constexpr int HOLES_AT = FACTORS_AT + BKV * 8;        // a word a wave: whether keys that it brought have no page
    static constexpr int STAGE = (HOLES_AT + 4 * WAVES + 255) / 256 * 256;
    static constexpr int SHARE = PIECES * 1024 + 256;            // the other share's sums: a wave's pieces [64] v4f, then maxima and sums [2][32]
    static constexpr int BYTES = 2 * STAGE, SMEM = SHARES > 1 && SETS * SHARE > BYTES ? SETS * SHARE : BYTES;
    static_assert(SMEM <= 160 * 1024, "LDS");
    static constexpr int PART = SETS * (PIECES * 256 + 64);      // floats that a range leaves in memory: of each 32 rows the pieces, then maxima and sums
};

// Where a workgroup's rows are: `rows` of them (0: none of this form's), the first of which is the row of token i0 of sequence b and of head g0 of those that share keys
struct Place {
    int b, rows, i0;
    unsigned g0;
};
template <int BQ>
__device__ __forceinline__ Place place_of(const PagedArgs &a, const PagedTileGrid &grid, int64_t slot, int lane, KvSeq &seq) {
    const KvPages &kv = a.pages;
    const int64_t G = a.attn.G;
    Place p = {0, 0, 0, 0};
    int64_t tile;
    if (kv.first) {
        // sequence b's slots are those from first[b] G / BQ + b on
        p.b = kv_find(kv, lane, [&](int k, int first) { return first * G / BQ + k <= slot; });
        if (p.b >= kv.B) return p;
        tile = slot - (min(max(kv.first[p.b], 0), kv.T) * G / BQ + p.b);
    } else if (grid.slots >> 32 == 0) {
        p.b = (int)((unsigned)slot / (unsigned)grid.per);
        tile = (unsigned)slot - (unsigned)p.b * (unsigned)grid.per;
    } else {
        p.b = (int)(slot / grid.per);
        tile = slot - p.b * grid.per;
    }
    seq = kv_seq(kv, p.b);
    const int64_t rows = G * seq.n, r0 = tile * BQ;
    if (rows < grid.least || tile < 0 || r0 >= rows) return p;
    p.rows = (int)min(rows - r0, (int64_t)BQ);
    p.i0 = r0 >> 32 == 0 ? (int)((unsigned)r0 / (unsigned)a.attn.G) : (int)(r0 / G);
    p.g0 = (unsigned)(r0 - p.i0 * G);
    return p;
}

// How many ranges a tile's blocks are shared out in: as many as their count asks for
__device__ __forceinline__ unsigned ranges_of(const PagedTileGrid &grid, const PagedTiles &blocks) {
    return (unsigned)min(max((blocks.all + grid.range - 1) / grid.range, 1), grid.splits);
}

template <int DK, int SETS, int TYPE, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, 2) k_paged_tiles(PagedArgs a, PagedTileGrid grid) {
    using G = TileGeom<DK, SETS>;
    using B = typename G::B;
    using T = KvType<TYPE>;
    constexpr int KS = DK / 16, DT = DK / 32, BKV = G::BKV, TILES = BKV / 32, BQ = G::BQ;
    using S = BlockShare<DK, T::BITS, BKV, 64 * WAVES>;
    constexpr int COLS = S::COLS, LANES = S::LANES, PASSES = S::PASSES, PLACES = S::PLACES;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const KvPages &kv = a.pages;
    const AttnArgs &at = a.attn;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 31, fhalf = lane >> 5;

    // a sequence's last tiles, the longest, first; heads of keys, and then ranges, go to the XCDs in turn, each of which has an L2 (the ranges behind all first ones: 175 us for 159)
    const unsigned rest = blockIdx.x / (unsigned)kv.heads, of_slot = rest / (unsigned)grid.splits, split = rest - of_slot * (unsigned)grid.splits;
    const int64_t slot = grid.slots - 1 - (grid.first + of_slot);
    const int hk = (int)(blockIdx.x - rest * (unsigned)kv.heads);
    KvSeq seq = {0, 0, 0};
    const Place place = place_of<BQ>(a, grid, slot, lane, seq);
    if (place.rows == 0) return;
    const int b = place.b;
    const int rows_here = place.rows, mine = wave % SETS * 32 + frow;
    const bool valid = mine < rows_here;
    // (the tile's first row is one of token i0, its group's head number g0)
    const unsigned G0 = (unsigned)at.G, r = place.g0 + (unsigned)(valid ? mine : rows_here - 1), over = r / G0;
    const int i = place.i0 + (int)over, head = hk * at.G + (int)(r - over * G0);
    auto token = [&](int of) { return place.i0 + (int)((place.g0 + (unsigned)of) / G0); };
    PagedRow row = paged_row(a, seq, i);
    if (!valid) row.end = 0;
    const bool live = row.end > 0;
    // what the workgroup's rows see together, and the wave's
    const PagedRow wg_low = paged_row(a, seq, place.i0), wg_high = paged_row(a, seq, token(rows_here - 1));
    const int w0 = min(wave % SETS * 32, rows_here - 1), w1 = min(wave % SETS * 32 + 31, rows_here - 1);
    const PagedRow low = paged_row(a, seq, token(w0)), high = paged_row(a, seq, token(w1));
    const int last = wave % SETS * 32 < rows_here ? high.end : 0;
    const PagedTiles blocks = paged_tiles_of(a, wg_low.begin, wg_high.end, G::SHIFT);
    const unsigned ranges = ranges_of(grid, blocks);
    if (split >= ranges) return;
    const int n_begin = (int)((unsigned)blocks.all * split / ranges), n_end = (int)((unsigned)blocks.all * (split + 1) / ranges);
    const float slope2 = at.slopes ? at.slopes[head] * at.bias2 : 0.0f;

    const unsigned base = lds_address(lds);
    // A pass brings 16 bytes a thread (paged_share.h).
    v4i x[PASSES];
    unsigned scales[PASSES];
    int entry[PLACES];
    unsigned gone = 0;                               // a bit a place: its key has no page
    const int32_t *const entries = kv.table + (int64_t)b * kv.table_ld;
    // where this lane's bytes of row zero of a page zero are, and the scale of that row
    const unsigned char *const k0 = kv.k + kv_row_at(kv, 0, hk, 0) + 16 * ((int)threadIdx.x % LANES), *const s0 = kv.k_scale + kv_scale_at(kv, 0, hk, 0);
    const int64_t to_v = kv.v - kv.k, to_v_scale = kv.v_scale - kv.k_scale;
    auto row_of = [&](int pass) { return S::row((int)threadIdx.x, pass); };
    auto has_row = [&](int pass) { return S::has_row((int)threadIdx.x, pass); };
    auto pos_of = [&](int n, int place) { return blocks.tile(n) * BKV + row_of(place) % BKV; };
    auto look = [&](int n) {
#pragma unroll
        for (int p = 0; p < PLACES; p++) entry[p] = entries[(unsigned)min(pos_of(n, p), wg_high.end - 1) >> kv.shift];
    };
    auto fetch = [&](int n) {
        const int c = (int)threadIdx.x % LANES;
        gone = 0;
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            x[p] = v4i{0, 0, 0, 0};
            scales[p] = 0;
        }
#pragma unroll
        for (int p = 0; p < PLACES; p++) {
            const int pos = pos_of(n, p);
            const bool page = pos < wg_high.end && kv_is_page(kv, entry[p]);
            if (S::misses((int)threadIdx.x, p, page)) gone |= 1u << p;
            if (page && has_row(p)) {
                const unsigned in_page = (unsigned)pos & ((1u << kv.shift) - 1);
                const unsigned char *const k = k0 + ((uint64_t)(unsigned)entry[p] * kv.page_bytes + __umul24(in_page, (unsigned)kv.row_bytes));
                const unsigned char *const k_scale = s0 + ((uint64_t)(unsigned)entry[p] * kv.page_scales + 4 * in_page);
                const bool some = (!PAD && DK != 96) || 16 * c < kv.row_bytes;
                if (PASSES > 1) {
                    if (some) {
                        x[p] = *reinterpret_cast<const v4i *>(k);
                        x[(p + PLACES) % PASSES] = *reinterpret_cast<const v4i *>(k + to_v);
                    }
                    scales[p] = *reinterpret_cast<const unsigned *>(k_scale);
                    scales[(p + PLACES) % PASSES] = *reinterpret_cast<const unsigned *>(k_scale + to_v_scale);
                } else {
                    const bool of_v = row_of(p) >= BKV;
                    if (some) x[p] = *reinterpret_cast<const v4i *>(of_v ? k + to_v : k);
                    scales[p] = *reinterpret_cast<const unsigned *>(of_v ? k_scale + to_v_scale : k_scale);
                }
            }
        }
    };
    auto stage = [&](unsigned cur) {
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const int at_row = row_of(p), c = (int)threadIdx.x % LANES, in_block = at_row % BKV;
            if (has_row(p)) {
                const bool of_v = PASSES > 1 ? p >= PLACES : at_row >= BKV;
                const unsigned to = base + cur + (of_v ? G::V_AT : 0);
                if (DK != 96 || c * COLS < DK) {
                    if constexpr (TYPE == AXHIP_KV_F16) write_chunk(to + B::at(in_block, c), x[p]);
                    if constexpr (TYPE == AXHIP_KV_I8) {
                        int h[8];
#pragma unroll
                        for (int e = 0; e < 4; e++) kv_bytes((unsigned)x[p][e], h[2 * e], h[2 * e + 1]);
                        write_chunk(to + B::at(in_block, 2 * c), v4i{h[0], h[1], h[2], h[3]});
                        write_chunk(to + B::at(in_block, 2 * c + 1), v4i{h[4], h[5], h[6], h[7]});
                    }
                    if constexpr (TYPE == AXHIP_KV_MX4) {
                        const float up = mx4_up(scales[p], mx4_top(scales[p]), c);
#pragma unroll
                        for (int e = 0; e < 4; e++) write_chunk(to + B::at(in_block, 4 * c + e), kv_nibbles((unsigned)x[p][e], up));
                    }
                }
                if (c == 0) {
                    const float f = kv_factor<TYPE>(scales[p]);
                    // (the sign of a value's factor says that there is no page)
                    write_float(base + cur + G::FACTORS_AT + 4 * at_row, !of_v ? f : ((gone >> (p % PLACES)) & 1) ? -0.0f : f * T::VALUE_UP * VALUES_DOWN);
                }
            }
        }
        const uint64_t any = __builtin_amdgcn_ballot_w64(gone != 0);
        if (lane == 0) *reinterpret_cast<int *>(lds + cur + G::HOLES_AT + 4 * wave) = any != 0;
    };

    int n = n_begin;
    if (n < n_end) {
        look(n);
        fetch(n);
        if (n + 1 < n_end) look(n + 1);
    }
    v4i qf[KS][2];                                   // step s: columns 16 s + 8 * half .. + 7 of this lane's query
    float q_down;
    {
        const float *q = at.Q + ((int64_t)seq.first + i) * at.ldq + (int64_t)head * kv.dk;
        float y[KS][8];
        load_row<PAD, 2>(y, q, live, fhalf, kv.dk);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) y[s][e] *= at.q_up;
        const float most = most_of(y);
        q_down = cut_row(y, fmaxf(most, __shfl_xor(most, 32, 64)), qf);
    }
    if (n < n_end) {
        stage(0);
        if (n + 1 < n_end) fetch(n + 1);
        if (n + 2 < n_end) look(n + 2);
    }
    __syncthreads();

    v16f acc[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[d][v] = 0.0f;
    float ref = ATTN_LOWEST, l_run = 0.0f;           // as in attn_fwd.hip: acc is 2^VALUE_BIAS times the sum
    const float one = hidden_one();

    const unsigned row_at = B::row_place(lane) + base, column_at = B::column_place(lane) + base + G::V_AT;
    auto attend = [&](int blk, unsigned cur) {
        const unsigned char *here = lds + cur;
        const v4i h0 = *reinterpret_cast<const v4i *>(here + G::HOLES_AT), h1 = *reinterpret_cast<const v4i *>(here + G::HOLES_AT + 16);
        const bool holes = __builtin_amdgcn_readfirstlane(h0[0] | h0[1] | h0[2] | h0[3] | h1[0] | h1[1] | h1[2] | h1[3]) != 0;
#pragma unroll 1
        for (int kt = wave / SETS; kt < TILES; kt += G::SHARES) {
            const int kt0 = blk * BKV + 32 * kt;
            if (kt0 >= last) break;
            if (kt0 + 32 <= low.begin && kt0 >= a.sinks) continue;
            const bool partly = holes || kt0 + 32 > low.end || (kt0 < high.begin && kt0 + 32 > a.sinks);
            const unsigned tile_at = cur + 32 * kt * B::PITCH, row_place = afresh(row_at) + tile_at, column_place = afresh(column_at) + tile_at;
            auto factors = [&](int what, int g) {    // of keys 8 g + 4 * half + 0..3 of the tile
                return *reinterpret_cast<const v4f *>(here + G::FACTORS_AT + what * BKV * 4 + 4 * (32 * kt + 8 * g + 4 * fhalf));
            };
            v4f kf[4], vf[4];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                kf[g] = factors(0, g);
                vf[g] = factors(1, g);
            }
            v16f s;
#pragma unroll
            for (int v = 0; v < 16; v++) s[v] = 0.0f;
            __builtin_amdgcn_s_setprio(1);
            if constexpr (DK <= 64) {
                v4i f[KS];
#pragma unroll
                for (int k = 0; k < KS; k++) f[k] = B::rows(row_place, k, 0);
                __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    s = mfma_halves(f[k], qf[k][1], s);
                    s = mfma_halves(f[k], qf[k][0], s);
                }
            } else
            products<KS>([&](int k, v4i (&f)[2]) { f[0] = B::rows(row_place, k, 0); },
                         [&](int k, const v4i (&f)[2]) {
                             s = mfma_halves(f[0], qf[k][1], s);
                             s = mfma_halves(f[0], qf[k][0], s);
                         });
            v4i vfrag[2 * DT];
            if constexpr (DK <= 64) {
                __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
                for (int m = 0; m < 2 * DT; m++) vfrag[m] = B::columns(column_place, 16 * (m / DT), m % DT, 0);
                __builtin_amdgcn_sched_barrier(0x6);
            }
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * g + e] *= kf[g][e];
            // what is left to the score: q_down, here where more is done to it, in the exponential's multiply-add otherwise
            const bool plain = at.cap == 0.0f && !at.slopes;
            const float down = plain ? q_down : 1.0f;
            if (__builtin_expect(!plain, 0))
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] *= q_down;
            if (__builtin_expect(at.cap > 0.0f, 0)) {
                float big = 0.0f;
#pragma unroll
                for (int v = 0; v < 16; v++) big = fmaxf(big, __builtin_fabsf(s[v]));
                if (__builtin_amdgcn_ballot_w64(!(big < at.cap_near)))
#pragma unroll
                    for (int v = 0; v < 16; v++) s[v] = capped(at, s[v]).score;
                else
#pragma unroll
                    for (int v = 0; v < 16; v++) s[v] = capped_near(at, s[v]).score;
            }
            if (__builtin_expect(at.slopes != nullptr, 0)) {
                const float from = (float)(row.p - kt0 - 4 * fhalf);
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] = __builtin_fmaf(-slope2, from - (float)(8 * (v >> 2) + (v & 3)), s[v]);
            }
            if (__builtin_expect(partly, 0)) {
                const int end = row.end - kt0 - 4 * fhalf, begin = row.begin - kt0 - 4 * fhalf, first = a.sinks - kt0 - 4 * fhalf;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int j = 8 * (v >> 2) + (v & 3);
                    if (j >= end || (j < begin && j >= first)) s[v] = -INFINITY;
                }
                if (holes)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (__float_as_uint(vf[v >> 2][v & 3]) == 0x80000000u) s[v] = -INFINITY;
            }
            // ---- online softmax ----
            v16f w;
            float most, l_blk;
            auto weigh = [&]() {
                most = l_blk = 0.0f;
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], down, -ref));
                    l_blk += p;
                    w[v] = p * vf[v >> 2][v & 3];
                    most = fmaxf(most, w[v]);
                }
            };
            weigh();
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > ROOM) != 0, 0)) {      // (always for the first finite scores)
                most = fmaxf(most, __shfl_xor(most, 32, 64));
                float top = -INFINITY;
#pragma unroll
                for (int v = 0; v < 16; v++) top = fmaxf(top, __builtin_fmaf(s[v], down, __builtin_amdgcn_logf(vf[v >> 2][v & 3])));
                top = fmaxf(top, __shfl_xor(top, 32, 64)) - (float)LARGEST;
                const float next = most > ROOM ? fmaxf(ref, top) : ref, alpha = __builtin_amdgcn_exp2f(ref - next);
                l_run = scaled(l_run, ref - next);
                ref = next;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) acc[d][v] *= alpha;
                weigh();
            }
            l_run += l_blk;
            // ---- O^T += V^T P^T ----
            v4i pf[2][2];
            cut_scaled(w, 0, one, pf[0]);
            cut_scaled(w, 1, one, pf[1]);
            __builtin_amdgcn_s_setprio(1);
            if constexpr (DK <= 64) {
#pragma unroll
                for (int m = 0; m < 2 * DT; m++) {
                    acc[m % DT] = mfma_halves(vfrag[m], pf[m / DT][1], acc[m % DT]);
                    acc[m % DT] = mfma_halves(vfrag[m], pf[m / DT][0], acc[m % DT]);
                }
            } else
            products<2 * DT>([&](int m, v4i (&f)[2]) { f[0] = B::columns(column_place, 16 * (m / DT), m % DT, 0); },
                             [&](int m, const v4i (&f)[2]) {
                                 acc[m % DT] = mfma_halves(f[0], pf[m / DT][1], acc[m % DT]);
                                 acc[m % DT] = mfma_halves(f[0], pf[m / DT][0], acc[m % DT]);
                             });
            __builtin_amdgcn_s_setprio(0);
        }
    };
    // Two blocks in LDS, the next in registers, the pages of the one after that.  The two waves of a SIMD (w, w + 4) put it beside the current block before and after that is multiplied, so
    // that one converts while the other's products run.
    unsigned cur = 0;
    for (; n < n_end; n++) {
        auto bring = [&]() {
            if (n + 1 < n_end) stage(cur ^ G::STAGE);
            if (n + 2 < n_end) fetch(n + 2);
            if (n + 3 < n_end) look(n + 3);
        };
        if (wave >= 4) bring();
        attend(blocks.tile(n), cur);
        if (wave < 4) bring();
        __syncthreads();
        cur ^= G::STAGE;
    }

    float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    if constexpr (G::SHARES == 2) {                  // the other share's keys (the last barrier has passed: no block is read any more)
        unsigned char *share = lds + wave % SETS * G::SHARE;
        v4f *sums = reinterpret_cast<v4f *>(share) + lane;
        float *of_row = reinterpret_cast<float *>(share + G::SHARE - 256) + frow;
        if (wave >= SETS) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int g = 0; g < 4; g++) sums[64 * (4 * d + g)] = v4f{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
            if (fhalf == 0) {
                of_row[0] = ref;
                of_row[32] = l_tot;
            }
        }
        __syncthreads();
        if (wave >= SETS) return;
        const float other = of_row[0], both = fmaxf(ref, other), ours = __builtin_amdgcn_exp2f(ref - both), theirs = __builtin_amdgcn_exp2f(other - both);
        l_tot = scaled(l_tot, ref - both) + scaled(of_row[32], other - both);
        ref = both;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4f sum = sums[64 * (4 * d + g)];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[d][4 * g + e] = __builtin_fmaf(acc[d][4 * g + e], ours, sum[e] * theirs);
            }
    }
    if (ranges > 1) {
        float *part = grid.parts + ((slot * kv.heads + hk) * grid.splits + split) * G::PART + wave * (G::PART / SETS);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<v4f *>(part + ((4 * d + g) * 64 + lane) * 4) =
                    v4f{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]} * two_to(-T::VALUE_BIAS);
        if (fhalf == 0) {
            part[G::PIECES * 256 + frow] = ref;
            part[G::PIECES * 256 + 32 + frow] = l_tot;
        }
        return;
    }

    // ---- normalise and write: a lane owns its query's columns 32 d + 8 g + 4 * half .. + 3 ----
    float seen = l_tot * 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) seen = __builtin_fmaf(acc[d][v], 0.0f, seen);
    const bool unfit = live && (!(seen == 0.0f) || l_tot == 0.0f);
    uint64_t again = __builtin_amdgcn_ballot_w64(unfit);
    again |= again >> 32;
    const float inv = 1.0f / l_tot;
    if (valid && !((again >> frow) & 1)) {
        const int64_t to = (int64_t)seq.first + i;
        float *o = at.O + to * at.ldo + (int64_t)head * kv.dk;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int col = 32 * d + 8 * g + 4 * fhalf;
                v4f out;
#pragma unroll
                for (int e = 0; e < 4; e++) out[e] = live ? acc[d][4 * g + e] * two_to(-T::VALUE_BIAS) * inv : 0.0f;
                if (!PAD || col < kv.dk) *reinterpret_cast<v4f *>(o + col) = out;
            }
        if (at.L && fhalf == 0) at.L[to * at.H + head] = live ? (ref + __builtin_amdgcn_logf(l_tot)) * LN2 : -INFINITY;
    }
    for (unsigned some = (unsigned)again; some; some &= some - 1) {
        const int m = __builtin_ctz(some);
        paged_again<TYPE>(a, b, seq, __builtin_amdgcn_readlane(head, m), __builtin_amdgcn_readlane(i, m), (int)afresh(lane));
    }
}

// What ranges of keys left, added in order: a workgroup for 32 rows and 32 columns, a quarter of the ranges a wave
template <int DK, int SETS, int TYPE>
__global__ void __launch_bounds__(256) k_paged_join(PagedArgs a, PagedTileGrid grid) {
    using G = TileGeom<DK, SETS>;
    constexpr int BQ = G::BQ, DT = DK / 32;
    __shared__ v4f sums[3][4][64];
    __shared__ float of_rows[4][2][32];
    const KvPages &kv = a.pages;
    const AttnArgs &at = a.attn;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 31, fhalf = lane >> 5;
    const unsigned of_set = blockIdx.x / DT, d = blockIdx.x % DT, of_unit = of_set / SETS, set = of_set % SETS, of_slot = of_unit / (unsigned)kv.heads;
    const int hk = (int)(of_unit - of_slot * (unsigned)kv.heads);
    const int64_t slot = grid.first + of_slot, unit = slot * kv.heads + hk;
    KvSeq seq = {0, 0, 0};
    const Place place = place_of<BQ>(a, grid, slot, lane, seq);
    const int rows_here = place.rows - 32 * (int)set;
    if (rows_here <= 0) return;
    const bool valid = frow < rows_here;
    const unsigned r = place.g0 + 32 * set + (unsigned)(valid ? frow : rows_here - 1), over = r / (unsigned)at.G;
    const int i = place.i0 + (int)over, head = hk * at.G + (int)(r - over * (unsigned)at.G);
    const PagedRow low = paged_row(a, seq, place.i0), high = paged_row(a, seq, place.i0 + (int)((place.g0 + (unsigned)place.rows - 1) / (unsigned)at.G));
    const int ranges = (int)ranges_of(grid, paged_tiles_of(a, low.begin, high.end, G::SHIFT));
    if (ranges == 1) return;                         // (it wrote its rows itself)
    const bool live = valid && paged_row(a, seq, i).end > 0;
    const float *parts = grid.parts + unit * grid.splits * G::PART + set * (G::PART / SETS);
    // this wave's ranges, against their largest reference
    const int from = ranges * wave / 4, to = ranges * (wave + 1) / 4;
    float m = ATTN_LOWEST, l = 0.0f;
    v4f sum[4];
#pragma unroll
    for (int g = 0; g < 4; g++) sum[g] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = from; s < to; s++) {
        const float *part = parts + (int64_t)s * G::PART;
        const float ref = part[G::PIECES * 256 + frow], more = part[G::PIECES * 256 + 32 + frow], both = fmaxf(m, ref);
        const float ours = __builtin_amdgcn_exp2f(m - both), theirs = __builtin_amdgcn_exp2f(ref - both);
        l = scaled(l, m - both) + scaled(more, ref - both);
        m = both;
#pragma unroll
        for (int g = 0; g < 4; g++) sum[g] = sum[g] * ours + *reinterpret_cast<const v4f *>(part + ((4 * d + g) * 64 + lane) * 4) * theirs;
    }
    if (wave > 0)
#pragma unroll
        for (int g = 0; g < 4; g++) sums[wave - 1][g][lane] = sum[g];
    if (fhalf == 0) {
        of_rows[wave][0][frow] = m;
        of_rows[wave][1][frow] = l;
    }
    __syncthreads();
    if (wave > 0) return;
    float top = m;
#pragma unroll
    for (int w = 1; w < 4; w++) top = fmaxf(top, of_rows[w][0][frow]);
    l = scaled(l, m - top);
    const float first = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int g = 0; g < 4; g++) sum[g] *= first;
#pragma unroll
    for (int w = 1; w < 4; w++) {
        const float ref = of_rows[w][0][frow], weight = __builtin_amdgcn_exp2f(ref - top);
        l += scaled(of_rows[w][1][frow], ref - top);
#pragma unroll
        for (int g = 0; g < 4; g++) sum[g] += sums[w - 1][g][lane] * weight;
    }
    float seen = l * 0.0f;
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen = __builtin_fmaf(sum[g][e], 0.0f, seen);
    uint64_t again = __builtin_amdgcn_ballot_w64(live && (!(seen == 0.0f) || l == 0.0f));
    again |= again >> 32;
    if (valid && !((again >> frow) & 1)) {
        const int64_t row = (int64_t)seq.first + i;
        float *o = at.O + row * at.ldo + (int64_t)head * kv.dk;
        const float inv = 1.0f / l;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int col = 32 * (int)d + 8 * g + 4 * fhalf;
            if (col < kv.dk) *reinterpret_cast<v4f *>(o + col) = live ? sum[g] * inv : v4f{0.f, 0.f, 0.f, 0.f};
        }
        if (at.L && d == 0 && fhalf == 0) at.L[row * at.H + head] = live ? (top + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
    }
    // (each workgroup its own columns of a row, and the first one its sum)
    for (unsigned rest = (unsigned)again; rest; rest &= rest - 1) {
        const int n = __builtin_ctz(rest);
        paged_again<TYPE>(a, place.b, seq, __builtin_amdgcn_readlane(head, n), __builtin_amdgcn_readlane(i, n), lane, 32 * (int)d, 32 * (int)d + 32);
    }
}

template <int DK, int SETS, int TYPE, bool PAD>
int launch_tiles(const PagedArgs &a, PagedTileGrid grid) {
    using G = TileGeom<DK, SETS>;
    static bool attr_set = false;
    if (!attr_set) {
        AXHIP_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(k_paged_tiles<DK, SETS, TYPE, PAD>), hipFuncAttributeMaxDynamicSharedMemorySize, G::SMEM), "hipFuncSetAttribute");
        attr_set = true;
    }
    if (grid.splits > 1) {
        grid.parts = static_cast<float *>(workspace((size_t)grid.slots * a.pages.heads * grid.splits * G::PART * sizeof(float)));
        if (!grid.parts) return AXHIP_ERR_ALLOC;
    }
    note_kernel(grid.splits > 1 ? (SETS == 8 ? "paged_tiles_256_ranges" : "paged_tiles_128_ranges") : SETS == 8 ? "paged_tiles_256" : "paged_tiles_128");
    // as many slots a launch as it holds
    const int64_t at_once = std::max<int64_t>(1, GRID_MOST / ((int64_t)a.pages.heads * grid.splits)), join_at_once = std::max<int64_t>(1, GRID_MOST / ((int64_t)a.pages.heads * SETS * (DK / 32)));
    for (grid.first = 0; grid.first < grid.slots; grid.first += at_once) {
        const int64_t here = std::min(grid.slots - grid.first, at_once);
        hipLaunchKernelGGL((k_paged_tiles<DK, SETS, TYPE, PAD>), dim3((unsigned)(here * a.pages.heads * grid.splits)), dim3(64 * WAVES), G::SMEM, kStream, a, grid);
        if (int rc = check_launch("attn_paged")) return rc;
    }
    if (grid.splits > 1)
        for (grid.first = 0; grid.first < grid.slots; grid.first += join_at_once) {
            const int64_t here = std::min(grid.slots - grid.first, join_at_once);
            hipLaunchKernelGGL((k_paged_join<DK, SETS, TYPE>), dim3((unsigned)(here * a.pages.heads * SETS * (DK / 32))), dim3(256), 0, kStream, a, grid);
            if (int rc = check_launch("attn_paged")) return rc;
        }
    return AXHIP_OK;
}

template <int DK, int SETS>
int launch_tiles(const PagedArgs &a, int type, PagedTileGrid grid) {
    using G = TileGeom<DK, SETS>;
    const int64_t rows = (int64_t)a.attn.G * a.pages.Sq, all_rows = (int64_t)a.attn.G * a.pages.T;
    grid.per = (rows + G::BQ - 1) / G::BQ;
    grid.slots = a.pages.first ? all_rows / G::BQ + a.pages.B : a.pages.B * grid.per;
    // (tiles of equal counts as they are, however those are given: 64 tokens over 8192 int8 keys, 32 heads, 8 of keys, of 128, counted as the two tiles that rows anywhere could touch took 50 us, so 42)
    const bool equal = !a.pages.first || a.pages.B == 1 || a.pages.T == (int64_t)a.pages.B * a.pages.Sq;
    const int64_t likely = (equal ? a.pages.B * grid.per : all_rows / G::BQ + 1) * a.pages.heads, blocks = paged_steps_most(a, G::SHIFT, G::BQ);
    // (each slot has a place for what its ranges leave, also those of sequences that turn out to have few rows: 256 MiB at most)
    const int64_t of_range = grid.slots * a.pages.heads * G::PART * (int64_t)sizeof(float);
    grid.splits = (int)std::max<int64_t>(1, std::min(paged_tile_splits(likely, blocks), (int64_t(256) << 20) / of_range));
    grid.range = (int)std::max<int64_t>((blocks + grid.splits - 1) / grid.splits, 1);
    auto run = [&](auto of) {
        constexpr int TYPE = decltype(of)::value;
        return a.pages.dk < DK ? launch_tiles<DK, SETS, TYPE, true>(a, grid) : launch_tiles<DK, SETS, TYPE, false>(a, grid);
    };
    return type == AXHIP_KV_F16 ? run(std::integral_constant<int, AXHIP_KV_F16>()) : type == AXHIP_KV_I8 ? run(std::integral_constant<int, AXHIP_KV_I8>())
                                                                                                         : run(std::integral_constant<int, AXHIP_KV_MX4>());
}

}  // namespace

namespace axhip {

int64_t paged_tile_splits(int64_t units, int64_t blocks) { return best_splits(units, blocks, blocks / 4, 2, 3); }

int paged_tiles(const PagedArgs &a, int type, int rows_least) {
    PagedTileGrid grid = {};
    grid.least = rows_least;
    const bool wide = (int64_t)a.attn.G * a.pages.Sq > 128;
    auto run = [&](auto width) {
        constexpr int DK = decltype(width)::value;
        return wide ? launch_tiles<DK, 8>(a, type, grid) : launch_tiles<DK, 4>(a, type, grid);
    };
    return a.pages.dk <= 32 ? run(std::integral_constant<int, 32>()) : a.pages.dk <= 64 ? run(std::integral_constant<int, 64>()) : a.pages.dk <= 96 ? run(std::integral_constant<int, 96>())
                                                                                                                                                : run(std::integral_constant<int, 128>());
}

}  // namespace axhip
