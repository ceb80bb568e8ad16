// Attention over a paged cache: tiles of queries on the f16 matrix core.
//
// A workgroup of eight waves owns 256 rows of queries (the new tokens of a sequence for all query heads that share keys, token by token), a wave 32 of them, or 128, two waves 32 of them and
// half of the keys each.  Keys and values come from their pages in blocks of 64 (128 of heads up to 64) and stand in LDS as f16, twice, so that the numbers of the cache are converted once for
// all rows; they are f16 exactly, so a product of fp32 is two of f16 terms, the query's or the probability's (f16x2.h).  The tiles of scores and outputs, the online softmax and its
// running reference are those of attn_fwd.hip.
// What rows see goes up with their positions: blocks before the window of a workgroup's first row, but for the first tokens that stay visible, and behind its last row's position are not
// fetched, 32-key tiles that no row of a wave sees not computed, and only tiles that some row sees in part pay for the mask.
// Where tiles would leave CUs idle, ranges of their keys go to workgroups of their own, and a second launch adds what they leave, in order.
#include "attn_launch.h"
#include "attn_tiles.h"
#include "paged.h"

namespace {
using namespace axhip;

constexpr int WAVES = 8, SPLITS_MOST = 64;

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

// Where a workgroup's rows are
struct Place {
    int b;
    int64_t tile, rows;                          // rows: of the sequence, for all heads that share keys; 0: none of this form's
};
template <int BQ>
__device__ __forceinline__ Place place_of(const PagedArgs &a, const PagedTileGrid &grid, int64_t slot, int lane, KvSeq &seq) {
    const KvPages &kv = a.pages;
    const int64_t G = a.attn.G;
    Place p = {0, 0, 0};
    if (kv.first) {
        // sequence b's slots are those from first[b] G / BQ + b on
        p.b = kv_find(kv, lane, [&](int k, int first) { return first * G / BQ + k <= slot; });
        if (p.b >= kv.B) return p;
        p.tile = slot - (min(max(kv.first[p.b], 0), kv.T) * G / BQ + p.b);
    } else {
        const int64_t per = (kv.Sq * G + BQ - 1) / BQ;
        p.b = (int)(slot / per);
        p.tile = slot - p.b * per;
    }
    seq = kv_seq(kv, p.b);
    const int64_t rows = G * seq.n;
    if (rows >= grid.least && p.tile >= 0 && p.tile * BQ < rows) p.rows = rows;
    return p;
}

template <int DK, int SETS, int TYPE, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, 2) k_paged_tiles(PagedArgs a, PagedTileGrid grid) {
    using G = TileGeom<DK, SETS>;
    using B = typename G::B;
    using T = KvType<TYPE>;
    constexpr int KS = DK / 16, DT = DK / 32, BKV = G::BKV, TILES = BKV / 32, BQ = G::BQ;
    constexpr int COLS = 128 / T::BITS, LANES = (DK == 96 ? 128 : DK) / COLS, PASSES = 2 * BKV * LANES > 64 * WAVES ? 2 * BKV * LANES / (64 * WAVES) : 1;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const KvPages &kv = a.pages;
    const AttnArgs &at = a.attn;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 31, fhalf = lane >> 5;

    // a sequence's last tiles, the longest, first; heads of keys go to the XCDs in turn
    const int64_t lin = grid.first + blockIdx.x, rest = lin / kv.heads, slot = grid.slots - 1 - rest / grid.splits;
    const int hk = (int)(lin - rest * kv.heads), split = (int)(rest % grid.splits);
    KvSeq seq = {0, 0, 0};
    const Place place = place_of<BQ>(a, grid, slot, lane, seq);
    if (place.rows == 0) return;
    const int b = place.b;
    const int64_t r0 = place.tile * BQ;
    const int rows_here = (int)min(place.rows - r0, (int64_t)BQ), mine = wave % SETS * 32 + frow;
    const bool valid = mine < rows_here;
    const int64_t r = r0 + (valid ? mine : rows_here - 1);
    const int i = (int)(r / at.G), head = hk * at.G + (int)(r - (int64_t)i * at.G);
    PagedRow row = paged_row(a, seq, i);
    if (!valid) row.end = 0;
    const bool live = row.end > 0;
    // what the workgroup's rows see together, and the wave's
    const PagedRow wg_low = paged_row(a, seq, (int)(r0 / at.G)), wg_high = paged_row(a, seq, (int)((r0 + rows_here - 1) / at.G));
    const int w0 = min(wave % SETS * 32, rows_here - 1), w1 = min(wave % SETS * 32 + 31, rows_here - 1);
    const PagedRow low = paged_row(a, seq, (int)((r0 + w0) / at.G)), high = paged_row(a, seq, (int)((r0 + w1) / at.G));
    const int last = wave % SETS * 32 < rows_here ? high.end : 0;
    const PagedTiles blocks = paged_tiles_of(a, wg_low.begin, wg_high.end, G::SHIFT);
    const int n_begin = (int)((int64_t)blocks.all * split / grid.splits), n_end = (int)((int64_t)blocks.all * (split + 1) / grid.splits);
    const float slope2 = at.slopes ? at.slopes[head] * at.bias2 : 0.0f;

    const unsigned base = lds_address(lds);
    // A pass brings 16 bytes a thread: LANES threads a row, rows of keys and then of values.
    constexpr int PLACES = PASSES > 1 ? PASSES / 2 : 1;          // with two passes or more, the second half brings the values of the first half's keys
    v4i x[PASSES];
    unsigned scales[PASSES];
    int entry[PLACES];
    unsigned gone = 0;                               // a bit a place: its key has no page
    auto row_of = [&](int pass) { return (pass * 64 * WAVES + (int)threadIdx.x) / LANES; };      // from BKV on a value's; from 2 BKV on none
    auto pos_of = [&](int n, int place) { return blocks.tile(n) * BKV + row_of(place) % BKV; };
    auto look = [&](int n) {
#pragma unroll
        for (int p = 0; p < PLACES; p++) entry[p] = kv_entry(kv, b, min(pos_of(n, p), wg_high.end - 1));
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
            if (pos < wg_high.end && kv_is_page(kv, entry[p]) && (2 * BKV * LANES >= 64 * WAVES || row_of(p) < 2 * BKV)) {
                const uint64_t at_row = kv_row_at(kv, entry[p], hk, pos) + 16 * c, at_scale = kv_scale_at(kv, entry[p], hk, pos);
                const bool some = (!PAD && DK != 96) || 16 * c < kv.row_bytes;
                if (PASSES > 1) {
                    if (some) {
                        x[p] = *reinterpret_cast<const v4i *>(kv.k + at_row);
                        x[(p + PLACES) % PASSES] = *reinterpret_cast<const v4i *>(kv.v + at_row);
                    }
                    scales[p] = *reinterpret_cast<const unsigned *>(kv.k_scale + at_scale);
                    scales[(p + PLACES) % PASSES] = *reinterpret_cast<const unsigned *>(kv.v_scale + at_scale);
                } else {
                    const bool of_v = row_of(p) >= BKV;
                    if (some) x[p] = *reinterpret_cast<const v4i *>((of_v ? kv.v : kv.k) + at_row);
                    scales[p] = *reinterpret_cast<const unsigned *>((of_v ? kv.v_scale : kv.k_scale) + at_scale);
                }
            } else {
                gone |= 1u << p;
            }
        }
    };
    auto stage = [&](unsigned cur) {
#pragma unroll
        for (int p = 0; p < PASSES; p++) {
            const int at_row = row_of(p), c = (int)threadIdx.x % LANES, in_block = at_row % BKV;
            if (2 * BKV * LANES >= 64 * WAVES || at_row < 2 * BKV) {
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
            products<KS>([&](int k, v4i (&f)[2]) { f[0] = B::rows(row_place, k, 0); },
                         [&](int k, const v4i (&f)[2]) {
                             s = mfma_halves(f[0], qf[k][1], s);
                             s = mfma_halves(f[0], qf[k][0], s);
                         });
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * g + e] *= kf[g][e];
            // what is left to the score: q_down, here where more is done to it, in the exponential's multiply-add otherwise
            const bool plain = at.cap == 0.0f && !at.slopes;
            const float down = plain ? q_down : 1.0f;
            if (!plain)
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] *= q_down;
            if (at.cap > 0.0f) {
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
            if (at.slopes) {
                const float from = (float)(row.p - kt0 - 4 * fhalf);
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] = __builtin_fmaf(-slope2, from - (float)(8 * (v >> 2) + (v & 3)), s[v]);
            }
            if (partly) {
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
            if (__builtin_amdgcn_ballot_w64(most > ROOM)) {      // (always for the first finite scores)
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
    if (grid.splits > 1) {
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

// What ranges of keys left, added in order: a workgroup for 32 rows, a wave for 32 columns
template <int DK, int SETS, int TYPE>
__global__ void __launch_bounds__(2 * DK) k_paged_join(PagedArgs a, PagedTileGrid grid) {
    using G = TileGeom<DK, SETS>;
    constexpr int BQ = G::BQ, DT = DK / 32;
    __shared__ unsigned flags[DT];
    const KvPages &kv = a.pages;
    const AttnArgs &at = a.attn;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 31, fhalf = lane >> 5;
    const int64_t lin = grid.first + blockIdx.x, unit = lin / SETS, slot = unit / kv.heads;
    const int set = (int)(lin - unit * SETS), hk = (int)(unit - slot * kv.heads);
    KvSeq seq = {0, 0, 0};
    const Place place = place_of<BQ>(a, grid, slot, lane, seq);
    const int64_t r0 = place.tile * BQ + 32 * set;
    if (place.rows == 0 || r0 >= place.rows) return;
    const int rows_here = (int)min(place.rows - r0, (int64_t)32);
    const bool valid = frow < rows_here;
    const int64_t r = r0 + (valid ? frow : rows_here - 1);
    const int i = (int)(r / at.G), head = hk * at.G + (int)(r - (int64_t)i * at.G);
    const bool live = valid && paged_row(a, seq, i).end > 0;
    const float *parts = grid.parts + unit * grid.splits * G::PART + set * (G::PART / SETS);
    float m = ATTN_LOWEST, l = 0.0f;
    for (int s = 0; s < grid.splits; s++) m = fmaxf(m, parts[(int64_t)s * G::PART + G::PIECES * 256 + frow]);
    v4f sum[4];
#pragma unroll
    for (int g = 0; g < 4; g++) sum[g] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < grid.splits; s++) {
        const float *part = parts + (int64_t)s * G::PART;
        const float ref = part[G::PIECES * 256 + frow], weight = __builtin_amdgcn_exp2f(ref - m);
        l += scaled(part[G::PIECES * 256 + 32 + frow], ref - m);
#pragma unroll
        for (int g = 0; g < 4; g++) sum[g] += *reinterpret_cast<const v4f *>(part + ((4 * wave + g) * 64 + lane) * 4) * weight;
    }
    float seen = l * 0.0f;
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) seen = __builtin_fmaf(sum[g][e], 0.0f, seen);
    const uint64_t unfit = __builtin_amdgcn_ballot_w64(live && (!(seen == 0.0f) || l == 0.0f));
    if (lane == 0) flags[wave] = (unsigned)(unfit | unfit >> 32);
    __syncthreads();
    unsigned again = 0;
#pragma unroll
    for (int w = 0; w < DT; w++) again |= flags[w];
    again = __builtin_amdgcn_readfirstlane(again);
    if (valid && !((again >> frow) & 1)) {
        const int64_t to = (int64_t)seq.first + i;
        float *o = at.O + to * at.ldo + (int64_t)head * kv.dk;
        const float inv = 1.0f / l;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int col = 32 * wave + 8 * g + 4 * fhalf;
            if (col < kv.dk) *reinterpret_cast<v4f *>(o + col) = live ? sum[g] * inv : v4f{0.f, 0.f, 0.f, 0.f};
        }
        if (at.L && wave == 0 && fhalf == 0) at.L[to * at.H + head] = live ? (m + __builtin_amdgcn_logf(l)) * LN2 : -INFINITY;
    }
    int nth = 0;
    for (unsigned rest = again; rest; rest &= rest - 1, nth++) {
        const int n = __builtin_ctz(rest);
        if (nth % DT == wave) paged_again<TYPE>(a, place.b, seq, __builtin_amdgcn_readlane(head, n), __builtin_amdgcn_readlane(i, n), lane);
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
    const int64_t units = grid.slots * a.pages.heads, all = units * grid.splits;
    if (grid.splits > 1) {
        grid.parts = static_cast<float *>(workspace((size_t)all * G::PART * sizeof(float)));
        if (!grid.parts) return AXHIP_ERR_ALLOC;
    }
    note_kernel(grid.splits > 1 ? (SETS == 8 ? "paged_tiles_256_ranges" : "paged_tiles_128_ranges") : SETS == 8 ? "paged_tiles_256" : "paged_tiles_128");
    for (grid.first = 0; grid.first < all; grid.first += GRID_MOST) {
        const int64_t left = all - grid.first;
        hipLaunchKernelGGL((k_paged_tiles<DK, SETS, TYPE, PAD>), dim3((unsigned)(left < GRID_MOST ? left : GRID_MOST)), dim3(64 * WAVES), G::SMEM, kStream, a, grid);
        if (int rc = check_launch("attn_paged")) return rc;
    }
    if (grid.splits > 1)                             // (few tiles: a launch holds them)
        for (grid.first = 0; grid.first < units * SETS; grid.first += GRID_MOST) {
            const int64_t left = units * SETS - grid.first;
            hipLaunchKernelGGL((k_paged_join<DK, SETS, TYPE>), dim3((unsigned)(left < GRID_MOST ? left : GRID_MOST)), dim3(2 * DK), 0, kStream, a, grid);
            if (int rc = check_launch("attn_paged")) return rc;
        }
    return AXHIP_OK;
}

template <int DK, int SETS>
int launch_tiles(const PagedArgs &a, int type, PagedTileGrid grid, int64_t keys) {
    using G = TileGeom<DK, SETS>;
    const int64_t rows = (int64_t)a.attn.G * a.pages.Sq, all_rows = (int64_t)a.attn.G * a.pages.T, cus = cu_count();
    grid.slots = a.pages.first ? all_rows / G::BQ + a.pages.B : a.pages.B * ((rows + G::BQ - 1) / G::BQ);
    const int64_t likely = (a.pages.first ? all_rows / G::BQ + 1 : grid.slots) * a.pages.heads, blocks = (keys + G::BKV - 1) / G::BKV;
    int64_t splits = cus / likely;
    if (splits > blocks / 4) splits = blocks / 4;
    if (splits > SPLITS_MOST) splits = SPLITS_MOST;
    if (splits < 1) splits = 1;
    grid.splits = (int)splits;
    auto run = [&](auto of) {
        constexpr int TYPE = decltype(of)::value;
        return a.pages.dk < DK ? launch_tiles<DK, SETS, TYPE, true>(a, grid) : launch_tiles<DK, SETS, TYPE, false>(a, grid);
    };
    return type == AXHIP_KV_F16 ? run(std::integral_constant<int, AXHIP_KV_F16>()) : type == AXHIP_KV_I8 ? run(std::integral_constant<int, AXHIP_KV_I8>())
                                                                                                         : run(std::integral_constant<int, AXHIP_KV_MX4>());
}

}  // namespace

namespace axhip {

int paged_tiles(const PagedArgs &a, int type, int rows_least, int64_t keys) {
    PagedTileGrid grid = {};
    grid.least = rows_least;
    const int64_t wide_tiles = ((int64_t)a.attn.G * a.pages.T + 255) / 256 * a.pages.heads;
    const bool wide = wide_tiles >= cu_count();
    auto run = [&](auto width) {
        constexpr int DK = decltype(width)::value;
        return wide ? launch_tiles<DK, 8>(a, type, grid, keys) : launch_tiles<DK, 4>(a, type, grid, keys);
    };
    return a.pages.dk <= 32 ? run(std::integral_constant<int, 32>()) : a.pages.dk <= 64 ? run(std::integral_constant<int, 64>()) : a.pages.dk <= 96 ? run(std::integral_constant<int, 96>())
                                                                                                                                                : run(std::integral_constant<int, 128>());
}

}  // namespace axhip
