// Attention forward under score rules: tiles of queries on the f16 matrix core.
//
// A workgroup of eight waves owns 256 rows of queries, a wave 32 of them, or 128, two waves 32 of them and half of the keys each; the rows are those of one query head, or,
// where a head has few, of all heads that share keys, one after the other.  Keys and values stream through LDS in blocks of 64 (128 of heads up to 64, half the barriers), cut into f16 terms on the
// way (f16x2.h; a query's row once, a probability when it is used).  As in plain attention (sdpa.hip) a lane owns query (l & 31) in the score tile and in the output:
//   S^T tile   A = keys' rows, B = the wave's queries; register v of a lane is key 8 (v >> 2) + 4 (l >> 5) + (v & 3)
//   softmax    online, in log2 units; the reference point moves only when a probability times its value row's factor no longer fits an operand
//   O^T tile   A = V^T, read from the rows by transposing LDS reads, B = the probabilities where the score tile left them
// What a query sees is the keys before `end` that have its document (AttnRow).  Blocks that no row of the workgroup sees are not fetched, 32-key tiles that no row of a
// wave sees not computed, and only tiles that some row sees in part pay for the mask; with documents the ranges of ids of each 32 keys, formed by a first
// launch, decide that.  A row whose sums are not finite (infinities, NaNs or values from 2^78 on that it sees, or that a masked key of a tile holds) is formed again with fp32
// instructions by its wave.
//
// Blocks of heads of 64, 64 keys -> 128 (us): 16 causal heads of [4096, 64] 142 -> 139, 128 of [1000, 64] under a cap 96 -> 93.5, 64 of [2048, 64] with 20 documents 74 -> 71.5, 512 of [512, 64] without a
// mask 145 and 146.
//
// What bounds it: three f16 products for each fp32 one, and vector instructions beside them.  A tile of 32 x 32 scores of heads of 128 is 48 matrix instructions, 1536 cycles
// of a SIMD, and 290 vector ones (a quarter of them cut keys and values), which the two waves of a SIMD overlap in part: the matrix core is busy 53 % of the time, 41 % with
// heads of 64.  64 heads of [1024, 128] without a mask take 107 to 113 us, about 310 TFLOP/s of fp32 products (a large library product in bf16 does a third of
// 1255), 512 heads of [512, 64] 146 us, 235 TFLOP/s; 64 causal heads of [1024, 128] under a cap 92 us.
// Tiles of heads past 96 keep seven registers of a lane in memory.
#include <algorithm>

#include "attn_launch.h"
#include "attn_tiles.h"

namespace {
using namespace axhip;

constexpr int WAVES = 8;

// SETS waves side by side along the queries, 32 each; with four, the others take the other half of each block's keys
template <int DK, int SETS>
struct FwdGeom {
    static constexpr int BQ = 32 * SETS, BKV = DK <= 64 ? 128 : 64, SHARES = WAVES / SETS;
    using B = Block<DK, BKV>;
    static constexpr int FACTORS_AT = 2 * B::BYTES;              // of each key row, then of each value row
    static constexpr int DOCS_AT = FACTORS_AT + BKV * 8;         // documents of the keys, then the ranges of their tiles
    static constexpr int STAGE = (DOCS_AT + BKV * 4 + BKV / 32 * 8 + 255) / 256 * 256;
    static constexpr int META_AT = 2 * STAGE;                    // a row of four ints a wave
    // the other share's sums: a wave's pieces [64] v4f, then maxima and sums [2][32]
    static constexpr int PART = DK / 8 * 1024 + 256;
    static constexpr int SMEM = META_AT + 16 * WAVES;
    static_assert(SMEM <= 160 * 1024 && (SHARES == 1 || SETS * PART <= META_AT), "LDS");
};

template <int DK, int SETS, bool PAD>
__global__ void __launch_bounds__(64 * WAVES, 2) k_attn_fwd(AttnArgs a, FwdGrid grid) {
    using G = FwdGeom<DK, SETS>;
    using B = typename G::B;
    constexpr int KS = DK / 16, DT = DK / 32, BKV = G::BKV, TILES = BKV / 32;
    constexpr bool EARLY = DK <= 96;                // registers for what the scores are scaled by before their products are formed
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, frow = lane & 31, fhalf = lane >> 5;

    // Workgroups go to the eight XCDs in turn.  A unit's tiles (a head's, or a group of heads') go to one: eight units at a time, or, causal, the last and longest tile of every
    // unit first, so that the short ones fill up what the long ones leave.
    const int64_t lin = grid.first + blockIdx.x, group = lin / (8 * (int64_t)grid.tiles), r8 = lin - group * 8 * grid.tiles;
    const int64_t left = grid.units - group * 8, width = left < 8 ? left : 8, unit = a.causal ? lin % grid.units : group * 8 + r8 % width;
    const int tile = a.causal ? grid.tiles - 1 - (int)(lin / grid.units) : (int)(r8 / width);
    const int per_b = a.H / grid.pack, b = (int)(unit / per_b), h0 = (int)(unit - (int64_t)b * per_b) * grid.pack, hk = h0 / a.G;
    const int rows = grid.pack * a.Sq, r = tile * G::BQ + wave % SETS * 32 + frow;
    const bool valid = r < rows;
    const int over = grid.pack == 1 ? 0 : (valid ? r : rows - 1) / a.Sq, head = h0 + over, i = (valid ? r : rows - 1) - over * a.Sq;
    AttnRow row = attn_row(a, b, head, i);
    if (!valid) row.end = 0;
    const bool live = row.end > 0;

    // what the wave sees, and what the workgroup does: the last end, the first end of rows that see anything, the range of documents
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
    const int nblocks = (wg_last + BKV - 1) / BKV;
    const bool docs = a.doc_q != nullptr;

    // the next block from `blk` on that some row may see: 64 at a time, a lane each
    const DocRange *ranges = grid.ranges + (int64_t)b * grid.range_tiles;
    uint64_t window = 0;
    int window_at = -64;
    auto next = [&](int blk) -> int {
        if (!docs) return blk;
        while (blk < nblocks) {
            if (blk - window_at >= 64) {
                window_at = blk & ~63;
                const int mine = window_at + lane;
                bool meets = false;
                if (mine < nblocks) {
#pragma unroll
                    for (int kt = 0; kt < TILES; kt++)
                        if (TILES * mine + kt < grid.range_tiles) meets |= ranges[TILES * mine + kt].meets(wg_low, wg_high);
                }
                window = __builtin_amdgcn_ballot_w64(meets);
            }
            const uint64_t ahead = window >> (blk - window_at);
            if (ahead) return blk + __builtin_ctzll(ahead);
            blk = window_at + 64;
        }
        return nblocks;
    };

    const float *Kb = a.K + (int64_t)b * a.kv_rows * a.ldk + (int64_t)hk * a.dk, *Vb = a.V + (int64_t)b * a.kv_rows * a.ldv + (int64_t)hk * a.dk;
    using S = Stage<DK, BKV, WAVES, PAD>;
    S ks, vs;
    const unsigned base = lds_address(lds);
    int doc_here = -1;
    DocRange range_here = {0, 0};
    auto load = [&](int blk) {
        const int64_t k0 = (int64_t)blk * BKV;
        const int end = wg_last - 1 - (int)k0;       // rows past it are read as it
        const int l = (int)afresh(lane);             // (places of lanes are formed anew: registers are dearer)
        ks.load(Kb + k0 * a.ldk, a.ldk, end, S::place(wave, l, a.ldk), l, a.dk);
        vs.load(Vb + k0 * a.ldv, a.ldv, end, S::place(wave, l, a.ldv), l, a.dk);
        if (docs && threadIdx.x < BKV) doc_here = (int)threadIdx.x <= end ? a.doc_k[(int64_t)b * a.Sk + k0 + threadIdx.x] : -1;
        if (docs && threadIdx.x < TILES) range_here = TILES * blk + (int)threadIdx.x < grid.range_tiles ? ranges[TILES * blk + threadIdx.x] : DocRange{0x7fffffff, -1};
    };
    auto stage = [&](unsigned cur) {
        unsigned char *at = lds + cur;
        const int l = (int)afresh(lane);
        const typename S::Place place = S::place(wave, l, 0);
        ks.put(base + cur, base + cur + G::FACTORS_AT, place, l, 1.0f, a.dk);
        vs.put(base + cur + B::BYTES, base + cur + G::FACTORS_AT + 4 * BKV, place, l, VALUES_UP, a.dk, VALUES_DOWN);
        if (docs && threadIdx.x < BKV) reinterpret_cast<int *>(at + G::DOCS_AT)[threadIdx.x] = doc_here;
        if (docs && threadIdx.x < TILES) reinterpret_cast<DocRange *>(at + G::DOCS_AT + BKV * 4)[threadIdx.x] = range_here;
    };

    int blk = next(0), ahead = nblocks;
    if (blk < nblocks) load(blk);
    v4i qf[KS][2];                                   // step s: columns 16 s + 8 * half .. + 7 of this lane's query
    float q_down;
    {
        const float *q = a.Q + ((int64_t)b * a.Sq + i) * a.ldq + (int64_t)head * a.dk;
        float x[KS][8];
        load_row<PAD, 2>(x, q, live, fhalf, a.dk);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[s][e] *= a.q_up;
        const float most = most_of(x);
        q_down = cut_row(x, fmaxf(most, __shfl_xor(most, 32, 64)), qf);
    }
    if (blk < nblocks) {
        stage(0);
        ahead = next(blk + 1);
        if (ahead < nblocks) load(ahead);
    }
    __syncthreads();

    v16f acc[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) acc[d][v] = 0.0f;
    // Probabilities are 2^(x - ref), l_run this lane half's share of their sum, acc 2^BIAS times that of their products.  The running reference keeps not the probabilities but
    // their products with the factors of the value rows, which go to the matrix core, below ROOM.
    float ref = ATTN_LOWEST, l_run = 0.0f;
    const float one = hidden_one();

    const unsigned row_at = B::row_place(lane) + base, column_at = B::column_place(lane) + base + B::BYTES;
    auto attend = [&](int blk, unsigned cur) {
        const unsigned char *at = lds + cur;
#pragma unroll 1
        for (int kt = wave / SETS; kt < TILES; kt += G::SHARES) {
            const int kt0 = blk * BKV + 32 * kt;
            if (kt0 >= last) break;
            bool partly = kt0 + 32 > sure;
            if (docs) {
                const v2i32 range = *reinterpret_cast<const v2i32 *>(at + G::DOCS_AT + BKV * 4 + 8 * kt);
                const DocRange here = {__builtin_amdgcn_readfirstlane(range[0]), __builtin_amdgcn_readfirstlane(range[1])};
                if (!here.meets(d_low, d_high)) continue;
                partly |= here.low != here.high || here.low != d_low || d_low != d_high;
            }
            const unsigned tile_at = cur + 32 * kt * B::PITCH, row_place = afresh(row_at) + tile_at, column_place = afresh(column_at) + tile_at;
            // ---- scores ----
            auto factors = [&](int what, int g) {    // of keys 8 g + 4 * half + 0..3 of the tile
                return *reinterpret_cast<const v4f *>(at + G::FACTORS_AT + what * BKV * 4 + 4 * (32 * kt + 8 * g + 4 * fhalf));
            };
            v4f ahead_k[4], ahead_v[4];
            if (EARLY)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    ahead_k[g] = factors(0, g);
                    ahead_v[g] = factors(1, g);
                }
            auto of_k = [&](int g) { return EARLY ? ahead_k[g] : factors(0, g); };
            auto of_v = [&](int g) { return EARLY ? ahead_v[g] : factors(1, g); };
            v16f s;
#pragma unroll
            for (int v = 0; v < 16; v++) s[v] = 0.0f;
            __builtin_amdgcn_s_setprio(1);           // matrix phases go ahead of the co-resident wave's vector work
            products<KS>(
                [&](int k, v4i (&f)[2]) {
                    f[1] = B::rows(row_place, k, 1);
                    f[0] = B::rows(row_place, k, 0);
                },
                [&](int k, const v4i (&f)[2]) { s = mfma_cut(f, qf[k], s); });
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4f f = of_k(g);
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * g + e] *= f[e];
            }
            // what is left to the score: q_down, here where more is done to it, in the exponential's multiply-add otherwise
            const bool plain = a.cap == 0.0f && !a.slopes;
            const float down = plain ? q_down : 1.0f;
            if (!plain)
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] *= q_down;
            if (a.cap > 0.0f) {
                float big = 0.0f;
#pragma unroll
                for (int v = 0; v < 16; v++) big = fmaxf(big, __builtin_fabsf(s[v]));
                if (__builtin_amdgcn_ballot_w64(!(big < a.cap_near)))
#pragma unroll
                    for (int v = 0; v < 16; v++) s[v] = capped(a, s[v]).score;
                else
#pragma unroll
                    for (int v = 0; v < 16; v++) s[v] = capped_near(a, s[v]).score;
            }
            if (a.slopes) {
                const float from = (float)(row.p - kt0 - 4 * fhalf);
#pragma unroll
                for (int v = 0; v < 16; v++) s[v] = __builtin_fmaf(-row.slope2, __builtin_fabsf(from - (float)(8 * (v >> 2) + (v & 3))), s[v]);
            }
            if (partly) {
                const int end = row.end - kt0 - 4 * fhalf;
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (8 * (v >> 2) + (v & 3) >= end) s[v] = -INFINITY;
                if (docs) {
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const v4i d = *reinterpret_cast<const v4i *>(at + G::DOCS_AT + 4 * (32 * kt + 8 * g + 4 * fhalf));
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (d[e] != row.doc) s[4 * g + e] = -INFINITY;
                    }
                }
            }
            // ---- online softmax ----
            v16f x;
            float most, l_blk;
            auto weigh = [&]() {
                most = l_blk = 0.0f;
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const v4f f = of_v(g);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int v = 4 * g + e;
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], down, -ref));
                        l_blk += p;
                        x[v] = p * f[e];
                        most = fmaxf(most, x[v]);
                    }
                }
            };
            weigh();
            if (__builtin_amdgcn_ballot_w64(most > ROOM)) {      // (always for the first finite scores)
                most = fmaxf(most, __shfl_xor(most, 32, 64));
                float top = -INFINITY;
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const v4f f = of_v(g);
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, __builtin_fmaf(s[4 * g + e], down, __builtin_amdgcn_logf(f[e])));
                }
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
            cut_scaled(x, 0, one, pf[0]);
            cut_scaled(x, 1, one, pf[1]);
            __builtin_amdgcn_s_setprio(1);
            products<2 * DT>(
                [&](int n, v4i (&f)[2]) {
                    f[1] = B::columns(column_place, 16 * (n / DT), n % DT, 1);
                    f[0] = B::columns(column_place, 16 * (n / DT), n % DT, 0);
                },
                [&](int n, const v4i (&f)[2]) { acc[n % DT] = mfma_cut(f, pf[n / DT], acc[n % DT]); });
            __builtin_amdgcn_s_setprio(0);
        }
    };
    // Two blocks in LDS and the next in registers.  The two waves of a SIMD (w, w + 4) put it beside the current block before and after that is
    // multiplied, so that one cuts while the other's products run.
    unsigned cur = 0;
    while (blk < nblocks) {
        const bool more = ahead < nblocks;
        int after = nblocks;
        auto bring = [&]() {
            stage(cur ^ G::STAGE);
            after = next(ahead + 1);
            if (after < nblocks) load(after);
        };
        if (more && wave >= 4) bring();
        attend(blk, cur);
        if (more && wave < 4) bring();
        __syncthreads();
        blk = ahead;
        ahead = after;
        cur ^= G::STAGE;
    }

    float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    if constexpr (G::SHARES == 2) {                  // the other share's keys (the last barrier has passed: no block is read any more)
        unsigned char *part = lds + wave % SETS * G::PART;
        v4f *sums = reinterpret_cast<v4f *>(part) + lane;
        float *of_row = reinterpret_cast<float *>(part + G::PART - 256) + frow;
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
        const float other = of_row[0], both = fmaxf(ref, other), mine = __builtin_amdgcn_exp2f(ref - both), theirs = __builtin_amdgcn_exp2f(other - both);
        l_tot = scaled(l_tot, ref - both) + scaled(of_row[32], other - both);
        ref = both;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4f sum = sums[64 * (4 * d + g)];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[d][4 * g + e] = __builtin_fmaf(acc[d][4 * g + e], mine, sum[e] * theirs);
            }
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
    const bool fit = !((again >> frow) & 1);
    const float inv = 1.0f / l_tot;
    if (valid && fit) {
        float *o = a.O + ((int64_t)b * a.Sq + i) * a.ldo + (int64_t)head * a.dk;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int col = 32 * d + 8 * g + 4 * fhalf;
                v4f out;
#pragma unroll
                for (int e = 0; e < 4; e++) out[e] = live ? acc[d][4 * g + e] * two_to(-BIAS) * inv : 0.0f;
                if (!PAD || col < a.dk) *reinterpret_cast<v4f *>(o + col) = out;
            }
        if (a.L && fhalf == 0) a.L[((int64_t)b * a.H + head) * a.Sq + i] = live ? (ref + __builtin_amdgcn_logf(l_tot)) * LN2 : -INFINITY;
    }
    for (unsigned rest = (unsigned)again; rest; rest &= rest - 1) {
        const int n = __builtin_ctz(rest);
        attn_fwd_row(a, b, __builtin_amdgcn_readlane(head, n), __builtin_amdgcn_readlane(i, n), (int)afresh(lane));
    }
}

// The ranges of documents of each 32 ids, a wave each
__global__ void __launch_bounds__(256) k_doc_ranges(const int32_t *ids, int64_t sequences, int S, int tiles, DocRange *out) {
    const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= sequences * tiles) return;
    const int64_t b = n / tiles;
    const int at = (int)(n - b * tiles) * 32 + (threadIdx.x & 31);
    const int id = at < S ? ids[b * S + at] : -1;
    int low = id < 0 ? 0x7fffffff : id, high = id;
    bool none = id < 0 && at < S;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        low = min(low, __shfl_xor(low, off, 32));
        high = max(high, __shfl_xor(high, off, 32));
        none |= __shfl_xor((int)none, off, 32) != 0;
    }
    if ((threadIdx.x & 31) == 0) out[n] = high < 0 ? DocRange{0x7fffffff, -1} : DocRange{none ? ~low : low, high};
}

template <int DK, int SETS, bool PAD>
int launch_fwd(const AttnArgs &a, FwdGrid grid) {
    using G = FwdGeom<DK, SETS>;
    static bool attr_set = false;
    if (!attr_set) {
        AXHIP_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(k_attn_fwd<DK, SETS, PAD>), hipFuncAttributeMaxDynamicSharedMemorySize, G::SMEM), "hipFuncSetAttribute");
        attr_set = true;
    }
    grid.tiles = (int)(((int64_t)grid.pack * a.Sq + G::BQ - 1) / G::BQ);
    const int64_t all = grid.units * grid.tiles;
    note_kernel(SETS == 8 ? "attn_tiles_256" : "attn_tiles_128");
    for (grid.first = 0; grid.first < all; grid.first += GRID_MOST) {
        const int64_t left = all - grid.first;
        hipLaunchKernelGGL((k_attn_fwd<DK, SETS, PAD>), dim3((unsigned)(left < GRID_MOST ? left : GRID_MOST)), dim3(64 * WAVES), G::SMEM, kStream, a, grid);
        if (int rc = check_launch("attn_fwd")) return rc;
    }
    return AXHIP_OK;
}

template <int DK>
int launch_fwd(const AttnArgs &a, const FwdGrid &grid, bool wide) {
    if (a.dk < DK) return wide ? launch_fwd<DK, 8, true>(a, grid) : launch_fwd<DK, 4, true>(a, grid);
    return wide ? launch_fwd<DK, 8, false>(a, grid) : launch_fwd<DK, 4, false>(a, grid);
}

}  // namespace

namespace axhip {

int doc_ranges(const int32_t *ids, int64_t B, int64_t S, void *out) {
    const int64_t tiles = (S + 31) / 32, n = B * tiles;
    if (n == 0) return AXHIP_OK;
    if ((n + 7) / 8 > GRID_MOST) return fail(AXHIP_ERR_SHAPE, "attention: too many documents");
    hipLaunchKernelGGL(k_doc_ranges, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, kStream, ids, B, (int)S, (int)tiles, static_cast<DocRange *>(out));
    return check_launch("document ranges");
}

int attn_fwd_tiles(const AttnArgs &a) {
    FwdGrid grid = {};
    // rows of all heads that share keys in one tile, where a head's own would leave most of it empty
    grid.pack = a.G > 1 && a.Sq <= 64 ? a.G : 1;
    grid.units = (int64_t)a.B * (a.H / grid.pack);
    if (a.doc_k) {
        grid.range_tiles = (int)(((int64_t)a.Sk + 31) / 32);
        void *ranges = workspace((size_t)a.B * grid.range_tiles * sizeof(DocRange));
        if (!ranges) return AXHIP_ERR_ALLOC;
        if (int rc = doc_ranges(a.doc_k, a.B, a.Sk, ranges)) return rc;
        grid.ranges = static_cast<DocRange *>(ranges);
    }
    // Tiles of 256 or 128 rows: the wide ones, which cut keys and values half as often, take one and a half times as long and not twice, but there are half as many to share out.
    // Rounds of tiles over the CUs, or, causal, the longest tile or all of them evenly, whichever is more (us, 128 -> 256: 64 heads of [1024, 128] 142 -> 115, causal 84 and 88, 32
    // causal ones of [3000, 96] 236 -> 206, but 36 causal ones of [777, 80] 42 -> 57).
    const int64_t rows = (int64_t)grid.pack * a.Sq, wide_tiles = (rows + 255) / 256, tiles = (rows + 127) / 128, cus = cu_count();
    int64_t wide_time, time;
    if (a.causal) {
        wide_time = std::max(6 * cus, 3 * grid.units * (wide_tiles + 1));
        time = std::max(4 * cus, 2 * grid.units * (tiles + 1));
    } else {
        wide_time = 3 * ((grid.units * wide_tiles + cus - 1) / cus);
        time = 2 * ((grid.units * tiles + cus - 1) / cus);
    }
    const bool wide = wide_time <= time;
    if (a.dk <= 32) return launch_fwd<32>(a, grid, wide);
    if (a.dk <= 64) return launch_fwd<64>(a, grid, wide);
    if (a.dk <= 96) return launch_fwd<96>(a, grid, wide);
    return launch_fwd<128>(a, grid, wide);
}

}  // namespace axhip
