// What the kernels of attention over a paged cache share (axhip_attn_paged): their arguments, what a query sees, and rows formed one at a time with fp32 instructions.
#pragma once
#include "attn_rules.h"
#include "f16x2.h"
#include "kv_pages.h"

namespace axhip {

struct PagedArgs {
    AttnArgs attn;                               // of which the cap, slopes and scale count, and Q, O, L, their pitches, H and G
    KvPages pages;
    int window, sinks;                           // window 0: none
};

struct PagedFewGrid {
    int first, here;                             // the launch's first sequence, and how many
    int row_tiles, splits;                       // of 16 rows each; ranges of keys
    int most;                                    // sequences with more rows (of all heads that share keys) are the tiles'
    float *parts;                                // what the ranges leave
    int *arrivals;
};

struct PagedTileGrid {
    int64_t first, slots, per;                   // the launch's first slot; slots: places for tiles, of which each sequence has as many as its rows could need (`per`, where they are equal)
    int splits, range;                           // the most ranges of keys that a tile has, one for every `range` blocks
    int least;                                   // sequences with fewer rows are the few-rows form's
    float *parts;
};

int paged_few(const PagedArgs &a, int type, int rows_most);
int paged_tiles(const PagedArgs &a, int type, int rows_least);

// What the cache holds, per type: bits of a number, and what the matrix core gets.  A row's numbers go in as f16 exactly, n or (MX4) n 2^12 under the largest scale of its groups; its
// factor brings them back.  Numbers reach 2^TOP; where they are summed over (P V) their factors carry 2^BIAS beyond, and are infinite for values of 2^78 and more (VALUES_UP, f16x2.h).
template <int TYPE>
struct KvType {
    static constexpr int BITS = TYPE == AXHIP_KV_F16 ? 16 : TYPE == AXHIP_KV_I8 ? 8 : 4, TOP = TYPE == AXHIP_KV_I8 ? 7 : 15;
    static constexpr float VALUE_UP = TYPE == AXHIP_KV_I8 ? VALUES_UP * 0x1p-7f : VALUES_UP;
    static constexpr int VALUE_BIAS = TYPE == AXHIP_KV_I8 ? BIAS - 7 : BIAS;
};
constexpr int MX4_UP = 12;

// The largest of a row's group codes that counts, and its factor.  (Rows below 2^KV_LEAST lose bits as those of the other types do; a NaN anywhere is one of the row, whose
// queries are then formed again.)
__device__ __forceinline__ int mx4_top(unsigned scales) {
    const unsigned a = max(scales & 255, (scales >> 8) & 255), b = max((scales >> 16) & 255, scales >> 24);
    return (int)max(max(a, b), (unsigned)(127 + KV_LEAST));
}
template <int TYPE>
__device__ __forceinline__ float kv_factor(unsigned scales) {
    if (TYPE != AXHIP_KV_MX4) return __uint_as_float(scales);
    const int top = mx4_top(scales);
    return top == 255 ? NAN : __uint_as_float((unsigned)(top - MX4_UP) << 23);
}
// What a group's numbers are taken times: 2^MX4_UP for those of the largest scale, next to nothing from 2^-40 of it on
__device__ __forceinline__ float mx4_up(unsigned scales, int top, int group) {
    const int code = (int)((scales >> (8 * group)) & 255);
    return __uint_as_float((unsigned)(max(code - top, -40) + MX4_UP + 127) << 23);
}

// A query's position and the keys that it sees: those from `begin` to `end`, and those before `sinks`, that have a page.  end = 0: none.
struct PagedRow {
    int p, begin, end;
};
__device__ __forceinline__ PagedRow paged_row(const PagedArgs &a, const KvSeq &s, int i) {
    PagedRow r;
    r.p = s.len - s.n + i;
    r.end = max(r.p + 1, 0);
    r.begin = a.window > 0 ? max(r.p + 1 - a.window, 0) : 0;
    return r;
}

// The 32-key tiles that rows see together: `ahead` of them from the first on, for the sinks, then those from `from` on; `all` in all.
struct PagedTiles {
    int ahead, from, all;
    __device__ int tile(int n) const { return n < ahead ? n : n - ahead + from; }
};
// of rows whose first begins at `begin` and whose last ends at `end`; in steps of 2^shift keys
__device__ __forceinline__ PagedTiles paged_tiles_of(const PagedArgs &a, int begin, int end, int shift) {
    PagedTiles t;
    const int step = (1 << shift) - 1, last = (end + step) >> shift;
    t.from = min(begin >> shift, last);
    t.ahead = a.window > 0 ? min((int)(((int64_t)a.sinks + step) >> shift), t.from) : 0;
    t.all = t.ahead + last - t.from;
    return t;
}

// The most steps of 2^shift keys that `rows` rows of one sequence, one token after the other, see together (above: from begin = p + 1 - window to the end of a later row)
inline int64_t paged_steps_most(const PagedArgs &a, int shift, int64_t rows) {
    const int64_t step = int64_t(1) << shift, all = (a.pages.room + step - 1) / step, tokens = rows / a.attn.G + 2 < a.pages.Sq ? rows / a.attn.G + 2 : a.pages.Sq;
    if (a.window == 0) return all;
    const int64_t most = (a.window + tokens - 1 + 2 * (step - 1)) / step + ((int64_t)a.sinks + step - 1) / step;
    return most < all ? most : all;
}

// In how many ranges the keys of `units` groups of rows are shared out, a workgroup each: of 1 to `most` (a wave with two tiles of keys or more for few rows, a workgroup with four blocks for tiles) those
// that take the fewest rounds over the CUs times their steps, `start` more for each round and `join` for the ranges' sums.
constexpr int PAGED_SPLITS = 64;
inline int64_t best_splits(int64_t units, int64_t steps, int64_t most, int64_t start, int64_t join) {
    const int64_t cus = cu_count();
    int64_t best = 1, least = INT64_MAX;
    if (units >= 2 * cus) return 1;                  // (groups of unlike length fill up the rounds)
    for (int64_t s = 1; s == 1 || (s <= most && s <= PAGED_SPLITS && units * s <= 8 * cus); s++) {
        const int64_t cost = (units * s + cus - 1) / cus * ((steps + s - 1) / s + start) + (s > 1 ? join : 0);
        if (cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}
int64_t paged_few_splits(int64_t units, int64_t tiles);
int64_t paged_tile_splits(int64_t units, int64_t blocks);

// ---- one row by one wave with fp32 instructions: what the matrix kernels fall back to where sums are not finite.  64 keys at a time, a score a lane; then a value column a lane (two
// where dk > 64), and only keys that are seen are touched. ----
template <int TYPE>
__device__ __forceinline__ void paged_again(const PagedArgs &a, int b, const KvSeq &s, int head, int i, int lane, int c0 = 0, int c1 = 128) {
    const KvPages &kv = a.pages;
    const PagedRow r = paged_row(a, s, i);
    const int hk = head / a.attn.G, dk = kv.dk;
    const int64_t at = (int64_t)s.first + i;
    const float *q = a.attn.Q + at * a.attn.ldq + (int64_t)head * dk;
    const float slope2 = a.attn.slopes ? a.attn.slopes[head] * a.attn.bias2 : 0.0f;
    // Sums of values near the largest float may pass it where their mean does not: such columns are formed once more, with 2^-25 of each weight, since there are up to 2^24 keys.
    float m, l, o0, o1, once0, once1, down = 1.0f;
    bool any;
#pragma unroll 1
    for (;;) {
        m = ATTN_LOWEST;
        l = o0 = o1 = 0.0f;
        any = false;
        for (int k0 = 0; k0 < r.end; k0 += 64) {
            if (k0 + 64 <= r.begin && k0 >= a.sinks) {   // nothing before the window's first 64
                k0 = (r.begin & ~63) - 64;
                continue;
            }
            const int key = k0 + lane;
            bool sees = key < r.end && (key >= r.begin || key < a.sinks);
            int page = 0;
            if (sees) {
                page = kv_page(kv, b, key);
                sees = page >= 0;
            }
            float x = -INFINITY;
            if (sees) {
                const unsigned scale = *reinterpret_cast<const unsigned *>(kv.k_scale + kv_scale_at(kv, page, hk, key));
                const unsigned char *row = kv.k + kv_row_at(kv, page, hk, key);
                float sum = 0.0f;
                for (int c = 0; 8 * c < dk; c++) {
                    float k[8];
                    kv_eight<TYPE>(row, scale, c, k);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (8 * c + e < dk) sum = __builtin_fmaf(q[8 * c + e] * a.attn.q_up, k[e], sum);
                }
                if (a.attn.cap > 0.0f) sum = capped(a.attn, sum).score;
                x = a.attn.slopes ? __builtin_fmaf(-slope2, (float)(r.p - key), sum) : sum;
            }
            uint64_t seen = __builtin_amdgcn_ballot_w64(sees);
            if (!seen) continue;
            any = true;
            const float m_new = fmaxf(m, wave_max(x)), alpha = __builtin_amdgcn_exp2f(m - m_new);
            const float p = sees ? __builtin_amdgcn_exp2f(x - m_new) : 0.0f;
            m = m_new;
            l = l * alpha + wave_sum(p);
            o0 *= alpha;
            o1 *= alpha;
            for (; seen; seen &= seen - 1) {
                const int j = __builtin_ctzll(seen);
                const float pj = from_lane(p, j) * down;
                const int of_j = __builtin_amdgcn_readlane(page, j);
                const unsigned scale = *reinterpret_cast<const unsigned *>(kv.v_scale + kv_scale_at(kv, of_j, hk, k0 + j));
                const unsigned char *row = kv.v + kv_row_at(kv, of_j, hk, k0 + j);
                float v[8];
                if (lane < dk) {
                    kv_eight<TYPE>(row, scale, lane >> 3, v);
                    float mine = v[0];
#pragma unroll
                    for (int e = 1; e < 8; e++) mine = (lane & 7) == e ? v[e] : mine;
                    o0 = __builtin_fmaf(pj, mine, o0);
                }
                if (lane + 64 < dk) {
                    kv_eight<TYPE>(row, scale, 8 + (lane >> 3), v);
                    float mine = v[0];
#pragma unroll
                    for (int e = 1; e < 8; e++) mine = (lane & 7) == e ? v[e] : mine;
                    o1 = __builtin_fmaf(pj, mine, o1);
                }
            }
        }
        if (down < 1.0f) break;
        once0 = o0;
        once1 = o1;
        if (!(l > 0.0f) || !__builtin_amdgcn_ballot_w64(!(__builtin_fabsf(o0) < INFINITY && __builtin_fabsf(o1) < INFINITY))) break;
        down = 0x1p-25f;
    }
    const float inv = any ? 1.0f / l : 0.0f;
    auto mean = [&](float once, float again) { return __builtin_fabsf(once) < INFINITY ? once * inv : again * inv * 0x1p25f; };
    float *o = a.attn.O + at * a.attn.ldo + (int64_t)head * dk;
    if (lane < dk && lane >= c0 && lane < c1) o[lane] = any ? mean(once0, o0) : 0.0f;
    if (lane + 64 < dk && lane + 64 >= c0 && lane + 64 < c1) o[lane + 64] = any ? mean(once1, o1) : 0.0f;
    // (a row that saw nothing but scores of -infinity: 0 / 0 above, and NaN here)
    if (a.attn.L && lane == 0 && c0 == 0) a.attn.L[at * a.attn.H + head] = !any ? -INFINITY : l == 0.0f ? NAN : (m + __builtin_amdgcn_logf(l)) * LN2;
}

}  // namespace axhip
