// Attention of new tokens over a paged cache of keys and values in few bits (axhip_attn_paged): checks, and who takes the call.
#include <math.h>

#include "attn_launch.h"
#include "paged.h"

namespace {
using namespace axhip;

// Which form takes rows of equal counts, by what each takes, in us: rounds of workgroups over the CUs, each its start and its steps of keys, and for tiles in ranges the launch that joins them.
// (16-row units of 8 waves that take 32 keys each; tiles of 256 rows, or 128, in blocks.)  Within a tenth or so of what was measured (us, tiles -> few rows: 1 x 128 tokens over 128 keys, 32 heads, 8
// of keys, of 128 19.6 -> 7.8, 1 x 512 over 512, 8 heads 31 -> 15.5, 4 x 64 over 500, 32 heads, 8 of keys 33 -> 25; the other side 64 x 32 over 100, 32 heads, 8 of keys 38 -> 58, 16 x 64 over 64, 16 heads, 4
// of keys, of 64 14.3 -> 20.7).  Up to 64 rows of a sequence few rows won throughout (8 x 8 tokens over 4096, 64 heads, 8 of keys 49 -> 44, 1 x 8 24 -> 17).
// Beside sequences of many rows those of more than 32 are the tiles': few rows run before the tiles and not beside them, so what they take is added, while tiles that few rows fill in part run in rounds that others fill.
// (us, of 32 -> of 64: 600 tokens and 16 sequences of 8 over up to 4096, 32 heads, 4 of keys, of 128, 64 rows each, int8 159 -> 174, f16 163 -> 203, 4 bits 162 -> 167; of 5, 64 heads, 8 of keys, f16 305 -> 341; 2000 and 8 of
// 64 over 500, 8 heads of 64, f16 46 -> 66; the other side four of 512 and 32 of 8, 8 heads, one of keys, int8 149 -> 139, and 1000 and 30 of 9, 16 heads, 4 of keys, of 80, f16 132 -> 122.)
constexpr int FEW_ROWS = 64, LIKE_ROWS = 32;
bool few_is_faster(const PagedArgs &a) {
    const int64_t rows = (int64_t)a.attn.G * a.pages.Sq, cus = cu_count();
    if (rows <= FEW_ROWS) return true;
    const int width = (a.pages.dk + 31) / 32 - 1;
    constexpr double FEW_STEP[] = {0.9, 1.3, 2.2, 2.5}, BLOCK[] = {3.0, 4.4, 4.0, 4.7};
    const int64_t units = a.pages.B * (int64_t)a.pages.heads * ((rows + 15) / 16), keys = paged_steps_most(a, 5, 16);
    if (units > 64 * cus) return false;
    const int64_t splits = paged_few_splits(units, keys), rounds = (units * splits + cus - 1) / cus, steps = ((keys + splits - 1) / splits + 7) / 8;
    const double few = (double)rounds * (5.5 + (double)steps * FEW_STEP[width]);
    const int64_t tile_rows = rows > 128 ? 256 : 128, tiles = a.pages.B * (int64_t)a.pages.heads * ((rows + tile_rows - 1) / tile_rows), blocks = paged_steps_most(a, a.pages.dk <= 64 ? 7 : 6, tile_rows);
    const int64_t ranges = paged_tile_splits(tiles, blocks), tile_rounds = (tiles * ranges + cus - 1) / cus;
    const double by_tiles = (double)tile_rounds * (10.0 + (double)((blocks + ranges - 1) / ranges) * BLOCK[width] * (tile_rows == 256 ? 1.0 : 0.7)) + (ranges > 1 ? 9.0 : 0.0);
    return few < by_tiles;
}

}  // namespace

extern "C" int axhip_attn_paged(const float *Q, int64_t ldq, const axhip_kv_cache *cache, float *O, int64_t ldo, float *L, const int32_t *first, const int32_t *lens, int64_t B,
                                int64_t T, int64_t H, int64_t Sq, int64_t Sk, float scale, const axhip_kv_rules *rules) {
    static const char who[] = "attn_paged";
    if (int rc = ensure_ready()) return rc;
    PagedArgs a = {};
    if (int rc = kv_arguments(who, a.pages, cache, first, lens, B, T, Sq)) return rc;
    if (!Q || !O) return fail(AXHIP_ERR_NULL_ARG, "%s: NULL tensor", who);
    if (H < 1 || H > (1 << 20) || H % cache->heads != 0) return fail(AXHIP_ERR_SHAPE, "%s: query heads must be a multiple of the heads of keys", who);
    if (Sk < 0 || Sk > (1 << 24)) return fail(AXHIP_ERR_SHAPE, "%s: bad extent", who);
    for (int64_t ld : {ldq, ldo})
        if (ld < H * cache->dk || ld % 4 != 0 || ld > (1 << 22)) return fail(AXHIP_ERR_SHAPE, "%s: row pitch must hold the heads, be a multiple of 4 and at most 2^22 floats", who);
    if ((((uintptr_t)Q | (uintptr_t)O) & 15) != 0) return fail(AXHIP_ERR_SHAPE, "%s: tensors must be 16-byte aligned", who);
    if (B * H > 0x7fffffff) return fail(AXHIP_ERR_SHAPE, "%s: too many sequences", who);
    axhip_kv_rules r = {};
    if (rules) r = *rules;
    if (!(r.cap >= 0.0f) || isinf(r.cap)) return fail(AXHIP_ERR_SHAPE, "%s: the cap must be zero or positive", who);
    if (r.cap > 0.0f && isinf(1.0f / (r.cap * LOG2E))) return fail(AXHIP_ERR_SHAPE, "%s: the cap must be zero or at least 2.1e-39", who);
    if (isfinite(scale) && isinf(scale * LOG2E)) return fail(AXHIP_ERR_SHAPE, "%s: the scale must be below 2.35e38", who);
    if (r.window < 0 || r.sinks < 0) return fail(AXHIP_ERR_SHAPE, "%s: window and first tokens must not be negative", who);
    if (B == 0 || T == 0 || Sq == 0) return AXHIP_OK;
    AttnArgs &t = a.attn;
    t.Q = Q;
    t.O = O;
    t.L = L;
    t.ldq = ldq;
    t.ldo = ldo;
    t.H = (int)H;
    t.G = (int)(H / cache->heads);
    t.scale = scale;
    t.q_up = scale * LOG2E;
    t.cap = r.cap;
    t.cap_down = r.cap > 0.0f ? (float)(1.0 / ((double)r.cap * LOG2E)) : 0.0f;
    t.cap_near = (float)((double)r.cap * LOG2E * TANH_NEAR);
    t.bias2 = LOG2E;
    t.slopes = r.slopes;
    constexpr int PAST = 1 << 25;                    // all positions; sums with it stay integers
    a.window = r.window < PAST ? r.window : PAST;
    a.sinks = r.window == 0 ? 0 : r.sinks < PAST ? r.sinks : PAST;
    if (a.pages.room > Sk) a.pages.room = (int)Sk;
    // How many rows each sequence has is on the device: where some may have many and others few, both forms are launched, each for its own.  (There a sequence is few rows' with 32 of them, or one
    // token of many heads.)  Either form is right for any counts; as many rows as there can be are taken to be equal ones, and half as many to be near enough for few rows to take all.
    const int64_t most = a.pages.Sq;
    const bool equal = !first || T == B * most;
    if ((equal || B == 1 || 2 * T >= B * most || t.G * most <= FEW_ROWS) && few_is_faster(a)) return paged_few(a, cache->type, 0x7fffffff);
    if (equal || B == 1) return paged_tiles(a, cache->type, 0);
    const int like = t.G > LIKE_ROWS ? (t.G + 15) / 16 * 16 : LIKE_ROWS;
    if (int rc = paged_few(a, cache->type, like)) return rc;
    return paged_tiles(a, cache->type, like + 1);
}
