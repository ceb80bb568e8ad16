// Attention of new tokens over a paged cache of keys and values in few bits (axhip_attn_paged): checks, and who takes the call.
#include <math.h>

#include "attn_launch.h"
#include "paged.h"

namespace {
using namespace axhip;

// Sequences with more rows than this (new tokens, times the query heads that share keys) go over tiles
constexpr int FEW_ROWS = 32;

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
    // A sequence with few rows is read by the form that shares out its keys, others by tiles.  How many rows each sequence has is on the device, so both may have to be launched, each
    // for its own; not where all have the same number of rows, or none can have more than a few.
    const int64_t rows = (int64_t)t.G * Sq;
    if (rows <= FEW_ROWS) return paged_few(a, cache->type, FEW_ROWS);
    if (!first || B == 1) return paged_tiles(a, cache->type, 0);
    if (int rc = paged_few(a, cache->type, FEW_ROWS)) return rc;
    return paged_tiles(a, cache->type, FEW_ROWS + 1);
}
