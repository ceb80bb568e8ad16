// Attention under score rules (capped, biased by distance, masked by documents, prefixes or lengths; shared heads of keys), forward and backward.
#include <math.h>

#include "attn_launch.h"

namespace {
using namespace axhip;

struct Tensor {
    const void *at;
    int64_t ld, heads;
};

// Checks that both entry points make, and the arguments that both pass on
int attn_arguments(const char *who, AttnArgs &a, const Tensor *tensors, int n, int64_t kv_rows, int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk,
                   int64_t dk, float scale, const axhip_attn_rules *rules) {
    for (int t = 0; t < n; t++)
        if (!tensors[t].at) return fail(AXHIP_ERR_NULL_ARG, "%s: NULL tensor", who);
    constexpr int64_t LONG = 1 << 24;
    if (B < 0 || H <= 0 || Hkv <= 0 || Sq < 0 || Sk < 0 || Sq > LONG || Sk > LONG) return fail(AXHIP_ERR_SHAPE, "%s: bad extent", who);
    if (H > (1 << 20)) return fail(AXHIP_ERR_SHAPE, "%s: too many heads", who);        // (more would not fit a row pitch, and their sizes might not fit 64 bits)
    if (H % Hkv != 0) return fail(AXHIP_ERR_SHAPE, "%s: query heads must be a multiple of the heads of keys", who);
    if (dk < 4 || dk > 128 || dk % 4 != 0) return fail(AXHIP_ERR_NOT_IMPLEMENTED, "%s: head size %lld (multiples of 4 up to 128 only)", who, (long long)dk);
    if (kv_rows < Sk) return fail(AXHIP_ERR_SHAPE, "%s: kv_rows must hold Sk rows", who);
    for (int t = 0; t < n; t++) {
        if (tensors[t].ld < tensors[t].heads * dk || tensors[t].ld % 4 != 0 || tensors[t].ld > (1 << 22))
            return fail(AXHIP_ERR_SHAPE, "%s: row pitch must hold the heads, be a multiple of 4 and at most 2^22 floats", who);
        if (((uintptr_t)tensors[t].at & 15) != 0) return fail(AXHIP_ERR_SHAPE, "%s: tensors must be 16-byte aligned", who);
    }
    if (B > 0x7fffff || B * H > 0x7fffffff || kv_rows > ((int64_t)1 << 40)) return fail(AXHIP_ERR_SHAPE, "%s: too many sequences", who);
    axhip_attn_rules r = {};
    if (rules) r = *rules;
    if (!(r.cap >= 0.0f) || isinf(r.cap)) return fail(AXHIP_ERR_SHAPE, "%s: the cap must be zero or positive", who);
    if (r.cap > 0.0f && isinf(1.0f / (r.cap * LOG2E))) return fail(AXHIP_ERR_SHAPE, "%s: the cap must be zero or at least 2.1e-39", who);
    if (isfinite(scale) && isinf(scale * LOG2E)) return fail(AXHIP_ERR_SHAPE, "%s: the scale must be below 2.35e38", who);
    if (r.prefix && !r.causal) return fail(AXHIP_ERR_SHAPE, "%s: a prefix without a causal mask", who);
    if ((r.doc_q == nullptr) != (r.doc_k == nullptr)) return fail(AXHIP_ERR_NULL_ARG, "%s: documents of queries and of keys, or neither", who);
    a.kv_rows = kv_rows;
    a.B = (int)B;
    a.H = (int)H;
    a.Hkv = (int)Hkv;
    a.G = (int)(H / Hkv);
    a.Sq = (int)Sq;
    a.Sk = (int)Sk;
    a.dk = (int)dk;
    a.scale = scale;
    a.q_up = scale * LOG2E;
    a.cap = r.cap;
    a.cap_down = r.cap > 0.0f ? (float)(1.0 / ((double)r.cap * LOG2E)) : 0.0f;
    a.cap_near = (float)((double)r.cap * LOG2E * TANH_NEAR);
    a.bias2 = LOG2E;
    a.slopes = r.slopes;
    a.prefix = r.prefix;
    a.start = r.start;
    a.lens = r.lens;
    a.doc_q = r.doc_q;
    a.doc_k = r.doc_k;
    a.causal = r.causal != 0;
    return AXHIP_OK;
}

}  // namespace

extern "C" int axhip_attn_fwd(const float *Q, int64_t ldq, const float *K, int64_t ldk, const float *V, int64_t ldv, int64_t kv_rows, float *O, int64_t ldo,
                              float *L, int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t dk, float scale, const axhip_attn_rules *rules) {
    if (int rc = ensure_ready()) return rc;
    AttnArgs a = {};
    const Tensor tensors[] = {{Q, ldq, H}, {K, ldk, Hkv}, {V, ldv, Hkv}, {O, ldo, H}};
    if (int rc = attn_arguments("attn_fwd", a, tensors, 4, kv_rows, B, H, Hkv, Sq, Sk, dk, scale, rules)) return rc;
    if (B == 0 || Sq == 0) return AXHIP_OK;
    a.Q = Q;
    a.K = K;
    a.V = V;
    a.O = O;
    a.L = L;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldo = ldo;
    int rc = AXHIP_OK;
    return attn_fwd_few(a, rc) ? rc : attn_fwd_tiles(a);
}

extern "C" int axhip_attn_bwd(const float *Q, int64_t ldq, const float *K, int64_t ldk, const float *V, int64_t ldv, int64_t kv_rows, const float *O,
                              int64_t ldo, const float *L, const float *dO, int64_t lddo, float *dQ, int64_t lddq, float *dK, int64_t lddk, float *dV,
                              int64_t lddv, int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t dk, float scale,
                              const axhip_attn_rules *rules) {
    if (int rc = ensure_ready()) return rc;
    if (!L) return fail(AXHIP_ERR_NULL_ARG, "attn_bwd: NULL log-sum-exp");
    AttnArgs a = {};
    const Tensor tensors[] = {{Q, ldq, H}, {K, ldk, Hkv}, {V, ldv, Hkv}, {O, ldo, H}, {dO, lddo, H}, {dQ, lddq, H}, {dK, lddk, Hkv}, {dV, lddv, Hkv}};
    if (int rc = attn_arguments("attn_bwd", a, tensors, 8, kv_rows, B, H, Hkv, Sq, Sk, dk, scale, rules)) return rc;
    if (B == 0) return AXHIP_OK;
    a.Q = Q;
    a.K = K;
    a.V = V;
    a.Oin = O;
    a.Lin = L;
    a.dO = dO;
    a.dQ = dQ;
    a.dK = dK;
    a.dV = dV;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldo = ldo;
    a.lddo = lddo;
    a.lddq = lddq;
    a.lddk = lddk;
    a.lddv = lddv;
    return Sk == 0 && Sq == 0 ? AXHIP_OK : attn_bwd_tiles(a);
}
