// What the kernels of attention under score rules share (axhip_attn_fwd, axhip_attn_bwd): their arguments, what a query sees, the cap, and rows and keys
// formed one at a time with fp32 instructions.
#pragma once
#include "common.h"

namespace axhip {

struct AttnArgs {
    const float *Q, *K, *V, *dO, *Oin, *Lin;
    float *O, *L, *dQ, *dK, *dV, *delta;         // delta [B, H, Sq]: sum of dO * O of each row
    int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv, kv_rows;
    int B, H, Hkv, G, Sq, Sk, dk;                // G: query heads to a head of keys
    float scale;                                 // gradients of q and k are sums of ds * scale
    float q_up;                                  // a query is taken times this: its products are scores in log2 units
    float cap, cap_down, cap_near;               // the cap (0: none); one over it in log2 units; how far scores are near zero for it, in log2 units
    float bias2;                                 // log2(e) for the slopes
    const float *slopes;
    const int32_t *prefix, *start, *lens, *doc_q, *doc_k;
    int causal;
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float ATTN_LOWEST = -3.402823466e+38f; // where a running maximum starts: finite, so that scores of -infinity weigh nothing

// A row of queries: which keys it sees are those before `end` whose document is `doc` (any where there are no documents).
struct AttnRow {
    int p, end, doc;
    float slope2;                                // log2 units
};

// What all rows of a sequence share: its keys, the position of its first query, its prefix
struct AttnSeq {
    int len, start, prefix;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int b) {
    constexpr int FAR = 1 << 24;
    AttnSeq s = {a.Sk, a.Sk - a.Sq, 0};
    if (a.lens) s.len = min(max(a.lens[b], 0), a.Sk);
    if (a.start) s.start = min(max(a.start[b], -FAR), FAR);
    if (a.prefix) s.prefix = a.prefix[b];
    return s;
}
// doc: of the row, where there are documents
__device__ __forceinline__ AttnRow attn_row(const AttnArgs &a, const AttnSeq &s, int i, int doc, float slope) {
    AttnRow r;
    r.p = s.start + i;
    r.end = s.len;
    if (a.causal) {
        const int e = max(r.p + 1, s.prefix);
        r.end = r.p >= s.len || e <= 0 ? 0 : min(e, s.len);
    }
    r.doc = a.doc_q ? doc : 0;
    if (r.doc < 0) r.end = 0;
    r.slope2 = slope * a.bias2;
    return r;
}
__device__ __forceinline__ AttnRow attn_row(const AttnArgs &a, int b, int head, int i) {
    return attn_row(a, attn_seq(a, b), i, a.doc_q ? a.doc_q[(int64_t)b * a.Sq + i] : 0, a.slopes ? a.slopes[head] : 0.0f);
}

// A score x in log2 units under a cap c in the same units, c tanh(u) with u = x / c, and its derivative.  Near zero tanh(u) is u (1 + w), w = u^2 p(u^2) a minimax fit
// of degree 4 on |u| < 0.6 (relative error 5e-9 before rounding), and the score is x + x w: as precise as x under any cap, though u may have lost its bits.
// Beyond, with r = 2 / (e^(2|u|) + 1), they are c (1 - r) and r (2 - r), neither of which cancels; c may be past the largest float, the cap itself is not.
constexpr float TANH_NEAR = 0.6f;
struct Capped {
    float score, slope;
};
__device__ __forceinline__ Capped capped_near(const AttnArgs &a, float x) {
    const float u = x * a.cap_down, uu = u * u;
    float p = __builtin_fmaf(uu, -0.005895156413316727f, 0.020795969292521477f);
    p = __builtin_fmaf(uu, p, -0.053783830255270004f);
    p = __builtin_fmaf(uu, p, 0.13331924378871918f);
    p = __builtin_fmaf(uu, p, -0.33333298563957214f);
    const float w = uu * p, t = __builtin_fmaf(u, w, u);
    return {__builtin_fmaf(x, w, x), __builtin_fmaf(-t, t, 1.0f)};
}
__device__ __forceinline__ Capped capped(const AttnArgs &a, float x) {
    const float u = __builtin_fabsf(x * a.cap_down);
    const float r = 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(u * 2.8853900817779268f) + 1.0f);
    const Capped near = capped_near(a, x);
    return u < TANH_NEAR ? near : Capped{__builtin_copysignf(__builtin_fmaf(-a.cap, r, a.cap) * LOG2E, x), r * (2.0f - r)};
}

// A score in log2 units from a product of q (times q_up) and k
__device__ __forceinline__ float attn_score(const AttnArgs &a, float product, const AttnRow &r, int key, float &slope) {
    slope = 1.0f;
    if (a.cap > 0.0f) {
        const Capped c = capped(a, product);
        product = c.score;
        slope = c.slope;
    }
    return a.slopes ? __builtin_fmaf(-r.slope2, (float)(r.p > key ? r.p - key : key - r.p), product) : product;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
__device__ __forceinline__ float from_lane(float v, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); }

__device__ __forceinline__ float attn_dot(const float *x, const float *y, int dk, float up) {
    float s = 0.0f;
    for (int c = 0; c < dk; c += 4) {
        const v4f p = *reinterpret_cast<const v4f *>(x + c), q = *reinterpret_cast<const v4f *>(y + c);
#pragma unroll
        for (int e = 0; e < 4; e++) s = __builtin_fmaf(p[e] * up, q[e], s);
    }
    return s;
}

__device__ __forceinline__ bool attn_sees(const AttnArgs &a, const AttnRow &r, int b, int key) {
    return key < r.end && (!a.doc_k || a.doc_k[(int64_t)b * a.Sk + key] == r.doc);
}

// ---- one row, or one key, by one wave with fp32 instructions: what the matrix kernels' tiles fall back to where sums are not finite.  64 keys (or
// rows) at a time, a score a lane; then a value column a lane (two where dk > 64) and only pairs that see each other are added, so what a masked
// pair holds is never touched. ----
__device__ __forceinline__ void attn_fwd_row(const AttnArgs &a, int b, int head, int i, int lane) {
    const AttnRow r = attn_row(a, b, head, i);
    const int hk = head / a.G;
    const float *q = a.Q + ((int64_t)b * a.Sq + i) * a.ldq + (int64_t)head * a.dk;
    const float *K = a.K + (int64_t)b * a.kv_rows * a.ldk + (int64_t)hk * a.dk, *V = a.V + (int64_t)b * a.kv_rows * a.ldv + (int64_t)hk * a.dk;
    float m = ATTN_LOWEST, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    bool any = false;
    for (int k0 = 0; k0 < r.end; k0 += 64) {
        const int key = k0 + lane;
        const bool sees = attn_sees(a, r, b, key);
        float x = -INFINITY, slope;
        if (sees) x = attn_score(a, attn_dot(q, K + (int64_t)key * a.ldk, a.dk, a.q_up), r, key, slope);
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
            const float pj = from_lane(p, j);
            const float *v = V + (int64_t)(k0 + j) * a.ldv;
            if (lane < a.dk) o0 = __builtin_fmaf(pj, v[lane], o0);
            if (lane + 64 < a.dk) o1 = __builtin_fmaf(pj, v[lane + 64], o1);
        }
    }
    float *o = a.O + ((int64_t)b * a.Sq + i) * a.ldo + (int64_t)head * a.dk;
    const float inv = any ? 1.0f / l : 0.0f;
    if (lane < a.dk) o[lane] = any ? o0 * inv : 0.0f;
    if (lane + 64 < a.dk) o[lane + 64] = any ? o1 * inv : 0.0f;
    // (a row that saw nothing but scores of -infinity: 0 / 0 above, and NaN here)
    if (a.L && lane == 0) a.L[((int64_t)b * a.H + head) * a.Sq + i] = !any ? -INFINITY : l == 0.0f ? NAN : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// p and ds = p (dp - delta) * slope of a pair that sees each other
__device__ __forceinline__ void attn_pair(const AttnArgs &a, const AttnRow &r, int key, const float *q, const float *k, const float *v, const float *d_o,
                                          float lse2, float delta, float &p, float &ds) {
    float slope;
    p = __builtin_amdgcn_exp2f(attn_score(a, attn_dot(q, k, a.dk, a.q_up), r, key, slope) - lse2);
    ds = p * (attn_dot(d_o, v, a.dk, 1.0f) - delta) * slope;
}

// The gradient of query row i.  (Its delta for the keys' side is left as the matrix kernel wrote it: of splits of a row's keys another workgroup did.)
__device__ __forceinline__ void attn_dq_row(const AttnArgs &a, int b, int head, int i, int lane) {
    const AttnRow r = attn_row(a, b, head, i);
    const int hk = head / a.G;
    const int64_t row = (int64_t)b * a.Sq + i, at = ((int64_t)b * a.H + head) * a.Sq + i;
    const float *q = a.Q + row * a.ldq + (int64_t)head * a.dk, *d_o = a.dO + row * a.lddo + (int64_t)head * a.dk;
    const float *o = a.Oin + row * a.ldo + (int64_t)head * a.dk;
    const float *K = a.K + (int64_t)b * a.kv_rows * a.ldk + (int64_t)hk * a.dk, *V = a.V + (int64_t)b * a.kv_rows * a.ldv + (int64_t)hk * a.dk;
    const float lse2 = a.Lin[at] * LOG2E;
    float delta = 0.0f, g0 = 0.0f, g1 = 0.0f;
    if (r.end > 0) {
        if (lane < a.dk) delta = d_o[lane] * o[lane];
        if (lane + 64 < a.dk) delta = __builtin_fmaf(d_o[lane + 64], o[lane + 64], delta);
        delta = wave_sum(delta);
    }
    for (int k0 = 0; k0 < r.end; k0 += 64) {
        const int key = k0 + lane;
        const bool sees = attn_sees(a, r, b, key);
        float p, ds = 0.0f;
        if (sees) attn_pair(a, r, key, q, K + (int64_t)key * a.ldk, V + (int64_t)key * a.ldv, d_o, lse2, delta, p, ds);
        for (uint64_t seen = __builtin_amdgcn_ballot_w64(sees); seen; seen &= seen - 1) {
            const int j = __builtin_ctzll(seen);
            const float dj = from_lane(ds, j);
            const float *k = K + (int64_t)(k0 + j) * a.ldk;
            if (lane < a.dk) g0 = __builtin_fmaf(dj, k[lane], g0);
            if (lane + 64 < a.dk) g1 = __builtin_fmaf(dj, k[lane + 64], g1);
        }
    }
    float *dq = a.dQ + row * a.lddq + (int64_t)head * a.dk;
    if (lane < a.dk) dq[lane] = g0 * a.scale;
    if (lane + 64 < a.dk) dq[lane + 64] = g1 * a.scale;
}

// The gradients of key and value row j of head hk
__device__ __forceinline__ void attn_dkv_row(const AttnArgs &a, int b, int hk, int j, int lane) {
    const int64_t row = (int64_t)b * a.kv_rows + j;
    const float *k = a.K + row * a.ldk + (int64_t)hk * a.dk, *v = a.V + row * a.ldv + (int64_t)hk * a.dk;
    float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
    for (int head = hk * a.G; head < (hk + 1) * a.G; head++)
        for (int i0 = 0; i0 < a.Sq; i0 += 64) {
            const int i = i0 + lane;
            const float *Q = a.Q + ((int64_t)b * a.Sq + i0) * a.ldq + (int64_t)head * a.dk, *dO = a.dO + ((int64_t)b * a.Sq + i0) * a.lddo + (int64_t)head * a.dk;
            bool sees = false;
            float p = 0.0f, ds = 0.0f;
            if (i < a.Sq) {
                const AttnRow r = attn_row(a, b, head, i);
                sees = attn_sees(a, r, b, j);
                const int64_t at = ((int64_t)b * a.H + head) * a.Sq + i;
                if (sees) attn_pair(a, r, j, Q + (int64_t)lane * a.ldq, k, v, dO + (int64_t)lane * a.lddo, a.Lin[at] * LOG2E, a.delta[at], p, ds);
            }
            for (uint64_t seen = __builtin_amdgcn_ballot_w64(sees); seen; seen &= seen - 1) {
                const int n = __builtin_ctzll(seen);
                const float pn = from_lane(p, n), dn = from_lane(ds, n);
                const float *q = Q + (int64_t)n * a.ldq, *d_o = dO + (int64_t)n * a.lddo;
                if (lane < a.dk) {
                    k0 = __builtin_fmaf(dn, q[lane], k0);
                    v0 = __builtin_fmaf(pn, d_o[lane], v0);
                }
                if (lane + 64 < a.dk) {
                    k1 = __builtin_fmaf(dn, q[lane + 64], k1);
                    v1 = __builtin_fmaf(pn, d_o[lane + 64], v1);
                }
            }
        }
    float *dk = a.dK + row * a.lddk + (int64_t)hk * a.dk, *dv = a.dV + row * a.lddv + (int64_t)hk * a.dk;
    if (lane < a.dk) {
        dk[lane] = k0 * a.scale;
        dv[lane] = v0;
    }
    if (lane + 64 < a.dk) {
        dk[lane + 64] = k1 * a.scale;
        dv[lane + 64] = v1;
    }
}

}  // namespace axhip
