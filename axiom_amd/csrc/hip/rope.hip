// Rotary positions and the norms of query and key heads, on rows that hold heads side by side.
//   rotation   pair (x, y) of a head -> amplitude (x cos a - y sin a, y cos a + x sin a), a = pos[row] * freq[pair]; backward: -a
//   norm       r = 1 / sqrt(mean x^2 + eps), y = rotation(gamma x r)
//   gradient   dn = rotation^T dy, dgamma = sum dn x r, dx = r (gamma dn - x r mean(gamma dn x r))
// HBM-bound: 8 bytes a value (12 backward) against some ten operations.  16000 rows of 24 heads of 128 turned 71 us, 5.5 TB/s; 8192 rows of 40 heads of 128 normed and turned 63 us, 5.35
// TB/s; the gradient for 4000 rows of 32 heads of 80 26 us, 4.7 TB/s, and 4 for the launch that joins the gammas' sums
// (a workgroup's sums in fp32, joined in 64 bits, in a fixed order: 0.9e-7 of their size there; 0.6e-7 would be 64 bits throughout, 1.3e-7 was fp32 throughout); 8 or 16 rows 4.5 to 4.8 us, what a launch and one trip to memory take.
//
// k_heads: a lane holds a unit of 8 columns of a head (two 16-byte accesses): four pairs, either eight neighbours or four from each half of the
// rotated part, so a rotation never leaves the lane and a norm is a sum over the 4 to 64 lanes of a head.  The four angles of a
// lane are the same for every head of a row: a group of lanes forms them once and walks over heads of the row, HEADS at a time in flight.
// k_heads_any, a wave per head, takes head sizes, rotated parts and pitches off that grid.
#include <math.h>

#include "common.h"

namespace {
using namespace axhip;

enum Mode { ROTATE, NORM, NORM_GRAD };

struct HeadsArgs {
    const float *x, *dy;                         // NORM_GRAD: dy beside x
    float *y, *inv;                              // y: dx for NORM_GRAD; inv: read by NORM_GRAD, written by NORM if not NULL
    const float *gamma_q, *gamma_k;              // NULL: ones
    float *partial;                              // NORM_GRAD: [workgroups, 2, dk] sums for dgamma
    const int32_t *pos;
    const float *freq;
    int64_t ldx, lddy, ldy, rows;
    int heads, q_heads, dk, rot, chunk, chunks;  // a group of lanes takes `chunk` heads of a row
    float eps, amplitude, sign;                  // sign: -1 turns back
    bool halves;
};

// amplitude * cos and sin of pos * freq.  The product of a 32-bit integer and a 24-bit float is formed in 64 bits, in turns; what is left of the nearest
// quarter turn fits 32 bits to 2^-28 turns, so positions in the millions are as exact as small ones.
__device__ __forceinline__ void turn_of(int pos, float freq, float amplitude, float sign, float &c, float &s) {
    const double t = (double)pos * (double)freq * 0.15915494309189535;
    const double quarter = __builtin_rint(t * 4.0);
    const float rest = (float)__builtin_fma(quarter, -0.25, t);
    float sr, cr;
    sincospif(2.0f * rest, &sr, &cr);
    const int q = (int)(quarter - 4.0 * __builtin_floor(quarter * 0.25));
    const float cq = (q & 1) ? sr : cr, sq = (q & 1) ? cr : sr;
    c = amplitude * (q == 1 || q == 2 ? -cq : cq);
    s = amplitude * sign * (q >= 2 ? -sq : sq);
}

// Columns of unit u: four from `a` on and four from `b` on
__device__ __forceinline__ void unit_columns(const HeadsArgs &p, int u, int &a, int &b) {
    const bool split = p.halves && 8 * u < p.rot;
    a = split ? 4 * u : 8 * u;
    b = split ? p.rot / 2 + 4 * u : 8 * u + 4;
}

// The pairs of a unit turned: pair i is (v[i], v[4 + i]) in halves, (v[2 i], v[2 i + 1]) otherwise.  Lanes past the rotated part hold c = 1, s = 0.
__device__ __forceinline__ void turn_unit(float (&v)[8], const float (&c)[4], const float (&s)[4], bool split) {
    float o[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = split ? v[i] : v[2 * i], y = split ? v[4 + i] : v[2 * i + 1];
        const float a = __builtin_fmaf(x, c[i], -(y * s[i])), b = __builtin_fmaf(y, c[i], x * s[i]);
        o[i] = a;
        o[4 + i] = b;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[split ? i : 2 * i] = o[i];
        v[split ? 4 + i : 2 * i + 1] = o[4 + i];
    }
}

template <int LANES>
__device__ __forceinline__ float sum_of_lanes(float v) {
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

template <Mode MODE, int LANES, bool HALVES>
__global__ void __launch_bounds__(256) k_heads(HeadsArgs p) {
    constexpr int HEADS = MODE == NORM_GRAD ? 2 : 4;
    constexpr int GROUPS = 256 / LANES;
    const int u = threadIdx.x % LANES;
    const bool in = 8 * u < p.dk, turned = 8 * u < p.rot, split = HALVES && turned;
    int ca, cb;
    unit_columns(p, u, ca, cb);
    float gq[8], gk[8], dgq[8], dgk[8];
    if (MODE != ROTATE)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int col = e < 4 ? ca + e : cb + e - 4;
            gq[e] = in && p.gamma_q ? p.gamma_q[col] : 1.0f;
            gk[e] = in && p.gamma_k ? p.gamma_k[col] : 1.0f;
            dgq[e] = dgk[e] = 0.0f;
        }
    const float over = 1.0f / (float)p.dk;
    const int64_t items = p.rows * p.chunks, step = (int64_t)gridDim.x * GROUPS;
    for (int64_t item = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES; item < items; item += step) {
        const int64_t row = p.chunks == 1 ? item : item / p.chunks;
        const int h0 = (int)(item - row * p.chunks) * p.chunk, h1 = h0 + p.chunk < p.heads ? h0 + p.chunk : p.heads;
        const float *x = p.x + row * p.ldx, *dy = MODE == NORM_GRAD ? p.dy + row * p.lddy : nullptr;
        float *y = p.y + row * p.ldy;
        float c[4], s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[i] = 1.0f;
            s[i] = 0.0f;
        }
        if (turned) {
            const int pos = p.pos[row];
            const v4f f = *reinterpret_cast<const v4f *>(p.freq + 4 * u);
#pragma unroll
            for (int i = 0; i < 4; i++) turn_of(pos, f[i], p.amplitude, p.sign, c[i], s[i]);
        }
        for (int h = h0; h < h1; h += HEADS) {
            float v[HEADS][8], d[HEADS][8], inv[HEADS];
#pragma unroll
            for (int n = 0; n < HEADS; n++) {
                v4f a = {0.f, 0.f, 0.f, 0.f}, b = a, da = a, db = a;
                const int at = (h + n) * p.dk;
                if (in && h + n < h1) {
                    a = *reinterpret_cast<const v4f *>(x + at + ca);
                    b = *reinterpret_cast<const v4f *>(x + at + cb);
                    if (MODE == NORM_GRAD) {
                        da = *reinterpret_cast<const v4f *>(dy + at + ca);
                        db = *reinterpret_cast<const v4f *>(dy + at + cb);
                    }
                }
                if (MODE == NORM_GRAD) inv[n] = h + n < h1 ? p.inv[row * p.heads + h + n] : 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[n][e] = a[e];
                    v[n][4 + e] = b[e];
                    d[n][e] = da[e];
                    d[n][4 + e] = db[e];
                }
            }
#pragma unroll
            for (int n = 0; n < HEADS; n++) {
                if (h + n >= h1) break;
                const bool is_q = h + n < p.q_heads;
                if (MODE == NORM) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; e++) sum = __builtin_fmaf(v[n][e], v[n][e], sum);
                    const float r = 1.0f / sqrtf(__builtin_fmaf(sum_of_lanes<LANES>(sum), over, p.eps));
                    if (p.inv && u == 0) p.inv[row * p.heads + h + n] = r;
#pragma unroll
                    for (int e = 0; e < 8; e++) v[n][e] *= r * (is_q ? gq[e] : gk[e]);
                }
                if (MODE == NORM_GRAD) {
                    turn_unit(d[n], c, s, split);
                    float inner = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float hat = v[n][e] * inv[n];
                        if (is_q) dgq[e] = __builtin_fmaf(d[n][e], hat, dgq[e]);
                        else dgk[e] = __builtin_fmaf(d[n][e], hat, dgk[e]);
                        d[n][e] *= is_q ? gq[e] : gk[e];
                        inner = __builtin_fmaf(d[n][e], hat, inner);
                        v[n][e] = hat;
                    }
                    inner = sum_of_lanes<LANES>(inner) * over;
#pragma unroll
                    for (int e = 0; e < 8; e++) v[n][e] = inv[n] * __builtin_fmaf(-inner, v[n][e], d[n][e]);
                } else {
                    turn_unit(v[n], c, s, split);
                }
                if (in) {
                    float *o = y + (h + n) * p.dk;
                    *reinterpret_cast<v4f *>(o + ca) = v4f{v[n][0], v[n][1], v[n][2], v[n][3]};
                    *reinterpret_cast<v4f *>(o + cb) = v4f{v[n][4], v[n][5], v[n][6], v[n][7]};
                }
            }
        }
    }
    if (MODE == NORM_GRAD && p.partial) {        // the groups of the workgroup, then one row of sums for it
        __shared__ float sums[2][256 * 8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            sums[0][e * 256 + threadIdx.x] = dgq[e];
            sums[1][e * 256 + threadIdx.x] = dgk[e];
        }
        __syncthreads();
        if ((int)threadIdx.x < LANES && in)
            for (int which = 0; which < 2; which++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float sum = 0.0f;
                    for (int g = 0; g < GROUPS; g++) sum += sums[which][e * 256 + g * LANES + u];
                    p.partial[((int64_t)blockIdx.x * 2 + which) * p.dk + (e < 4 ? ca + e : cb + e - 4)] = sum;
                }
    }
}

// Any even rotated part of any head: a wave per head, columns of a lane 64 apart.  A lane touches the same columns in both passes, so results may
// take the place of what is read.
template <Mode MODE>
__global__ void __launch_bounds__(64) k_heads_any(HeadsArgs p) {
    extern __shared__ float sums[];              // NORM_GRAD with sums wanted: [2][dk]
    const int lane = threadIdx.x, half = p.rot / 2;
    const float over = 1.0f / (float)p.dk;
    const bool sums_wanted = MODE == NORM_GRAD && p.partial;
    if (sums_wanted)
        for (int c = lane; c < 2 * p.dk; c += 64) sums[c] = 0.0f;
    __syncthreads();
    const int64_t items = p.rows * p.heads;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t row = item / p.heads;
        const int h = (int)(item - row * p.heads), at = h * p.dk;
        const bool is_q = h < p.q_heads;
        const float *x = p.x + row * p.ldx + at, *dy = MODE == NORM_GRAD ? p.dy + row * p.lddy + at : nullptr, *gamma = is_q ? p.gamma_q : p.gamma_k;
        float *y = p.y + row * p.ldy + at, *dg = sums + (is_q ? 0 : p.dk);
        const int pos = p.rot ? p.pos[row] : 0;
        float r = 1.0f, inner = 0.0f;
        if (MODE == NORM) {
            float sum = 0.0f;
            for (int c = lane; c < p.dk; c += 64) sum = __builtin_fmaf(x[c], x[c], sum);
            r = 1.0f / sqrtf(__builtin_fmaf(sum_of_lanes<64>(sum), over, p.eps));
            if (p.inv && lane == 0) p.inv[item] = r;
        }
        if (MODE == NORM_GRAD) r = p.inv[item];
        for (int pass = MODE == NORM_GRAD ? 0 : 1; pass < 2; pass++) {
            auto column = [&](int col, float dn) {   // the gradient from the turned dn on
                const float hat = x[col] * r, gdn = dn * (gamma ? gamma[col] : 1.0f);
                if (pass == 0) {
                    inner = __builtin_fmaf(gdn, hat, inner);
                    if (sums_wanted) dg[col] = __builtin_fmaf(dn, hat, dg[col]);
                } else {
                    y[col] = r * __builtin_fmaf(-inner, hat, gdn);
                }
            };
            for (int i = lane; i < half; i += 64) {
                const int ca = p.halves ? i : 2 * i, cb = p.halves ? half + i : 2 * i + 1;
                float c, s;
                turn_of(pos, p.freq[i], p.amplitude, p.sign, c, s);
                float a = MODE == NORM_GRAD ? dy[ca] : x[ca], b = MODE == NORM_GRAD ? dy[cb] : x[cb];
                if (MODE == NORM) {
                    a *= r * (gamma ? gamma[ca] : 1.0f);
                    b *= r * (gamma ? gamma[cb] : 1.0f);
                }
                const float ta = __builtin_fmaf(a, c, -(b * s)), tb = __builtin_fmaf(b, c, a * s);
                if (MODE == NORM_GRAD) {
                    column(ca, ta);
                    column(cb, tb);
                } else {
                    y[ca] = ta;
                    y[cb] = tb;
                }
            }
            for (int col = p.rot + lane; col < p.dk; col += 64) {
                if (MODE == NORM_GRAD) column(col, dy[col]);
                else y[col] = MODE == NORM ? x[col] * (r * (gamma ? gamma[col] : 1.0f)) : x[col];
            }
            if (MODE == NORM_GRAD && pass == 0) inner = sum_of_lanes<64>(inner) * over;
        }
    }
    if (sums_wanted) {
        __syncthreads();
        for (int c = lane; c < 2 * p.dk; c += 64) p.partial[(int64_t)blockIdx.x * 2 * p.dk + c] = sums[c];
    }
}

// dgamma from the workgroups' sums, in 64 bits and rounded once: 16 columns a workgroup, its 64 parts take the sums in turn, sixteen loads of each under way
__global__ void __launch_bounds__(1024) k_gamma_sums(const float *partial, int n, int dk, float *dgq, float *dgk) {
    __shared__ double parts[64][16];
    const int here = threadIdx.x & 15, col = blockIdx.x * 16 + here, part = threadIdx.x >> 4;
    double sum = 0.0;
    if (col < 2 * dk) {
#pragma unroll 16
        for (int b = part; b < n; b += 64) sum += partial[(int64_t)b * 2 * dk + col];
    }
    parts[part][here] = sum;
    __syncthreads();
    for (int half = 32; half > 0; half >>= 1) {
        if (part < half) parts[part][here] += parts[part + half][here];
        __syncthreads();
    }
    if (part != 0 || col >= 2 * dk) return;
    float *out = col < dk ? dgq : dgk;
    if (out) out[col < dk ? col : col - dk] = (float)parts[0][here];
}

constexpr int64_t GRAD_GROUPS = 1024;            // workgroups of four waves at most whose sums are joined by k_gamma_sums (of one: four times as many)

template <Mode MODE, int LANES>
int launch_heads(HeadsArgs &p, unsigned grid) {
    note_kernel(MODE == ROTATE ? "rope_rows" : MODE == NORM ? "qk_norm_rope" : "qk_norm_rope_grad");
    if (p.halves) hipLaunchKernelGGL((k_heads<MODE, LANES, true>), dim3(grid), dim3(256), 0, kStream, p);
    else hipLaunchKernelGGL((k_heads<MODE, LANES, false>), dim3(grid), dim3(256), 0, kStream, p);
    return check_launch("rope");
}

template <Mode MODE>
int run_heads(HeadsArgs &p, float *dgq, float *dgk) {
    auto off = [](const void *q, int64_t ld) { return q && (((uintptr_t)q & 15) != 0 || ld % 4 != 0); };
    const bool sums_wanted = MODE == NORM_GRAD && (dgq || dgk);
    const bool units = p.dk % 8 == 0 && p.rot % 8 == 0 && p.dk <= 512 && !off(p.x, p.ldx) && !off(p.y, p.ldy) && !off(p.dy, p.lddy) && !off(p.freq, 0);
    int64_t grid;
    int lanes = 4;
    if (units) {
        while (8 * lanes < p.dk) lanes *= 2;
        const int64_t groups = 256 / lanes;
        // A group of lanes takes four heads of a row, what it has under way at a time, so that its angles serve four; fewer where that leaves less than eight waves a
        // CU.  (us, whole rows -> four heads: 16000 rows of 24 heads of 128 89 -> 78, but one head each 80; 2000 rows of 20 heads of 64, two each 6.2, one each 7.5.)
        const int64_t want = (int64_t)cu_count() * 8 * 64 / lanes;
        p.chunk = 4;
        while (p.chunk > 1 && p.rows * ((p.heads + p.chunk - 1) / p.chunk) < want) p.chunk /= 2;
        p.chunks = (p.heads + p.chunk - 1) / p.chunk;
        grid = (p.rows * p.chunks + groups - 1) / groups;
    } else {
        grid = p.rows * p.heads;
    }
    const int64_t most = !sums_wanted ? 1 << 22 : units ? GRAD_GROUPS : 4 * GRAD_GROUPS;
    if (grid > most) grid = most;
    if (sums_wanted && !(p.partial = static_cast<float *>(workspace((size_t)grid * 2 * p.dk * sizeof(float))))) return AXHIP_ERR_ALLOC;
    int rc;
    if (!units) {
        note_kernel(MODE == ROTATE ? "rope_rows_any" : MODE == NORM ? "qk_norm_rope_any" : "qk_norm_rope_grad_any");
        hipLaunchKernelGGL((k_heads_any<MODE>), dim3((unsigned)grid), dim3(64), sums_wanted ? 2 * p.dk * sizeof(float) : 0, kStream, p);
        rc = check_launch("rope");
    } else if (lanes == 4) rc = launch_heads<MODE, 4>(p, (unsigned)grid);
    else if (lanes == 8) rc = launch_heads<MODE, 8>(p, (unsigned)grid);
    else if (lanes == 16) rc = launch_heads<MODE, 16>(p, (unsigned)grid);
    else if (lanes == 32) rc = launch_heads<MODE, 32>(p, (unsigned)grid);
    else rc = launch_heads<MODE, 64>(p, (unsigned)grid);
    if (rc || !sums_wanted) return rc;
    hipLaunchKernelGGL(k_gamma_sums, dim3((unsigned)((2 * p.dk + 15) / 16)), dim3(1024), 0, kStream, p.partial, (int)grid, p.dk, dgq, dgk);
    return check_launch("rope gamma sums");
}

// What the three entry points ask of rows, heads and rotation alike
int check_heads(const char *who, int64_t rows, int64_t H, int64_t Hk, int64_t dk, int64_t rot, int layout, const int32_t *pos, const float *freq) {
    if (rows < 0 || H < 0 || Hk < 0 || dk <= 0 || dk > 4096 || H > (1 << 20) || Hk > (1 << 20)) return fail(AXHIP_ERR_SHAPE, "%s: bad extent", who);
    if ((H + Hk) * dk > 0x7fffffff || rows > ((int64_t)1 << 40)) return fail(AXHIP_ERR_SHAPE, "%s: too many heads or rows", who);
    if (rot < 0 || rot > dk || rot % 2 != 0) return fail(AXHIP_ERR_SHAPE, "%s: the rotated part must be even and within the head", who);
    if (layout != AXHIP_ROPE_INTERLEAVED && layout != AXHIP_ROPE_HALVES) return fail(AXHIP_ERR_SHAPE, "%s: unknown layout %d", who, layout);
    if (rot > 0 && (!pos || !freq)) return fail(AXHIP_ERR_NULL_ARG, "%s: NULL positions or frequencies", who);
    return AXHIP_OK;
}

}  // namespace

extern "C" int axhip_rope_frequencies(float *freq, int64_t rot, double theta, int scaling, double factor, double slow, double fast, int64_t trained) {
    if (int rc = ensure_ready()) return rc;
    if (!freq) return fail(AXHIP_ERR_NULL_ARG, "rope_frequencies: NULL output");
    if (rot < 0 || rot > 4096 || rot % 2 != 0) return fail(AXHIP_ERR_SHAPE, "rope_frequencies: the rotated part must be even and at most 4096");
    if (!(theta > 0) || !isfinite(theta)) return fail(AXHIP_ERR_SHAPE, "rope_frequencies: theta must be positive");
    if (scaling < AXHIP_ROPE_PLAIN || scaling > AXHIP_ROPE_BY_PARTS) return fail(AXHIP_ERR_SHAPE, "rope_frequencies: unknown scaling %d", scaling);
    if (scaling != AXHIP_ROPE_PLAIN && (!(factor >= 1) || !isfinite(factor))) return fail(AXHIP_ERR_SHAPE, "rope_frequencies: factor must be at least 1");
    if (scaling == AXHIP_ROPE_BY_PARTS && (!(slow >= 0) || !(fast > slow) || !isfinite(fast) || trained < 1))
        return fail(AXHIP_ERR_SHAPE, "rope_frequencies: scaling by parts needs 0 <= slow < fast and a trained length");
    if (rot == 0) return AXHIP_OK;
    float host[2048];
    if (scaling == AXHIP_ROPE_NTK && rot > 2) theta *= pow(factor, (double)rot / (double)(rot - 2));
    for (int64_t i = 0; i < rot / 2; i++) {
        double f = pow(theta, -2.0 * (double)i / (double)rot);
        if (scaling == AXHIP_ROPE_LINEAR) f /= factor;
        if (scaling == AXHIP_ROPE_BY_PARTS) {
            double keep = ((double)trained * f / 6.283185307179586 - slow) / (fast - slow);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / factor * (1 - keep);
        }
        host[i] = (float)f;
    }
    return axhip_memcpy_h2d(freq, host, (size_t)(rot / 2) * sizeof(float));
}

extern "C" int axhip_rope_rows(const float *x, int64_t ldx, float *y, int64_t ldy, const int32_t *pos, const float *freq, int64_t rows, int64_t H,
                               int64_t dk, int64_t rot, float amplitude, int layout, int backward) {
    if (int rc = ensure_ready()) return rc;
    if (!x || !y) return fail(AXHIP_ERR_NULL_ARG, "rope_rows: NULL tensor");
    if (int rc = check_heads("rope_rows", rows, H, 0, dk, rot, layout, pos, freq)) return rc;
    if (ldx < H * dk || ldy < H * dk) return fail(AXHIP_ERR_SHAPE, "rope_rows: row pitch must hold H * dk floats");
    if (x == y && ldx != ldy) return fail(AXHIP_ERR_SHAPE, "rope_rows: in place with two pitches");
    if (rows == 0 || H == 0) return AXHIP_OK;
    HeadsArgs p = {};
    p.x = x;
    p.y = y;
    p.pos = pos;
    p.freq = freq;
    p.ldx = ldx;
    p.ldy = ldy;
    p.rows = rows;
    p.heads = p.q_heads = (int)H;
    p.dk = (int)dk;
    p.rot = (int)rot;
    p.amplitude = amplitude;
    p.sign = backward ? -1.0f : 1.0f;
    p.halves = layout == AXHIP_ROPE_HALVES;
    return run_heads<ROTATE>(p, nullptr, nullptr);
}

extern "C" int axhip_qk_norm_rope_fwd(const float *x, int64_t ldx, float *y, int64_t ldy, float *inv_rms, const float *gamma_q, const float *gamma_k,
                                      float eps, const int32_t *pos, const float *freq, int64_t rows, int64_t H, int64_t Hk, int64_t dk, int64_t rot,
                                      float amplitude, int layout) {
    if (int rc = ensure_ready()) return rc;
    if (!x || !y) return fail(AXHIP_ERR_NULL_ARG, "qk_norm_rope_fwd: NULL tensor");
    if (int rc = check_heads("qk_norm_rope_fwd", rows, H, Hk, dk, rot, layout, pos, freq)) return rc;
    if (ldx < (H + Hk) * dk || ldy < (H + Hk) * dk) return fail(AXHIP_ERR_SHAPE, "qk_norm_rope_fwd: row pitch must hold (H + Hk) * dk floats");
    if (x == y && ldx != ldy) return fail(AXHIP_ERR_SHAPE, "qk_norm_rope_fwd: in place with two pitches");
    if (!(eps >= 0)) return fail(AXHIP_ERR_SHAPE, "qk_norm_rope_fwd: eps must not be negative");
    if (rows == 0 || H + Hk == 0) return AXHIP_OK;
    HeadsArgs p = {};
    p.x = x;
    p.y = y;
    p.inv = inv_rms;
    p.gamma_q = gamma_q;
    p.gamma_k = gamma_k;
    p.pos = pos;
    p.freq = freq;
    p.ldx = ldx;
    p.ldy = ldy;
    p.rows = rows;
    p.heads = (int)(H + Hk);
    p.q_heads = (int)H;
    p.dk = (int)dk;
    p.rot = (int)rot;
    p.eps = eps;
    p.amplitude = amplitude;
    p.sign = 1.0f;
    p.halves = layout == AXHIP_ROPE_HALVES;
    return run_heads<NORM>(p, nullptr, nullptr);
}

extern "C" int axhip_qk_norm_rope_bwd(const float *dy, int64_t lddy, const float *x, int64_t ldx, const float *inv_rms, float *dx, int64_t lddx,
                                      const float *gamma_q, const float *gamma_k, float *dgamma_q, float *dgamma_k, const int32_t *pos, const float *freq,
                                      int64_t rows, int64_t H, int64_t Hk, int64_t dk, int64_t rot, float amplitude, int layout) {
    if (int rc = ensure_ready()) return rc;
    if (!dy || !x || !inv_rms || !dx) return fail(AXHIP_ERR_NULL_ARG, "qk_norm_rope_bwd: NULL tensor");
    if (int rc = check_heads("qk_norm_rope_bwd", rows, H, Hk, dk, rot, layout, pos, freq)) return rc;
    if (ldx < (H + Hk) * dk || lddy < (H + Hk) * dk || lddx < (H + Hk) * dk)
        return fail(AXHIP_ERR_SHAPE, "qk_norm_rope_bwd: row pitch must hold (H + Hk) * dk floats");
    if ((dx == dy && lddx != lddy) || (dx == x && lddx != ldx)) return fail(AXHIP_ERR_SHAPE, "qk_norm_rope_bwd: in place with two pitches");
    if (rows == 0 || H + Hk == 0) {
        if (dgamma_q)
            if (int rc = axhip_fill_f32(dgamma_q, 0.0f, dk)) return rc;
        return dgamma_k ? axhip_fill_f32(dgamma_k, 0.0f, dk) : AXHIP_OK;
    }
    HeadsArgs p = {};
    p.x = x;
    p.dy = dy;
    p.y = dx;
    p.inv = const_cast<float *>(inv_rms);        // read only
    p.gamma_q = gamma_q;
    p.gamma_k = gamma_k;
    p.pos = pos;
    p.freq = freq;
    p.ldx = ldx;
    p.lddy = lddy;
    p.ldy = lddx;
    p.rows = rows;
    p.heads = (int)(H + Hk);
    p.q_heads = (int)H;
    p.dk = (int)dk;
    p.rot = (int)rot;
    p.amplitude = amplitude;
    p.sign = -1.0f;
    p.halves = layout == AXHIP_ROPE_HALVES;
    return run_heads<NORM_GRAD>(p, dgamma_q, dgamma_k);
}
