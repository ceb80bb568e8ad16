// Rows of keys and values into a paged cache in few bits, and back.
//
// One pass each.  Writing: a wave takes a row of both arrays, LANES lanes a head of it, eight columns a lane (two 16-byte accesses); the largest magnitude is an integer maximum of the bits over
// the lanes of a head (of a group of 32 columns, four lanes), which infinities and NaNs pass.  Many rows are HBM-bound, AHEAD heads of a lane group under way at once; few rows are five trips to
// memory one after the other (arguments, the row's sequence, its length, the page, the row), with a head a lane group.
// 14768 rows of 8 heads of 128 into 4 bits 33 us, 4.1 TB/s, and back 25, 5.4 TB/s; into f16 48, 3.8 TB/s, and back 29, 6.2 TB/s, of 80 32, 3.6 TB/s (six of sixteen lanes hold nothing), and back 22; 16 rows into int8 3.3 to
// 3.7 (5.6 with four heads a lane group).
#include "kv_pages.h"

namespace {
using namespace axhip;

constexpr int WAVES = 4;
constexpr int64_t GRID_MOST = int64_t(1) << 22;  // workgroups of a launch: a grid holds fewer than 2^32 threads

typedef unsigned v2u __attribute__((ext_vector_type(2)));

struct RowsArgs {
    KvPages pages;
    float *k, *v;                                // of the caller
    int64_t ldk, ldv, first;                     // first: the launch's first row
    int per_row;                                 // waves to a row
};

// The largest of each LANES neighbouring lanes' bits, in all of them
template <int LANES>
__device__ __forceinline__ unsigned most_bits(unsigned v) {
#define AX_MOVED(ctrl) v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, ctrl, 0xf, 0xf, true))
    AX_MOVED(0xb1);                              // lane ^ 1, lane ^ 2, then 8 and 16 lanes mirrored
    AX_MOVED(0x4e);
    if (LANES >= 8) AX_MOVED(0x141);
    if (LANES >= 16) AX_MOVED(0x140);
#undef AX_MOVED
    return v;
}

// e of top = m 2^e, 1 <= m < 2, from its bits; -127 and less for what is below the normal numbers
__device__ __forceinline__ int exponent_of(unsigned bits) {
    const unsigned field = bits >> 23;
    return field ? (int)field - 127 : bits ? -118 - (int)__builtin_clz(bits) : -1000;
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// n nearest to x / s, ties to even, of the exact quotient; inv is about 1 / s.  x inv is off by less than 2^-15 here, so that n is off by one at most, and only next to a half; there x - n s is a float.
__device__ __forceinline__ int nearest(float x, float s, float inv) {
    float n = rintf(x * inv);
    const float twice = 2.0f * __builtin_fmaf(-n, s, x);
    const bool odd = ((int)n & 1) != 0;
    if (twice > s || (twice == s && odd)) n += 1.0f;
    if (twice < -s || (twice == -s && odd)) n -= 1.0f;
    return (int)fminf(fmaxf(n, -127.0f), 127.0f);
}

template <int TYPE, int LANES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) k_kv_write(RowsArgs a) {
    const KvPages &p = a.pages;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane % LANES;
    const unsigned item = blockIdx.x * WAVES + wave, row = item / (unsigned)a.per_row;
    const int64_t t = a.first + row;
    if (t >= p.T) return;
    const int task0 = (int)(item - row * (unsigned)a.per_row) * (AHEAD * 64 / LANES) + lane / LANES, tasks = 2 * p.heads;
    v4f x[AHEAD][2];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
        const int task = task0 + i * (64 / LANES);
        const bool of_v = task >= p.heads;
        const float *from = (of_v ? a.v + t * a.ldv : a.k + t * a.ldk) + (int64_t)(of_v ? task - p.heads : task) * p.dk + 8 * c;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            x[i][h] = v4f{0.f, 0.f, 0.f, 0.f};
            if (task < tasks && 8 * c + 4 * h < p.dk) x[i][h] = *reinterpret_cast<const v4f *>(from + 4 * h);
        }
    }
    const int b = p.first ? kv_find(p, lane, [&](int, int first) { return first <= t; }) : (int)((unsigned)t / (unsigned)p.Sq);
    if (b >= p.B) return;
    const KvSeq s = kv_seq(p, b);
    const int i0 = (int)t - s.first, pos = s.len - s.n + i0;
    if (i0 < 0 || i0 >= s.n || pos < 0) return;
    const int page = kv_page(p, b, pos);
    if (page < 0) return;
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
        const int task = task0 + i * (64 / LANES);
        const bool of_v = task >= p.heads;
        const int head = of_v ? task - p.heads : task;
        unsigned char *const to = (of_v ? p.v : p.k) + kv_row_at(p, page, head, pos), *const scales = (of_v ? p.v_scale : p.k_scale) + kv_scale_at(p, page, head, pos);
        float y[8];
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = x[i][e / 4][e % 4];
            top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
        }
        top = most_bits<(TYPE == AXHIP_KV_MX4 ? 4 : LANES)>(top);
        const bool finite = top < 0x7f800000u;
        if (!finite)
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = 0.0f;
        const bool live = task < tasks;
        if constexpr (TYPE == AXHIP_KV_F16) {
            const int e2 = max(exponent_of(top) - 14, KV_LEAST);
            const float up = power(-e2);
            v4i n;
#pragma unroll
            for (int e = 0; e < 4; e++) n[e] = __builtin_bit_cast(int, __builtin_convertvector(kv_float2{y[2 * e] * up, y[2 * e + 1] * up}, kv_half2));
            if (live && 16 * c < p.row_bytes) *reinterpret_cast<v4i *>(to + 16 * c) = n;
            if (live && c == 0) *reinterpret_cast<float *>(scales) = finite ? power(e2) : NAN;
        } else if constexpr (TYPE == AXHIP_KV_I8) {
            const float scale = finite ? fmaxf(__uint_as_float(top) / 127.0f, power(KV_LEAST)) : NAN, inv = finite ? 1.0f / scale : 0.0f;
            uint64_t n = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) n |= (uint64_t)(uint8_t)(finite ? nearest(y[e], scale, inv) : 0) << (8 * e);
            if (live && 8 * c < p.row_bytes) *reinterpret_cast<uint64_t *>(to + 8 * c) = n;
            if (live && c == 0) *reinterpret_cast<float *>(scales) = scale;
        } else {
            const int e2 = max(exponent_of(top) - 2, -127);
            const float up = power(-e2);
            unsigned n = 0;
            n = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(n, y[0] * up, y[1] * up, 1.0f, 0);
            n = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(n, y[2] * up, y[3] * up, 1.0f, 1);
            n = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(n, y[4] * up, y[5] * up, 1.0f, 2);
            n = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(n, y[6] * up, y[7] * up, 1.0f, 3);
            if (live && 4 * c < p.row_bytes) *reinterpret_cast<unsigned *>(to + 4 * c) = n;
            unsigned code = c % 4 == 0 && 8 * c < p.dk ? (finite ? (unsigned)(e2 + 127) : 255u) << (8 * (c / 4)) : 0u;
            if (LANES >= 8) code |= (unsigned)__shfl_xor((int)code, 4, 64);
            if (LANES >= 16) code |= (unsigned)__shfl_xor((int)code, 8, 64);
            if (live && c == 0) *reinterpret_cast<unsigned *>(scales) = code;
        }
    }
}

// Here a lane has four columns, so that the stores of neighbours are: with eight, in two of 16 bytes each, 8 sequences of up to 8192 rows of 8 heads of 80 in f16 came back in 102 us (4.0 TB/s), so in 83.
template <int TYPE, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) k_kv_read(RowsArgs a) {
    const KvPages &p = a.pages;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned item = blockIdx.x * WAVES + wave, row = item / (unsigned)a.per_row;
    const int64_t t = a.first + row;
    if (t >= p.T) return;
    const int b = p.first ? kv_find(p, lane, [&](int, int first) { return first <= t; }) : (int)((unsigned)t / (unsigned)p.Sq);
    if (b >= p.B) return;
    const KvSeq s = kv_seq(p, b);
    const int i0 = (int)t - s.first, pos = s.len - s.n + i0;
    if (i0 < 0 || i0 >= s.n || pos < 0) return;
    const int page = kv_page(p, b, pos);
    if (page < 0) return;
    const unsigned quads = (unsigned)p.dk / 4, all = (unsigned)p.heads * quads, unit0 = (item - row * (unsigned)a.per_row) * 64 * AHEAD + lane;
    const uint64_t row_at = kv_row_at(p, page, 0, pos), scale_at = kv_scale_at(p, page, 0, pos);
    const unsigned head_rows = (unsigned)p.row_bytes << p.shift, head_scales = 4u << p.shift;
    v2u n[AHEAD];
    unsigned scale[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
        const unsigned u = unit0 + 64 * i, of = u < all ? u : u - all;
        if (u >= 2 * all) break;
        const unsigned head = of / quads, c = of - head * quads;
        const unsigned char *from = (u < all ? p.k : p.v) + row_at + (uint64_t)head * head_rows;
        scale[i] = *reinterpret_cast<const unsigned *>((u < all ? p.k_scale : p.v_scale) + scale_at + (uint64_t)head * head_scales);
        if constexpr (TYPE == AXHIP_KV_F16) n[i] = *reinterpret_cast<const v2u *>(from + 8 * c);
        if constexpr (TYPE == AXHIP_KV_I8) n[i][0] = *reinterpret_cast<const unsigned *>(from + 4 * c);
        if constexpr (TYPE == AXHIP_KV_MX4) n[i][0] = *reinterpret_cast<const uint16_t *>(from + 2 * c);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
        const unsigned u = unit0 + 64 * i, of = u < all ? u : u - all;
        if (u >= 2 * all) break;
        const unsigned head = of / quads, c = of - head * quads;
        v4f x;
        if constexpr (TYPE == AXHIP_KV_F16) {
            const unsigned lo = n[i][0], hi = n[i][1];
            const kv_half2 two[2] = {__builtin_bit_cast(kv_half2, lo), __builtin_bit_cast(kv_half2, hi)};
            x = v4f{(float)two[0][0], (float)two[0][1], (float)two[1][0], (float)two[1][1]} * __uint_as_float(scale[i]);
        }
        if constexpr (TYPE == AXHIP_KV_I8) {
            const int four = (int)n[i][0];
            x = v4f{(float)(int8_t)four, (float)(int8_t)(four >> 8), (float)(int8_t)(four >> 16), (float)(four >> 24)} * __uint_as_float(scale[i]);
        }
        if constexpr (TYPE == AXHIP_KV_MX4) {
            const unsigned four = n[i][0];
            const kv_float2 two[2] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, 1.0f, 1)};
            x = v4f{two[0][0], two[0][1], two[1][0], two[1][1]} * kv_group_scale((scale[i] >> (8 * (c / 8))) & 255);
        }
        *reinterpret_cast<v4f *>((u < all ? a.k + t * a.ldk : a.v + t * a.ldv) + 4 * of) = x;
    }
}

int rows_arguments(const char *who, RowsArgs &a, const axhip_kv_cache *cache, const float *K, int64_t ldk, const float *V, int64_t ldv, const int32_t *first,
                   const int32_t *lens, int64_t B, int64_t T, int64_t Sq) {
    if (int rc = ensure_ready()) return rc;
    if (int rc = kv_arguments(who, a.pages, cache, first, lens, B, T, Sq)) return rc;
    if (!K || !V) return fail(AXHIP_ERR_NULL_ARG, "%s: NULL tensor", who);
    for (int64_t ld : {ldk, ldv})
        if (ld < cache->heads * cache->dk || ld % 4 != 0 || ld > (1 << 22))
            return fail(AXHIP_ERR_SHAPE, "%s: row pitch must hold the heads, be a multiple of 4 and at most 2^22 floats", who);
    if ((((uintptr_t)K | (uintptr_t)V) & 15) != 0) return fail(AXHIP_ERR_SHAPE, "%s: tensors must be 16-byte aligned", who);
    a.k = const_cast<float *>(K);
    a.v = const_cast<float *>(V);
    a.ldk = ldk;
    a.ldv = ldv;
    return AXHIP_OK;
}

// units: of which a wave takes 64 at a time; AHEAD at a time where there are rows enough for all CUs, one where there are few
template <typename Launch>
int launch_rows(RowsArgs &a, const char *who, int64_t units, Launch launch) {
    const int64_t waves = (units + 63) / 64;
    const bool many = waves * a.pages.T >= 16 * (int64_t)cu_count();
    a.per_row = (int)(many ? (waves + 3) / 4 : waves);
    const int64_t at_once = GRID_MOST * WAVES / a.per_row;       // rows a launch; (a row has at most 2^20 waves)
    for (a.first = 0; a.first < a.pages.T; a.first += at_once) {
        const int64_t rows = a.pages.T - a.first < at_once ? a.pages.T - a.first : at_once;
        const dim3 grid((unsigned)((rows * a.per_row + WAVES - 1) / WAVES));
        if (many) launch(std::integral_constant<int, 4>(), grid);
        else launch(std::integral_constant<int, 1>(), grid);
        if (int rc = check_launch(who)) return rc;
    }
    return AXHIP_OK;
}

template <int LANES, int AHEAD>
void launch_write(int type, const RowsArgs &a, dim3 grid) {
    if (type == AXHIP_KV_F16) hipLaunchKernelGGL((k_kv_write<AXHIP_KV_F16, LANES, AHEAD>), grid, dim3(64 * WAVES), 0, kStream, a);
    else if (type == AXHIP_KV_I8) hipLaunchKernelGGL((k_kv_write<AXHIP_KV_I8, LANES, AHEAD>), grid, dim3(64 * WAVES), 0, kStream, a);
    else hipLaunchKernelGGL((k_kv_write<AXHIP_KV_MX4, LANES, AHEAD>), grid, dim3(64 * WAVES), 0, kStream, a);
}

}  // namespace

namespace axhip {

int kv_arguments(const char *who, KvPages &a, const axhip_kv_cache *cache, const int32_t *first, const int32_t *lens, int64_t B, int64_t T, int64_t Sq) {
    if (!cache) return fail(AXHIP_ERR_NULL_ARG, "%s: NULL cache", who);
    const axhip_kv_cache &c = *cache;
    if (c.type < AXHIP_KV_F16 || c.type > AXHIP_KV_MX4) return fail(AXHIP_ERR_SHAPE, "%s: no such type of cache", who);
    if (c.dk < 4 || c.dk > 128 || c.dk % 4 != 0) return fail(AXHIP_ERR_NOT_IMPLEMENTED, "%s: head size %lld (multiples of 4 up to 128 only)", who, (long long)c.dk);
    if (c.page_rows < 1 || c.page_rows > (1 << 16) || (c.page_rows & (c.page_rows - 1)) != 0)
        return fail(AXHIP_ERR_SHAPE, "%s: rows of a page must be a power of two up to 2^16", who);
    if (c.heads < 1 || c.heads > (1 << 20)) return fail(AXHIP_ERR_SHAPE, "%s: 1 to 2^20 heads of keys", who);
    if (c.pages < 0 || c.pages > 0x7fffffff || c.pages > (int64_t(1) << 40) / (c.heads * c.page_rows)) return fail(AXHIP_ERR_SHAPE, "%s: bad count of pages", who);
    const int64_t row_bytes = axhip_kv_row_bytes(c.type, c.dk);
    if (c.heads * c.page_rows > 0xffffffff / row_bytes) return fail(AXHIP_ERR_SHAPE, "%s: a page of keys must be below 4 GiB", who);
    constexpr int64_t LONG = 1 << 24;
    if (B < 0 || B > 0x7fffff || T < 0 || T > LONG || Sq < 0 || Sq > LONG) return fail(AXHIP_ERR_SHAPE, "%s: bad extent", who);
    if (!first && T != B * Sq) return fail(AXHIP_ERR_SHAPE, "%s: without `first` there are B * Sq rows", who);
    if (c.table_ld < 0 || c.table_ld > (int64_t(1) << 40)) return fail(AXHIP_ERR_SHAPE, "%s: bad table pitch", who);
    if (B > 0 && T > 0 && (!lens || !c.table || !c.k || !c.v || !c.k_scale || !c.v_scale)) return fail(AXHIP_ERR_NULL_ARG, "%s: NULL cache or lengths", who);
    if ((((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.k_scale | (uintptr_t)c.v_scale) & 15) != 0) return fail(AXHIP_ERR_SHAPE, "%s: caches must be 16-byte aligned", who);
    a = {};
    a.k = static_cast<unsigned char *>(c.k);
    a.v = static_cast<unsigned char *>(c.v);
    a.k_scale = static_cast<unsigned char *>(c.k_scale);
    a.v_scale = static_cast<unsigned char *>(c.v_scale);
    a.table = c.table;
    a.first = first;
    a.lens = lens;
    a.table_ld = c.table_ld;
    a.pages = c.pages;
    a.heads = (int)c.heads;
    a.dk = (int)c.dk;
    a.shift = __builtin_ctz((unsigned)c.page_rows);
    a.row_bytes = (int)row_bytes;
    a.page_bytes = (uint32_t)(c.heads * c.page_rows * row_bytes);
    a.page_scales = (uint32_t)(c.heads * c.page_rows * 4);
    a.B = (int)B;
    a.T = (int)T;
    a.Sq = (int)(first && T < Sq ? T : Sq);          // (a bound: no sequence has more rows than there are)
    a.room = (int)(c.table_ld < LONG >> a.shift ? c.table_ld << a.shift : LONG);
    return AXHIP_OK;
}

}  // namespace axhip

extern "C" int64_t axhip_kv_row_bytes(int type, int64_t dk) {
    if (type < AXHIP_KV_F16 || type > AXHIP_KV_MX4 || dk < 4 || dk > 128 || dk % 4 != 0) return 0;
    const int64_t bytes = type == AXHIP_KV_F16 ? 2 * dk : type == AXHIP_KV_I8 ? dk : dk / 2;
    return (bytes + 15) / 16 * 16;
}

extern "C" int axhip_kv_write(const axhip_kv_cache *cache, const float *K, int64_t ldk, const float *V, int64_t ldv, const int32_t *first, const int32_t *lens, int64_t B,
                              int64_t T, int64_t Sq) {
    RowsArgs a = {};
    if (int rc = rows_arguments("kv_write", a, cache, K, ldk, V, ldv, first, lens, B, T, Sq)) return rc;
    if (B == 0 || T == 0 || Sq == 0) return AXHIP_OK;
    const int lanes = a.pages.dk <= 32 ? 4 : a.pages.dk <= 64 ? 8 : 16;
    return launch_rows(a, "kv_write", 2 * cache->heads * lanes, [&](auto ahead, dim3 grid) {
        constexpr int AHEAD = decltype(ahead)::value;
        if (lanes == 4) launch_write<4, AHEAD>(cache->type, a, grid);
        else if (lanes == 8) launch_write<8, AHEAD>(cache->type, a, grid);
        else launch_write<16, AHEAD>(cache->type, a, grid);
    });
}

extern "C" int axhip_kv_read(const axhip_kv_cache *cache, float *K, int64_t ldk, float *V, int64_t ldv, const int32_t *first, const int32_t *lens, int64_t B, int64_t T,
                             int64_t Sq) {
    RowsArgs a = {};
    if (int rc = rows_arguments("kv_read", a, cache, K, ldk, V, ldv, first, lens, B, T, Sq)) return rc;
    if (B == 0 || T == 0 || Sq == 0) return AXHIP_OK;
    return launch_rows(a, "kv_read", 2 * cache->heads * (cache->dk / 4), [&](auto ahead, dim3 grid) {
        constexpr int AHEAD = decltype(ahead)::value;
        if (cache->type == AXHIP_KV_F16) hipLaunchKernelGGL((k_kv_read<AXHIP_KV_F16, AHEAD>), grid, dim3(64 * WAVES), 0, kStream, a);
        else if (cache->type == AXHIP_KV_I8) hipLaunchKernelGGL((k_kv_read<AXHIP_KV_I8, AHEAD>), grid, dim3(64 * WAVES), 0, kStream, a);
        else hipLaunchKernelGGL((k_kv_read<AXHIP_KV_MX4, AHEAD>), grid, dim3(64 * WAVES), 0, kStream, a);
    });
}
