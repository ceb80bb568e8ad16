// A paged cache of keys and values in few bits: where its rows are, and what their bytes stand for (axhip_kv_write, axhip_kv_read, axhip_attn_paged).
#pragma once
#include "common.h"

namespace axhip {

struct KvPages {
    unsigned char *k, *v, *k_scale, *v_scale;
    const int32_t *table, *first, *lens;
    int64_t table_ld, pages;
    int heads, dk, shift, row_bytes;             // page_rows is 2^shift
    uint32_t page_bytes, page_scales;            // of a page of k or v and of its scales
    int B, T, Sq, room;                          // room: the most positions that a sequence is taken to have
};

// Checks that the entry points share, and the arguments that all pass on
int kv_arguments(const char *who, KvPages &a, const axhip_kv_cache *cache, const int32_t *first, const int32_t *lens, int64_t B, int64_t T, int64_t Sq);

// Scales of rows, and of groups, are no less than this: what is below loses bits
constexpr int KV_LEAST = -100;

// The new rows of a sequence: rows first .. first + n - 1, of which row i is at position len - n + i
struct KvSeq {
    int first, n, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvPages &a, int b) {
    KvSeq s;
    if (a.first) {
        s.first = min(max(a.first[b], 0), a.T);
        s.n = min(max(min(max(a.first[b + 1], 0), a.T) - s.first, 0), a.Sq);
    } else {
        s.first = b * a.Sq;
        s.n = a.Sq;
    }
    s.len = min(max(a.lens[b], 0), a.room);
    return s;
}

// How many of first[1 .. B] the predicate holds for, which holds for the first of them and no longer from some place on: the sequence that a row, or a tile, belongs to.  By all
// lanes of a wave together, 64 places at a time: one trip to memory for up to 64 sequences, two for 4096.
template <typename Before>
__device__ __forceinline__ int kv_find(const KvPages &a, int lane, Before before) {
    int low = 0, high = a.B;                         // it holds for `low`, and for none past `high`
    while (low < high) {
        const int step = (high - low + 63) / 64, k = min(low + (lane + 1) * step, high);
        const int here = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before(k, min(max(a.first[k], 0), a.T))));
        const int from = low;
        low = min(from + here * step, high);
        if (here < 64) high = max(min(from + (here + 1) * step, high) - 1, low);
    }
    return low;
}

// The table's entry for a position below a sequence's length, and whether it is a page: apart, so that entries can be under way while nothing waits for them
__device__ __forceinline__ int kv_entry(const KvPages &a, int b, int pos) { return a.table[(int64_t)b * a.table_ld + (pos >> a.shift)]; }
__device__ __forceinline__ bool kv_is_page(const KvPages &a, int entry) { return (unsigned)entry < (unsigned)a.pages; }
__device__ __forceinline__ int kv_page(const KvPages &a, int b, int pos) {
    const int entry = kv_entry(a, b, pos);
    return kv_is_page(a, entry) ? entry : -1;
}
// Where a row of a head is in k and v, and its scale in k_scale and v_scale, in bytes.  (A page is below 4 GiB, its rows fewer than 2^24 / 256.)
__device__ __forceinline__ uint64_t kv_row_at(const KvPages &a, int page, int head, int pos) {
    const unsigned in_page = (unsigned)pos & ((1u << a.shift) - 1);
    return (uint64_t)(unsigned)page * a.page_bytes + ((unsigned)head << a.shift) * (unsigned)a.row_bytes + __umul24(in_page, (unsigned)a.row_bytes);
}
__device__ __forceinline__ uint64_t kv_scale_at(const KvPages &a, int page, int head, int pos) {
    const unsigned in_page = (unsigned)pos & ((1u << a.shift) - 1);
    return (uint64_t)(unsigned)page * a.page_scales + (((unsigned)head << a.shift) + in_page) * 4;
}

typedef _Float16 kv_half2 __attribute__((ext_vector_type(2)));
typedef float kv_float2 __attribute__((ext_vector_type(2)));

// 2^(code - 127), NaN for 255
__device__ __forceinline__ float kv_group_scale(unsigned code) {
    return __uint_as_float(code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23);
}

// Four int8 as two pairs of f16: with the sign bit turned over, a byte n + 128 in the low bits of 1024 is 1152 + n.
__device__ __forceinline__ void kv_bytes(unsigned four, int &first, int &second) {
    const unsigned u = four ^ 0x80808080u;
    const kv_half2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    first = __builtin_bit_cast(int, __builtin_bit_cast(kv_half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
    second = __builtin_bit_cast(int, __builtin_bit_cast(kv_half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
}
// Eight 4-bit values times a power of two as four pairs of f16
__device__ __forceinline__ v4i kv_nibbles(unsigned eight, float scale) {
    return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 0)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 1)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 2)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(eight, scale, 3))};
}

// Eight columns of a row from column 8 c on, in fp32
template <int TYPE>
__device__ __forceinline__ void kv_eight(const unsigned char *row, unsigned scale, int c, float (&x)[8]) {
    if constexpr (TYPE == AXHIP_KV_F16) {
        const v4i n = *reinterpret_cast<const v4i *>(row + 16 * c);
        const float s = __uint_as_float(scale);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int pair = n[e];                // (a bit cast of an element itself takes the first one)
            const kv_half2 two = __builtin_bit_cast(kv_half2, pair);
            x[2 * e] = (float)two[0] * s;
            x[2 * e + 1] = (float)two[1] * s;
        }
    } else if constexpr (TYPE == AXHIP_KV_I8) {
        const int64_t n = *reinterpret_cast<const int64_t *>(row + 8 * c);
        const float s = __uint_as_float(scale);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)(int)(int8_t)(n >> (8 * e)) * s;
    } else {
        const unsigned n = *reinterpret_cast<const unsigned *>(row + 4 * c);
        const float s = kv_group_scale((scale >> (8 * (c / 4))) & 255);
        const kv_float2 two[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(n, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(n, 1.0f, 1),
                                  __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(n, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(n, 1.0f, 3)};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = two[e][0] * s;
            x[2 * e + 1] = two[e][1] * s;
        }
    }
}

}  // namespace axhip
