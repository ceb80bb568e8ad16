// fp32 products on the f16 matrix core: every operand as the sum of two f16 terms under a power of two of its own.
//
// A group of values (a row, or eight rows, of a head) is taken times 2^e so that its largest lies in [2^14, 2^15), and each is cut into hi = f16(x) and
// lo = f16(x - hi): 11 bits each, so hi + lo is x to 2^-23 of itself.  A product of two values is formed of three products of terms, hi hi + hi lo + lo hi,
// added in fp32; lo lo, left out, is at most 2^-22 of it.  Half of what six products of bf16 terms cost (bf16x3.h), for one bit of each operand: the matrix core
// multiplies f16 subnormals exactly (measured), so what a value below 2^-17 of its group's largest loses is an absolute 2^-40 of that.
// Cutting a pair: two products, two conversions of pairs, two mixed multiply-adds.
// (Sums of products of split operands: Dekker, "A floating-point technique for extending the available precision", 1971.)
#pragma once
#include "common.h"

namespace axhip {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef int v2i32 __attribute__((ext_vector_type(2)));

// N values (4 or 8) times `up`, as two terms
template <int N> using Half = std::conditional_t<N == 8, v4i, v2i32>;
template <int N>
__device__ __forceinline__ void cut_halves(const float (&x)[N], float up, Half<N> (&t)[2]) {
    typedef float v2f __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const v2h hi = __builtin_convertvector(v2f{x[e] * up, x[e + 1] * up}, v2h);
        const float ra = __builtin_fmaf(x[e], up, -(float)hi[0]), rb = __builtin_fmaf(x[e + 1], up, -(float)hi[1]);
        const v2h lo = __builtin_convertvector(v2f{ra, rb}, v2h);
        t[0][e / 2] = __builtin_bit_cast(int, hi);
        t[1][e / 2] = __builtin_bit_cast(int, lo);
    }
}

__device__ __forceinline__ v16f mfma_halves(const v4i &a, const v4i &b, const v16f &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// c + a b of terms, the small products first
__device__ __forceinline__ v16f mfma_cut(const v4i (&a)[2], const v4i (&b)[2], v16f c) {
    c = mfma_halves(a[1], b[0], c);
    c = mfma_halves(a[0], b[1], c);
    return mfma_halves(a[0], b[0], c);
}

// The exponent e of a group whose largest magnitude is `most`.  At most 120, which a group of zeros gets too, so that 2^e and 2^-e are floats.
constexpr int MOST_UP = 120;
__device__ __forceinline__ int up_of(float most) {
    const int e = 15 - __builtin_amdgcn_frexp_expf(most);
    return most == 0.0f || e > MOST_UP ? MOST_UP : e;
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((unsigned)((e < -126 ? -126 : e) + 127) << 23); }

// The largest of the 64 lanes' values, in every lane
__device__ __forceinline__ float most_of_wave(float v) {
#define AX_ROTATED(ctrl) v = fmaxf(v, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), ctrl, 0xf, 0xf, true)))
    AX_ROTATED(0x128);                           // rotations by 8, 4, 2 and 1 within each row of 16 lanes
    AX_ROTATED(0x124);
    AX_ROTATED(0x122);
    AX_ROTATED(0x121);
#undef AX_ROTATED
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const unsigned w = __float_as_uint(v);
    const auto h = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// Four rows of one column each from LDS: lane l of a group of 16 lanes gives the address of four columns of one row (rows go with l / 4, columns with
// l % 4) and gets column l of the four rows.
__device__ __forceinline__ v2i32 read_columns(const unsigned char *at) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(v2i32, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)at));
}

}  // namespace axhip
