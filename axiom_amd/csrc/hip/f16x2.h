// fp32 products on the f16 matrix core: every operand as the sum of two f16 terms under a power of two of its own.
//
// A row of a head is taken times 2^e so that its largest value lies in [2^14, 2^15), and each value is cut into hi = f16(x) and lo = f16(x - hi): 11 bits each,
// so hi + lo is x to 2^-23 of itself.  A product of two values is formed of three products of terms, hi hi + hi lo + lo hi, added in fp32; lo lo, left out,
// is at most 2^-22 of it.  Half of what six products of bf16 terms cost (bf16x3.h), for one bit of each operand.  The matrix core multiplies f16
// subnormals exactly (measured), so what a value below 2^-17 of its row's largest loses is an absolute 2^-39 of that at most.
// Every row has a power of its own, and not a block: a row of 1e30 that a mask hides would otherwise take the bits of its neighbours.  Where rows are summed over
// (P V), their powers go to the other operand, whose largest so far a running exponent holds.
// Cutting a pair: two products (none where the values come scaled), two conversions of pairs, two mixed multiply-adds, four cycles each.  (Mixed multiply-adds
// that give f16 do without the conversions, but take eight cycles: 41 million instructions instead of 44 in a forward
// pass, and 3 % more cycles.)
// (Sums of products of split operands: Dekker, "A floating-point technique for extending the available precision", 1971.)
#pragma once
#include "common.h"

namespace axhip {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef int v2i32 __attribute__((ext_vector_type(2)));

// Eight values times `up`, as two terms.  (`hi` passes through a register that the compiler cannot see through: it would convert twice, once for
// the pair and once for each value.)
__device__ __forceinline__ void cut_pair(float x, float y, float up, int &first, int &second) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    first = __builtin_bit_cast(int, __builtin_convertvector(v2f{x * up, y * up}, v2h));
    asm("" : "+v"(first));
    const v2h hi = __builtin_bit_cast(v2h, first);
    second = __builtin_bit_cast(int, __builtin_convertvector(v2f{__builtin_fmaf(x, up, -(float)hi[0]), __builtin_fmaf(y, up, -(float)hi[1])}, v2h));
}
__device__ __forceinline__ void cut_halves(const float (&x)[8], float up, v4i (&t)[2]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        int a, b;
        cut_pair(x[e], x[e + 1], up, a, b);
        t[0][e / 2] = a;
        t[1][e / 2] = b;
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

__device__ __forceinline__ float two_to(int e) { return __uint_as_float((unsigned)((e < -126 ? -126 : e) + 127) << 23); }

// Tiles of 16 x 16 and 32 k
__device__ __forceinline__ v4f mfma_cut16(const v4i (&a)[2], const v4i (&b)[2], v4f c) {
    auto one = [&](const v4i &x, const v4i &y) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), c, 0, 0, 0); };
    one(a[1], b[0]);
    one(a[0], b[1]);
    one(a[0], b[0]);
    return c;
}

// What a row whose largest magnitude is `most` is taken times, 2^e, straight from the exponent field E of `most`, which is 2^(E - 127) to twice that: e = 141 - E, at most MOST_UP (rows of
// zeros, and rows below 2^-102, which lose bits); and the factor kept with it, 2^-e.  Products of two cut rows times the factor of the one and then the other's pass 2^128 on the way
// only for results of 2^27 and more.  (Scores so large are off by more than the exponential reaches, and the log-sum-exp that stands against them is.)
constexpr int MOST_UP = 100;
__device__ __forceinline__ float row_up(float most) {
    const unsigned bits = ((127u + 141u) << 23) - (__float_as_uint(most) & 0x7f800000u);
    return __uint_as_float(min(bits, (127u + MOST_UP) << 23));
}
__device__ __forceinline__ float row_factor(float up) { return __uint_as_float((254u << 23) - __float_as_uint(up)); }
// What probabilities (in their exponent) or their rows' factors carry beyond that, so that what small rows are multiplied by does not run out of exponents
constexpr int BIAS = 24;
// Values from 2^78 on get an infinite factor, so that what sees them is formed again.  A probability's reference is the largest of the scores and their values' factors: with a value of 2^x the
// largest probability is 2^-x or more, and one below 2^-126 is taken as nothing.  Below this border 2^24 keys lost like that are less than a rounding of the sum.
constexpr float VALUES_UP = 0x1p64f, VALUES_DOWN = 0x1p-40f;      // a factor times the one and the other: 2^BIAS, past the largest float from 2^78 on
static_assert(VALUES_UP * VALUES_DOWN == 1 << BIAS, "as other factors");

// The largest of each LANES neighbouring lanes' values (4, 8 or 16), in all of them
template <int LANES>
__device__ __forceinline__ float most_of_lanes(float v) {
#define AX_MOVED(ctrl) v = fmaxf(v, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), ctrl, 0xf, 0xf, true)))
    AX_MOVED(0xb1);                              // lane ^ 1, lane ^ 2, then 8 and 16 lanes mirrored
    AX_MOVED(0x4e);
    if (LANES >= 8) AX_MOVED(0x141);
    if (LANES >= 16) AX_MOVED(0x140);
#undef AX_MOVED
    return v;
}

// What an operand may reach, and where a running reference puts the largest so far when it has gone past that: the room between is for others.
constexpr float ROOM = 32768.0f;
constexpr int LARGEST = 10;

// x 2^e for e down to -252, in two steps: the exponential alone gives nothing below 2^-126.  For sums of probabilities, whose references go with the values' factors and may
// lie further apart than that (values of nothing before one of 1e13) though the probabilities do not.
__device__ __forceinline__ float scaled(float x, float e) {
    const float half = __builtin_amdgcn_exp2f(0.5f * e);
    return x * half * half;
}

// A running scale for sums over what has none of its own, a power of two: it starts at 2^MOST_UP and falls when the largest so far, `most`, times it is past ROOM
__device__ __forceinline__ float regrown(float most, float scale) {
    return most * scale > ROOM ? two_to(min(LARGEST - __builtin_amdgcn_frexp_expf(most), MOST_UP)) : scale;
}

// 1.0f that the compiler does not know: times it, a mixed multiply-add is one instruction and not a conversion and a subtraction
__device__ __forceinline__ float hidden_one() {
    float one = 1.0f;
    asm("" : "+s"(one));
    return one;
}
// Eight values that come scaled, as two terms
__device__ __forceinline__ void cut_scaled(const float (&x)[8], float one, v4i (&t)[2]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        typedef float v2f __attribute__((ext_vector_type(2)));
        int hi = __builtin_bit_cast(int, __builtin_convertvector(v2f{x[e], x[e + 1]}, v2h));
        asm("" : "+v"(hi));
        const v2h h = __builtin_bit_cast(v2h, hi);
        t[0][e / 2] = hi;
        t[1][e / 2] = __builtin_bit_cast(int, __builtin_convertvector(v2f{__builtin_fmaf(x[e], one, -(float)h[0]), __builtin_fmaf(x[e + 1], one, -(float)h[1])}, v2h));
    }
}
// Registers 8 s .. 8 s + 7 of a result tile, scaled, as an operand
__device__ __forceinline__ void cut_scaled(const v16f &x, int s, float one, v4i (&t)[2]) {
    const float part[8] = {x[8 * s], x[8 * s + 1], x[8 * s + 2], x[8 * s + 3], x[8 * s + 4], x[8 * s + 5], x[8 * s + 6], x[8 * s + 7]};
    cut_scaled(part, one, t);
}

// Over the four lanes that hold the parts of a row in 16-wide tiles (lane, lane ^ 16, lane ^ 32, lane ^ 48)
template <typename Join>
__device__ __forceinline__ float over_parts(float v, Join join) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = join(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return join(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float most_of_parts(float v) {
    return over_parts(v, [](float a, float b) { return fmaxf(a, b); });
}

// A lane's part of a row as operand terms, whose largest value over all parts is `most`; gives back the row's factor
template <int KS>
__device__ __forceinline__ float cut_row(const float (&x)[KS][8], float most, v4i (&t)[KS][2]) {
    const float up = row_up(most);
#pragma unroll
    for (int s = 0; s < KS; s++) cut_halves(x[s], up, t[s]);
    return row_factor(up);
}
template <int KS>
__device__ __forceinline__ float most_of(const float (&x)[KS][8]) {
    float most = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int e = 0; e < 8; e++) most = fmaxf(most, __builtin_fabsf(x[s][e]));
    return most;
}

// LDS by its address in it
typedef __attribute__((address_space(3))) unsigned char lds_byte;
__device__ __forceinline__ unsigned lds_address(const unsigned char *p) { return (unsigned)(uintptr_t)(const lds_byte *)p; }
__device__ __forceinline__ v4i read_chunk(unsigned at) { return *reinterpret_cast<const __attribute__((address_space(3))) v4i *>(at); }
__device__ __forceinline__ void write_chunk(unsigned at, const v4i &v) { *reinterpret_cast<__attribute__((address_space(3))) v4i *>(at) = v; }
__device__ __forceinline__ void write_float(unsigned at, float v) { *reinterpret_cast<__attribute__((address_space(3))) float *>(at) = v; }

// Four rows of one column each from LDS: lane l of a group of 16 lanes gives the address of four columns of one row (rows go with l / 4, columns with
// l % 4) and gets column l of the four rows.
__device__ __forceinline__ v2i32 read_columns(unsigned at) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(v2i32, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) v4s *>(at)));
}

}  // namespace axhip
