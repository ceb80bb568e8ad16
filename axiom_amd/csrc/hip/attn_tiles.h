// Blocks of rows of a head in LDS as two f16 terms, for the matrix kernels of attention under score rules.
#pragma once
#include "attn_rules.h"
#include "f16x2.h"

namespace axhip {

// A block of ROWS rows of DK columns: two planes of terms, rows of 2 DK bytes whose 16-byte chunks are exchanged by row, so that both ways
// of reading it touch every bank once: 16 lanes with one chunk of 16 rows (operands whose rows are these rows), and 32 lanes with four
// columns of four rows each (read_columns: operands whose rows are these columns).
template <int DK, int ROWS>
struct Block {
    static_assert(DK == 32 || DK == 64 || DK == 96 || DK == 128, "head dimension");
    static constexpr int PITCH = DK * 2, PLANE = ROWS * PITCH, BYTES = 2 * PLANE;
    __device__ static unsigned at(int row, int chunk) {
        const int key = DK == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : DK == 64 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : (row >> 2) & 3;
        return (unsigned)(row * PITCH + ((chunk ^ key) << 4));
    }
    // rows r0 .. r0 + 31 as the rows of an operand, columns 16 ks + 8 * half ..
    __device__ static v4i rows(const unsigned char *base, int r0, int ks, int lane, int term) {
        return *reinterpret_cast<const v4i *>(base + at(r0 + (lane & 31), 2 * ks + (lane >> 5)) + term * PLANE);
    }
    // columns 32 d .. 32 d + 31 as the rows of an operand; its eight k are rows r0 + 4 * half + 0..3 and 8 more on: those that registers 8 s .. 8 s + 7
    // of a result tile hold
    __device__ static v4i columns(const unsigned char *base, int r0, int d, int lane, int term) {
        const int l = lane & 15, row = r0 + 4 * (lane >> 5) + (l >> 2), chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((l & 3) >> 1);
        const v2i32 a = read_columns(base + at(row, chunk) + 8 * (l & 1) + term * PLANE), b = read_columns(base + at(row + 8, chunk) + 8 * (l & 1) + term * PLANE);
        return v4i{a[0], a[1], b[0], b[1]};
    }
};

// How the waves of a workgroup bring a block from memory: wave w rows RPW w .. RPW w + RPW - 1, a lane PIECES pieces of E columns of a row.
template <int DK, int ROWS, int WAVES>
struct Stage {
    static constexpr int RPW = ROWS / WAVES;
    static constexpr int E = RPW * DK % 512 == 0 ? 8 : 4;
    static constexpr int PIECES = RPW * DK / (64 * E);
    static_assert(RPW % 8 == 0 && PIECES * 64 * E == RPW * DK, "a block divides over the lanes");
    using B = Block<DK, ROWS>;
    float x[PIECES][E];
    // row r of the block is at base + min(r, last) * pitch; columns from dk on are zero
    __device__ __forceinline__ void load(const float *base, int64_t pitch, int last, int wave, int lane, int dk) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int q = lane + 64 * i, row = wave * RPW + q / (DK / E), col = q % (DK / E) * E;
            const float *p = base + (int64_t)(row < last ? row : last) * pitch + col;
#pragma unroll
            for (int h = 0; h < E / 4; h++) {
                v4f a = {0.f, 0.f, 0.f, 0.f};
                if (dk == DK || col + 4 * h < dk) a = *reinterpret_cast<const v4f *>(p + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; e++) x[i][4 * h + e] = a[e];
            }
        }
    }
    // to LDS, cut; returns the exponent that this wave's rows were taken up by
    __device__ __forceinline__ int put(unsigned char *block, int wave, int lane, float factor) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (factor != 1.0f) x[i][e] *= factor;
                most = fmaxf(most, __builtin_fabsf(x[i][e]));
            }
        const int up = up_of(most_of_wave(most));
        const float by = two_to(up);
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int q = lane + 64 * i, row = wave * RPW + q / (DK / E), col = q % (DK / E) * E;
            Half<E> t[2];
            cut_halves(x[i], by, t);
            unsigned char *to = block + B::at(row, col / 8) + col % 8 * 2;
            *reinterpret_cast<Half<E> *>(to) = t[0];
            *reinterpret_cast<Half<E> *>(to + B::PLANE) = t[1];
        }
        return up;
    }
};

// The documents of 32 keys (or rows): the lowest and highest id there, -1 and below not counted; `low` is ~lowest where some are not
// counted, so that one document all over is low == high.  No id at all: (INT_MAX, -1).
struct DocRange {
    int low, high;
    __device__ bool meets(int from, int to) const { return high >= from && (low < 0 ? ~low : low) <= to; }
};

}  // namespace axhip
