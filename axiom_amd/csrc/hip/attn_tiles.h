// Blocks of rows of a head in LDS as two f16 terms, for the matrix kernels of attention under score rules.
#pragma once
#include "attn_rules.h"
#include "f16x2.h"

namespace axhip {

// A block of ROWS rows of DK columns: two planes of terms, rows of 2 DK bytes whose 16-byte chunks are exchanged by row, so that both ways
// of reading it touch every bank once: 16 lanes with one chunk of 16 rows (operands whose rows are these rows), and 32 lanes with 32 columns of four rows, or 16
// columns of eight (read_columns: operands whose rows are these columns).
template <int DK, int ROWS>
struct Block {
    static_assert(DK == 32 || DK == 64 || DK == 96 || DK == 128, "head dimension");
    static constexpr int PITCH = DK * 2, PLANE = ROWS * PITCH, BYTES = 2 * PLANE;
    __device__ static constexpr int low_key(int row) { return ((row >> 2 ^ row >> 3) & 1) << 1 | (row >> 3 & 1); }
    __device__ static unsigned at(int row, int chunk) {
        const int key = low_key(row) | (DK == 128 ? (row & 3) << 2 : DK == 64 ? ((row >> 1) & 1) << 2 : 0);
        return (unsigned)(row * PITCH + ((chunk ^ key) << 4));
    }
    // A lane's place for rows(): row (lane & 31), chunk (lane >> 5); and for columns(): see read_columns.  Other rows and chunks are a distance and an exchange
    // of bits away (the bits of MASK are those that rows leave free), so a lane holds two addresses and not one for every fragment.
    static constexpr unsigned MASK = DK == 96 ? 63 : PITCH - 1;
    __device__ static unsigned row_place(int lane) { return at(lane & 31, lane >> 5); }
    __device__ static unsigned column_place(int lane) {
        const int l = lane & 15;
        return at(4 * (lane >> 5) + (l >> 2), 2 * ((lane >> 4) & 1) + ((l & 3) >> 1)) + 8 * (l & 1);
    }
    __device__ static unsigned moved(unsigned place, unsigned by) { return (place ^ (by & MASK)) + (by & ~MASK); }
    // `place` with the block's address added (a multiple of 256, which leaves the bits of MASK free).
    // rows r0 .. r0 + 31 as the rows of an operand, columns 16 k + 8 * half ..
    __device__ static v4i rows(unsigned place, int k, int term) { return read_chunk(moved(place, 32 * k) + term * PLANE); }
    // columns 32 d .. 32 d + 31 as the rows of an operand; its eight k are rows r0 + 4 * half + 0..3 and 8 more on (r0 a multiple of 16): those that registers
    // 8 s .. 8 s + 7 of a result tile hold
    __device__ static v4i columns(unsigned place, int r0, int d, int term) {
        const unsigned near = moved(place, 64 * d);
        const v2i32 a = read_columns(near + r0 * PITCH + term * PLANE), b = read_columns((near ^ 48) + (r0 + 8) * PITCH + term * PLANE);
        return v4i{a[0], a[1], b[0], b[1]};
    }
    // The same for operands of 16 rows and 32 k: rows r0 .. r0 + 15, columns 32 k + 8 * (lane / 16) ..; and columns 16 n .. 16 n + 15, whose eight k are rows
    // r0 + 4 * (lane / 16) + 0..3 and 16 more on: those that a lane's two result tiles hold
    __device__ static unsigned row_place16(int lane) { return at(lane & 15, lane >> 4); }
    __device__ static unsigned column_place16(int lane) {
        const int l = lane & 15;
        return at(4 * (lane >> 4) + (l >> 2), (l & 3) >> 1) + 8 * (l & 1);
    }
    __device__ static v4i rows16(unsigned place, int r0, int k, int term) { return read_chunk(moved(place, 64 * k) + r0 * PITCH + term * PLANE); }
    __device__ static v4i columns16(unsigned place, int n, int term) {
        const unsigned near = moved(place, 32 * n) + term * PLANE;
        const v2i32 a = read_columns(near), b = read_columns(near + 16 * PITCH);
        return v4i{a[0], a[1], b[0], b[1]};
    }
};

// A value that the compiler may not carry through a loop in other forms
__device__ __forceinline__ unsigned afresh(unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
}

// How the waves of a workgroup bring a block from memory: wave w rows RPW w .. RPW w + RPW - 1, eight columns a lane and piece, LANES lanes a row, STEP rows a piece.
template <int DK, int ROWS, int WAVES, bool PAD>
struct Stage {
    static constexpr int RPW = ROWS / WAVES, LANES = DK <= 32 ? 4 : DK <= 64 ? 8 : 16, STEP = 64 / LANES, PIECES = RPW / STEP;
    static_assert(PIECES * STEP == RPW && RPW % 8 == 0, "a block divides over the lanes");
    static constexpr bool SOME = PAD || DK != 8 * LANES;         // some lanes have columns past the head
    using B = Block<DK, ROWS>;
    float x[PIECES][8];
    // Of a lane: its row and column in the first piece in memory (bytes) and in LDS
    struct Place {
        unsigned from, to, row;
    };
    __device__ static Place place(int wave, int lane, int64_t pitch) {
        const unsigned row = wave * RPW + lane / LANES, chunk = lane % LANES;
        return {row * (unsigned)pitch * 4 + 32 * chunk, B::at(row, chunk), row};
    }
    // Row r of the block is at base + min(r, last) * pitch (below 2^32 bytes: pitches are up to 2^24 bytes).  Lanes past the head read its first columns.
    __device__ __forceinline__ void load(const float *base, int64_t pitch, int last, const Place &at, int lane, int dk) {
        const char *from = reinterpret_cast<const char *>(base);
        const int col = lane % LANES * 8;
        const unsigned step = (unsigned)pitch * 4 * STEP;
        unsigned off[PIECES];
        if (last >= ROWS - 1) {
#pragma unroll
            for (int i = 0; i < PIECES; i++) off[i] = at.from + i * step;
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; i++) off[i] = (unsigned)min((int)at.row + i * STEP, last) * (unsigned)pitch * 4 + 4 * col;
        }
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const unsigned there = !SOME || col + 4 * h < dk ? off[i] + 16 * h : off[i] - 4 * col;
                const v4f a = *reinterpret_cast<const v4f *>(from + (uint64_t)there);
#pragma unroll
                for (int e = 0; e < 4; e++) x[i][4 * h + e] = a[e];
            }
    }
    // to LDS at `block`, cut; the rows' factors, times `by` and then `down`, beside them.  A piece further on is STEP rows and an exchange of chunks away.
    __device__ __forceinline__ void put(unsigned block, unsigned factors, const Place &at, int lane, float by, int dk, float down = 1.0f) {
        const int chunk = lane % LANES;
        const unsigned to = at.to + block;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            if (PAD)                                 // columns from dk on are zero
#pragma unroll
                for (int e = 0; e < 8; e++) x[i][e] = 8 * chunk + (e & 4) < dk ? x[i][e] : 0.0f;
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) most = fmaxf(most, __builtin_fabsf(x[i][e]));
            const float up = row_up(most_of_lanes<LANES>(most));
            v4i t[2];
            cut_halves(x[i], up, t);
            if (8 * LANES == DK || 8 * chunk < DK) {
                const unsigned there = (to ^ (B::low_key(i * STEP) << 4)) + i * STEP * B::PITCH;
                write_chunk(there, t[0]);
                write_chunk(there + B::PLANE, t[1]);
            }
            if (chunk == 0) write_float(factors + 4 * (at.row + i * STEP), row_factor(up) * by * down);
        }
    }
};

// A lane's part of a row, of PARTS: columns 8 (PARTS s + part) .. + 7 for step s.  Rows that are not live are zero, and not read.
template <bool PAD, int PARTS, int KS>
__device__ __forceinline__ void load_row(float (&x)[KS][8], const float *row, bool live, int part, int dk) {
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int col = 8 * (PARTS * s + part) + 4 * h;
            v4f v = {0.f, 0.f, 0.f, 0.f};
            if (live && (!PAD || col < dk)) v = *reinterpret_cast<const v4f *>(row + col);
#pragma unroll
            for (int e = 0; e < 4; e++) x[s][4 * h + e] = v[e];
        }
}

// The least or most of the values of 32 lanes (each half of a wave), in all of them
template <typename Pick>
__device__ __forceinline__ int of_half_wave(int v, Pick pick) {
    v = pick(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true));
    v = pick(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true));
    v = pick(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true));
    v = pick(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true));
    const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    return pick((int)r[0], (int)r[1]);
}
// What 32 rows see together: the last end, the first end of those that see anything, the range of their documents
struct RowsSeen {
    int last, sure, low, high;
};
__device__ __forceinline__ RowsSeen rows_seen(const AttnRow &row) {
    auto least = [](int a, int b) { return min(a, b); };
    auto most = [](int a, int b) { return max(a, b); };
    const bool live = row.end > 0;
    return {of_half_wave(row.end, most), of_half_wave(live ? row.end : 0x7fffffff, least), of_half_wave(live ? row.doc : 0x7fffffff, least), of_half_wave(live ? row.doc : -1, most)};
}
__device__ __forceinline__ RowsSeen same_for_wave(const RowsSeen &s) {
    return {__builtin_amdgcn_readfirstlane(s.last), __builtin_amdgcn_readfirstlane(s.sure), __builtin_amdgcn_readfirstlane(s.low), __builtin_amdgcn_readfirstlane(s.high)};
}

// STEPS steps of products: fetch(i, f) reads the operand of step i from LDS, multiply(i, f) uses it.  Reads go out two steps ahead, so that no product waits for a
// read that was only just asked for; left alone, the compiler saves registers, asks for each operand right before its use, and the matrix core
// idles for the LDS's latency at every step.
template <int STEPS, typename Fetch, typename Multiply>
__device__ __forceinline__ void products(Fetch fetch, Multiply multiply) {
    constexpr int ALU = 0x6;                         // vector and scalar instructions may pass from step to step, memory and matrix ones not
    v4i f[3][2];
    fetch(0, f[0]);
    if (STEPS > 1) fetch(1, f[1]);
    __builtin_amdgcn_sched_barrier(ALU);
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        if (s + 2 < STEPS) fetch(s + 2, f[(s + 2) % 3]);
        multiply(s, f[s % 3]);
        __builtin_amdgcn_sched_barrier(ALU);
    }
}

// The documents of 32 keys (or rows): the lowest and highest id there, -1 and below not counted; `low` is ~lowest where some are not
// counted, so that one document all over is low == high.  No id at all: (INT_MAX, -1).
struct DocRange {
    int low, high;
    __device__ bool meets(int from, int to) const { return high >= from && (low < 0 ? ~low : low) <= to; }
};

}  // namespace axhip
