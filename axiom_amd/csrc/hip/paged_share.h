// Which part of a block of keys and values each thread of a tile's workgroup brings (paged_tiles.hip): 16 bytes a pass, LANES threads a row, rows of keys and then of values.
#pragma once

namespace axhip {

template <int DK, int BITS, int BKV, int THREADS>
struct BlockShare {
    static constexpr int COLS = 128 / BITS, LANES = (DK == 96 ? 128 : DK) / COLS, ALL = 2 * BKV * LANES, PASSES = ALL > THREADS ? ALL / THREADS : 1;
    static constexpr int PLACES = PASSES > 1 ? PASSES / 2 : 1;   // with two passes or more, the second half brings the values of the first half's keys
    static_assert(ALL <= THREADS || ALL % (2 * THREADS) == 0, "whole passes of keys");
    // from BKV on a value's; from 2 BKV on none
    __host__ __device__ static constexpr int row(int thread, int pass) { return (pass * THREADS + thread) / LANES; }
    __host__ __device__ static constexpr bool has_row(int thread, int pass) { return ALL >= THREADS || row(thread, pass) < 2 * BKV; }
    // Whether a thread's key has no page.  (Heads of up to 32 in 4 bits leave half of the threads without a row: said of those, every block would have holes and
    // every tile pay for the mask: two chunks of 2048 tokens over 4096, 32 heads, 8 of keys, of 32, 4 bits, took 344 us so, and take 174.)
    __host__ __device__ static constexpr bool misses(int thread, int pass, bool page) { return !page && has_row(thread, pass); }
};

}  // namespace axhip
