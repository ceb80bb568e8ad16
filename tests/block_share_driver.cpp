// Which thread brings what of a block of keys and values (paged_share.h) on the host: prints a line for each kind of block.
#define __host__
#define __device__
#include "paged_share.h"

#include <cstdio>
#include <vector>

constexpr int THREADS = 512;

template <int DK, int BITS>
void one() {
    constexpr int BKV = DK <= 64 ? 128 : 64;
    using S = axhip::BlockShare<DK, BITS, BKV, THREADS>;
    const char *bad = nullptr;
    std::vector<int> brought(2 * BKV * S::LANES), holes(BKV);
    int idle = 0;
    for (int thread = 0; thread < THREADS; thread++) {
        bool any = false;
        for (int pass = 0; pass < S::PASSES; pass++) {
            const int row = S::row(thread, pass);
            if (!S::has_row(thread, pass)) continue;
            any = true;
            if (row >= 2 * BKV) bad = "a row that is none";
            else brought[row * S::LANES + thread % S::LANES]++;
            // the values of a pass's keys come half of the passes later, to the same thread
            if (S::PASSES > 1 && pass < S::PLACES && S::row(thread, pass + S::PLACES) != row + BKV) bad = "values of other keys";
        }
        idle += !any;
        for (int place = 0; place < S::PLACES; place++) {
            if (S::misses(thread, place, true)) bad = "a hole where there is a page";
            // a thread without a row never finds a page for it
            if (S::misses(thread, place, false)) {
                if (S::has_row(thread, place)) holes[S::row(thread, place) % BKV]++;
                else bad = "a hole without a row";
            }
        }
    }
    for (int n : brought)
        if (n != 1) bad = "not every piece once";
    for (int n : holes)
        if (n == 0) bad = "a hole that nobody reports";
    printf("%d %d %s, %d idle\n", DK, BITS, bad ? bad : "ok", idle);
}

int main() {
    one<32, 16>(), one<64, 16>(), one<96, 16>(), one<128, 16>();
    one<32, 8>(), one<64, 8>(), one<96, 8>(), one<128, 8>();
    one<32, 4>(), one<64, 4>(), one<96, 4>(), one<128, 4>();
}
