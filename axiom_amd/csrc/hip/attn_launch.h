// How the parts of attention under score rules call each other on the host.
#pragma once
#include "attn_rules.h"

namespace axhip {

struct DocRange;
constexpr int64_t GRID_MOST = int64_t(1) << 22;  // workgroups of a launch: a grid holds fewer than 2^32 threads

struct FwdGrid {
    int64_t first, units;                        // units: heads, or groups of `pack` heads that share keys
    int tiles, pack;
    const DocRange *ranges;                      // [B, range_tiles], with documents
    int range_tiles;
};

struct FewGrid {
    int row_tiles, splits;                       // of 32 rows each; ranges of keys
    float *parts;                                // what the ranges leave
    int *arrivals;
};

struct BwdGrid {
    int64_t first, units;                        // units: query heads, or heads of keys
    int tiles, splits;                           // splits: of what a tile runs over, each a workgroup's
    const DocRange *key_ranges, *row_ranges;     // [B, key_tiles], [B, row_tiles], with documents
    int key_tiles, row_tiles;
    float *parts;                                // what the splits leave
    int *arrivals;
};

// The ranges of ids [B, S] in each 32 (8 bytes each)
int doc_ranges(const int32_t *ids, int64_t B, int64_t S, void *out);
int attn_fwd_tiles(const AttnArgs &a);
bool attn_fwd_few(const AttnArgs &a, int &rc);
int attn_bwd_tiles(AttnArgs &a);

}  // namespace axhip
