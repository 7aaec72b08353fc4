// How an expert layer's call is cut: sizes, workspace regions and work ranges.  Plain C++ shared by the host and the
// kernels.
//
// An entry is one (token, choice) pair; entry t * k + j is token t's choice j.  Entries of valid experts are
// sorted by expert, and a tile is up to `rows` sorted entries of one expert.
#pragma once
#include <stddef.h>
#include <stdint.h>

#if defined(__CUDACC__)
#define W4A16_HD __host__ __device__
#else
#define W4A16_HD
#endif

namespace w4a16 {

constexpr int kMoeMaxExperts = 1024;
constexpr int kMoeChunks = 8;        // 64-wide K chunks of a stage
constexpr int kMoeRows = 8;          // entries of a tile
// Up to this many entries every CTA of the products sorts them for itself; above, one kernel does it for all.
constexpr int kMoeFewEntries = 1024;

struct MoeTile {
    int32_t expert, start, count, pad;   // sorted entries [start, start + count)
};

// The start of the workspace; the arrays follow it.
struct MoeHead {
    int32_t tiles;       // filled tiles
    int32_t entries;     // sorted (valid) entries
    int32_t pad[62];
};

// What a grouped product reads of it: the tiles, and how far apart the experts' weights and scales are.
struct MoeGroups {
    const MoeHead* head;
    const MoeTile* tiles;
    int32_t blocks;          // n16 blocks of one expert's weight
    int32_t scale_rows;      // rows of one expert's scales
};

struct MoePlan {
    int32_t rows;            // entries of a tile
    int32_t max_tiles;       // no routing makes more
    int32_t splits;          // K ranges of the second product
    bool few;                // every CTA sorts the entries
    bool grouped;            // many entries an expert: the tensor-core products of prompts over sorted rows
    // offsets in the workspace: tiles, entries in sorted order, where each entry went (grouped), rows of x in sorted
    // order (grouped), the gated product's results, the second one's
    size_t tiles_at, order_at, place_at, rows_at, inner_at, out_at, bytes;
};

// More entries an expert than this, on average, are grouped; the second if both products have groups of 128.
constexpr int kMoeGroupedEntries = 14, kMoeGroupedEntriesWide = 10;

constexpr int kMoeGroupedRows = 64;  // entries of a grouped product's tile, at most

W4A16_HD inline size_t moe_align(size_t n) { return (n + 255) / 256 * 256; }

// wide_groups: both products' scales are of groups of 128.
inline MoePlan moe_plan(int64_t tokens, int k, int experts, int hidden, int inner, int num_sms, bool wide_groups = false) {
    MoePlan p = {};
    const int64_t entries = tokens * k;
    // many entries an expert: its words are worth making into tensor-core operands for all of them.  As few and grouped, us from
    // a graph, even loads, 8, 10, 12, 16 and 24 entries an expert:
    //     128 experts of 2048 x 768, groups of 128     139 144   160 144   180 145   221 147   301 151
    //      64 of 2048 x 1408, 128                      108 126   124 126   143 126   178 127   244 132
    //       8 of 4096 x 14336, 128                     213 281   270 281   280 281   367 282   539 283
    //      64 of 2048 x 1408, 64                       108 162   128 163   144 164   176 166   250 172
    // With groups of 64 the grouped products drain twice as often, and the forms meet at 15 instead of 9 to 12.  Entries and experts
    // are the call's, as it is told them: entries of experts outside the layer count (a slice of 8 of 64 experts, 32 tokens of 6:
    // grouped 39 us, as few 23), and how they are spread does not (96 tokens to the same 6 of 64: as few 86, grouped 44).
    p.grouped = entries > (wide_groups ? kMoeGroupedEntriesWide : kMoeGroupedEntries) * (int64_t)experts;
    // else 8, the width of mma.m16n8k16: with 16 a tile's two products for every word cost more than reading the words
    // of an expert twice (64 experts, 3 entries each: 82 us and 102; 8 each: 118 and 128)
    p.rows = p.grouped ? kMoeGroupedRows : kMoeRows;
    // every expert's last tile may be short; no tile is empty
    const int64_t most = entries / p.rows + (experts < entries ? experts : entries);
    p.max_tiles = (int32_t)(most < entries ? most : entries);
    // the second product's K is cut where its column blocks would leave an SM more than an eighth behind the
    // average: few entries, narrow outputs
    const int64_t units = (entries < experts ? entries : experts) * (hidden / 16);
    const int stages = (inner / 64 + kMoeChunks - 1) / kMoeChunks;
    p.splits = 1;
    while (!p.grouped && p.splits < 4 && 2 * p.splits <= stages && units * p.splits < 8 * (int64_t)num_sms) p.splits *= 2;
    p.few = !p.grouped && entries <= kMoeFewEntries;
    p.tiles_at = sizeof(MoeHead);
    p.order_at = moe_align(p.tiles_at + (size_t)p.max_tiles * sizeof(MoeTile));
    p.place_at = moe_align(p.order_at + (size_t)entries * 4);
    p.rows_at = moe_align(p.place_at + (p.grouped ? (size_t)entries * 4 : 0));
    p.inner_at = moe_align(p.rows_at + (p.grouped ? (size_t)entries * hidden * 2 : 0));
    p.out_at = moe_align(p.inner_at + (size_t)entries * inner * 2);
    p.bytes = moe_align(p.out_at + (size_t)p.splits * entries * hidden * 4);
    return p;
}

}  // namespace w4a16
