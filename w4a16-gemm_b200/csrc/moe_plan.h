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

struct MoePlan {
    int32_t rows;            // entries of a tile
    int32_t max_tiles;       // no routing makes more
    int32_t splits;          // K ranges of the second product
    bool few;                // every CTA sorts the entries
    size_t tiles_at, order_at, inner_at, out_at, bytes;    // offsets in the workspace
};

W4A16_HD inline size_t moe_align(size_t n) { return (n + 255) / 256 * 256; }

inline MoePlan moe_plan(int64_t tokens, int k, int experts, int hidden, int inner, int num_sms) {
    MoePlan p = {};
    const int64_t entries = tokens * k;
    // 8 entries a tile where an expert seldom gets more (at most 8 tokens, or 4 entries for each expert), else 16
    p.rows = tokens <= 8 || entries <= 4 * (int64_t)experts ? 8 : 16;
    // every expert's last tile may be short; no tile is empty
    const int64_t most = entries / p.rows + (experts < entries ? experts : entries);
    p.max_tiles = (int32_t)(most < entries ? most : entries);
    // the second product's K is cut where its column blocks would leave an SM more than an eighth behind the
    // average: few entries, narrow outputs
    const int64_t units = (entries < experts ? entries : experts) * (hidden / 16);
    const int stages = (inner / 64 + kMoeChunks - 1) / kMoeChunks;
    p.splits = 1;
    while (p.splits < 4 && 2 * p.splits <= stages && units * p.splits < 8 * (int64_t)num_sms) p.splits *= 2;
    p.few = entries <= kMoeFewEntries;
    p.tiles_at = sizeof(MoeHead);
    p.order_at = moe_align(p.tiles_at + (size_t)p.max_tiles * sizeof(MoeTile));
    p.inner_at = moe_align(p.order_at + (size_t)entries * 4);
    p.out_at = moe_align(p.inner_at + (size_t)entries * inner * 2);
    p.bytes = moe_align(p.out_at + (size_t)p.splits * entries * hidden * 4);
    return p;
}

}  // namespace w4a16
