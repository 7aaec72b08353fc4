// How an attention call over the 4-bit cache is run: which kernel, its grid, its workspace.  Plain host C++,
// by sizes only, so that it can be checked without a GPU.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>

#include "../../include/w4a16.h"
#include "cache_partition.h"
#include "cache_schedule.h"

namespace w4a16 {

// What a grid of prompt CTAs does.
struct CpGrid {
    int blocks;      // row blocks of the longest sequence
    int splits;      // CTAs that share the tiles of one row block: 1, results are written at once; else joined
    int kv2;         // 128 rows or fewer: the halves take alternate tiles
};

struct AttentionPlan {
    int row_blocks;      // blocks of 8 rows of the decode kernel; 0: the prompt kernel
    int grid;
    CpGrid prompt;
    size_t workspace;
};

inline AttentionPlan plan_decode(const w4a16_cache& c, const w4a16_cache_attention_args& a, int num_sms) {
    const int64_t rows = (int64_t)a.max_q * (a.q_heads / c.kv_heads);
    const int64_t blocks = (rows + kCdRows - 1) / kCdRows, segments = (int64_t)a.batch * c.kv_heads * blocks;
    const int64_t tiles = ((int64_t)a.table_pages * c.page_size + kCdTile - 1) / kCdTile;
    AttentionPlan p = {};
    p.row_blocks = (int)blocks;
    p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(segments * tiles, (int64_t)kCdCtas * num_sms));
    p.workspace = cd_info_bytes(segments) + 2 * (size_t)p.grid * cd_slot_floats(c.head_dim) * sizeof(float);
    return p;
}

// Row blocks of 256 (128, with the halves on alternate tiles, if no sequence has more rows).  A
// block's tiles are split over as many CTAs as an estimate says is shortest: a tile 2.4 us, a CTA's
// start and end 7 us (measured); the work spread over the SMs, and for the last wave, as far as it is not
// full, a CTA of the block with fewest tiles (heavy blocks come first); and the parts written and
// joined.  Measured, 32/8 heads, unsplit / as chosen: 800 queries over 16384 tokens (104 blocks) 292 / 285 us,
// 1200 (152) 556 / 443, 2 x 12 over up to 16384 204 / 42; a prompt of 1500 (192, unsplit) 43.
// Results of split blocks pass through the workspace, which is kept at 256 MB or below.
//
// Lengths are not known here: the page table's width stands for them, so that a table far wider than its
// sequences splits blocks that have nothing to split.  A prompt of 1500: 43 us with a table of its
// size, 108 with one of 32768 tokens; of 4096: 177 and 301.  A caller who knows the lengths passes a view of the
// columns in use.
inline AttentionPlan plan_prompt(const w4a16_cache& c, const w4a16_cache_attention_args& a, int num_sms) {
    const int64_t shared = a.q_heads / c.kv_heads, rows = a.max_q * shared;
    AttentionPlan p = {};
    p.prompt.kv2 = rows <= kCpRows;
    const int64_t block_rows = p.prompt.kv2 ? kCpRows : 2 * kCpRows;
    p.prompt.blocks = (int)((rows + block_rows - 1) / block_rows);
    const int64_t busy = c.kv_heads * std::min<int64_t>((int64_t)p.prompt.blocks * a.batch,
                                                        a.q_tokens * shared / block_rows + a.batch);
    const int64_t tiles = ((int64_t)a.table_pages * c.page_size + kCpTile - 1) / kCpTile;
    const size_t part_bytes = (size_t)(a.q_tokens * a.q_heads) * (size_t)(c.head_dim + 2) * sizeof(float);
    const double block_tiles = (double)block_rows / (double)shared / kCpTile;          // that a block's tokens make
    const double most = a.window > 0 ? std::min((double)tiles, (double)a.window / kCpTile + block_tiles + 1.0) : (double)tiles;
    const double least = a.causal ? std::min(most, std::max(1.0, (double)tiles - (p.prompt.blocks - 1) * block_tiles)) : most;
    double best = 0.0;
    for (int64_t s = 1; s <= std::max<int64_t>(1, (int64_t)most / 4) && (s == 1 || (size_t)s * part_bytes <= (256u << 20)); ++s) {
        const double waves = (double)(busy * s) / num_sms, idle = std::ceil(waves) - waves;
        const double longest = 2.4 * most / (double)s + 7.0, shortest = 2.4 * least / (double)s + 7.0;
        const double join = s == 1 ? 0.0 : 4.0 + 2.0 * (double)s * (double)part_bytes / 4e6;     // written and read at 4 TB/s
        const double t = std::max(longest, waves * (longest + shortest) / 2.0 + idle * shortest) + join;
        if (s == 1 || t < 0.95 * best) { best = t; p.prompt.splits = (int)s; }
        if (waves >= 8.0) break;
    }
    p.grid = (int)((int64_t)p.prompt.blocks * a.batch * c.kv_heads * p.prompt.splits);
    if (p.prompt.splits > 1) p.workspace = (size_t)p.prompt.splits * part_bytes;
    return p;
}

// Up to 32 rows a (sequence, key head) go to the decode kernel, which streams the codes once for
// each 8 of them; more to the prompt kernel, whose 128-row products cost the same for few rows.
// Measured with 4 rows a query (decode / prompt kernel, us): 16 sequences of up to 4096 tokens, 5
// queries 43 / 65, 8 queries 53 / 65, 9 queries 64 / 65, 12 queries 75 / 65; 64 of up to 512, 8 queries
// 54 / 52, 9 queries 65 / 53; 2 of up to 16384, 8 queries 33 / 40, 9 queries 37 / 41, 12 queries 41 / 41.
constexpr int64_t kDecodeRows = 32;

inline AttentionPlan plan_attention(const w4a16_cache& c, const w4a16_cache_attention_args& a, int num_sms) {
    const int64_t rows = (int64_t)a.max_q * (a.q_heads / c.kv_heads);
    return rows > kDecodeRows ? plan_prompt(c, a, num_sms) : plan_decode(c, a, num_sms);
}

}  // namespace w4a16
