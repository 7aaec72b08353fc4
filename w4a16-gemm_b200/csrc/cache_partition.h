// How the cache's decode kernel cuts its work, and where the parts of cut segments go.  Plain C++ shared by
// the host planner, cache_decode_kernel, cache_decode_combine_kernel and a host-only checker that compiles
// it without nvcc.
//
// A segment is a (sequence, key head, block of rows); its units are the tiles of cached tokens that some row
// of the sequence sees.  The cost of all segments, one a unit and kCdSegmentCost for its start, is laid out
// segment by segment and cut into equal ranges, one a CTA.  A CTA passes over starts.
#pragma once
#include <stddef.h>
#include <stdint.h>

#if defined(__CUDACC__)
#define W4A16_HD __host__ __device__
#else
#define W4A16_HD
#endif

namespace w4a16 {

constexpr int kCdTile = 128;        // tokens of a unit
constexpr int kCdRows = 8;          // rows of a block: the right side of an m16n8k16 product
constexpr int kCdCtas = 3;          // CTAs of an SM (shared memory, 128 registers a thread)

// What the start and end of a segment cost beside its units (queries, merge), in units: ranges
// are cut by cost, so that a CTA with many short segments is not the last to finish.
constexpr int kCdSegmentCost = 2;

W4A16_HD inline int cd_max(int a, int b) { return a > b ? a : b; }

// The first token that a query at position pos sees.
W4A16_HD inline int seen_from(int window, int pos) { return window ? cd_max(0, cd_max(pos + 1, 0) - window) : 0; }

// floor(a * b / c) and floor(a / c) of non-negative numbers; 32-bit divisions where they do (a 64-bit one
// takes some 400 cycles, and a short call has several of them in a row).
W4A16_HD inline long long mul_div(long long a, long long b, long long c) {
    const unsigned long long ab = (unsigned long long)a * (unsigned long long)b;
    return (ab | (unsigned long long)c) >> 32 ? (long long)(ab / (unsigned long long)c) : (long long)((uint32_t)ab / (uint32_t)c);
}

// The segments of one sequence, all of one size: `blocks` a key head, of `tiles` units from tile `first` on.
struct CdShape {
    int first, tiles, blocks;
    W4A16_HD long long cost(int heads) const {
        return tiles ? (long long)(tiles + kCdSegmentCost) * ((long long)heads * blocks) : 0;
    }
};

// nq queries that are answered, of `shared` rows each, the first at position pos0; len cached tokens.
W4A16_HD inline CdShape cd_shape(int nq, int shared, int len, int pos0, int window) {
    CdShape s;
    s.first = seen_from(window, pos0) / kCdTile;
    s.tiles = nq == 0 || len == 0 ? 0 : (len + kCdTile - 1) / kCdTile - s.first;
    s.blocks = (nq * shared + kCdRows - 1) / kCdRows;
    return s;
}

// The cost of a call cut into ranges.
struct CdCut {
    long long total, ctas;         // cost of all segments; CTAs with a range, at least one position each
    W4A16_HD CdCut(long long cost, int grid) : total(cost), ctas(cost < grid ? cost : grid) {}
    W4A16_HD long long begin(long long cta) const { return mul_div(total, cta, ctas > 0 ? ctas : 1); }
    // The CTA that holds the position before `end`: floor((end * ctas - 1) / total).
    W4A16_HD int cta_before(long long end) const {
        const unsigned long long x = (unsigned long long)end * (unsigned long long)ctas - 1ull;
        return (x | (unsigned long long)total) >> 32 ? (int)(x / (unsigned long long)total) : (int)((uint32_t)x / (uint32_t)total);
    }
};

// A CTA's way through its range, unit by unit.  A sequence that is done is followed by the next that has
// units, which the caller finds.
struct CdWalk {
    long long u0, u1;              // the range
    long long u, seg0;             // position of the unit, and of its segment's first unit
    int seg, tile;                 // segment of the sequence, unit of the segment
    CdShape sh;
    // base: position at which the sequence of u0 begins
    W4A16_HD CdWalk(const CdCut& cut, long long cta, long long base, const CdShape& shape)
        : u0(cut.begin(cta)), u1(cut.begin(cta + 1)), sh(shape) {
        const long long local = u0 - base;
        seg = (int)mul_div(local, 1, sh.tiles + kCdSegmentCost);
        tile = (int)(local - (long long)seg * (sh.tiles + kCdSegmentCost)) - kCdSegmentCost;
        u = u0;
        if (tile < 0) { u -= tile; tile = 0; }
        seg0 = u - tile;
    }
    W4A16_HD bool more() const { return u < u1; }
    W4A16_HD int head() const { return seg / sh.blocks; }
    W4A16_HD int block() const { return seg % sh.blocks; }
    W4A16_HD bool ends_segment() const { return tile + 1 == sh.tiles; }
    W4A16_HD bool ends() const { return ends_segment() || u + 1 == u1; }                             // this CTA's part of it
    W4A16_HD bool last() const { return u + 1 + (ends_segment() ? kCdSegmentCost : 0) >= u1; }        // unit of this CTA
    W4A16_HD bool part() const { return seg0 < u0 || seg0 + sh.tiles > u1; }                          // of a segment, not all
    // Workspace slot of this CTA's part: 0 of a segment that began in an earlier CTA, 1 of one that begins here.
    W4A16_HD int slot(int cta) const { return 2 * cta + (seg0 >= u0 ? 1 : 0); }
    // To the next unit; true if that is another sequence's: follow() then gives its segments.
    W4A16_HD bool advance(int heads) {
        ++u;
        if (++tile < sh.tiles) return false;
        tile = 0;
        u += kCdSegmentCost;
        seg0 = u;
        return ++seg == heads * sh.blocks && u < u1;
    }
    W4A16_HD void follow(const CdShape& shape) { seg = 0; sh = shape; }
};

// The slot in which the c-th of the CTAs that share a segment, the first being CTA `first`, left its part.
W4A16_HD inline int cd_part_slot(int first, int c) { return 2 * (first + c) + (c == 0 ? 1 : 0); }

// Workspace: per segment the CTAs {first, last} that hold parts of it, then 2 slots
// a CTA of kCdRows x (D + 2) floats: sums, maxima, sums of weights.
W4A16_HD inline size_t cd_info_bytes(int64_t segments) { return (size_t)(segments * 8 + 255) / 256 * 256; }
W4A16_HD inline size_t cd_slot_floats(int D) { return (size_t)kCdRows * (D + 2); }

}  // namespace w4a16
