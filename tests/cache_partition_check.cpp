// Host-only check of how the cache's attention cuts its work (csrc/cache_partition.h and csrc/cache_plan.h), built
// with g++ by tests/test_cache_plan_cpu.py.  It walks every CTA of the decode kernel as its producer warp does
// and checks what the consumers and cache_decode_combine_kernel rely on:
//   * every unit of every segment is done once, by a CTA whose range holds it, and units hold every token that
//     a row of the sequence sees;
//   * the last unit of a CTA, and only that, is marked as such;
//   * a segment inside one CTA is not marked as a part; the parts of a cut one go to distinct slots, at those from
//     which the combine kernel reads, with the first and last CTA noted by the CTA of its first unit.
// And of the plans: grids and workspaces within their bounds, enough for what the kernels write.
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <utility>
#include <vector>

#include "cache_partition.h"
#include "cache_plan.h"

using namespace w4a16;

static int g_fail = 0;
static long g_cases = 0;

#define CHECK(cond, ...)                                                    \
    do {                                                                    \
        if (!(cond)) {                                                      \
            if (g_fail++ < 20) {                                            \
                std::printf("FAIL %s: ", where);                            \
                std::printf(__VA_ARGS__);                                   \
                std::printf("\n");                                          \
            }                                                               \
            return;                                                         \
        }                                                                   \
    } while (0)

struct Seq { int nq, all, len; };     // queries answered, queries, cached tokens

static void check_call(const char* where, const std::vector<Seq>& seqs, int heads, int shared, int window, int grid) {
    ++g_cases;
    std::vector<CdShape> shape;
    std::vector<long long> base;
    long long total = 0;
    for (const Seq& s : seqs) {
        const int pos0 = s.len - s.all;
        shape.push_back(cd_shape(s.nq, shared, s.len, pos0, window));
        const CdShape& h = shape.back();
        base.push_back(total);
        total += h.cost(heads);
        if (s.nq && s.len) {
            CHECK(h.tiles > 0 && h.first >= 0, "no units for %d queries over %d tokens", s.nq, s.len);
            CHECK((long long)h.first * kCdTile <= seen_from(window, pos0) && (long long)(h.first + h.tiles) * kCdTile >= s.len,
                  "units %d + %d for %d tokens", h.first, h.tiles, s.len);
            CHECK((long long)h.blocks * kCdRows >= (long long)s.nq * shared, "blocks %d", h.blocks);
        } else {
            CHECK(h.tiles == 0, "units of an empty sequence");
        }
    }
    const CdCut cut(total, grid);
    CHECK(cut.ctas <= grid && cut.begin(0) == 0 && (total == 0 || cut.begin(cut.ctas) == total), "range ends");
    std::map<std::pair<int, int>, std::vector<int>> did;          // (sequence, segment) -> CTA of each unit
    std::map<std::pair<int, int>, std::pair<int, int>> info;
    std::map<int, std::pair<int, int>> slots;
    std::map<std::pair<int, int>, bool> whole;
    for (int c = 0; c < cut.ctas; ++c) {
        const long long u0 = cut.begin(c), u1 = cut.begin(c + 1);
        CHECK(u1 > u0, "an empty range");
        int b = -1;
        for (size_t i = 0; i < seqs.size(); ++i)
            if (u0 >= base[i] && u0 < base[i] + shape[i].cost(heads)) b = (int)i;
        CHECK(b >= 0, "no sequence for position %lld", u0);
        CdWalk w(cut, c, base[b], shape[b]);
        bool begins = true, ended = false, part = false;
        while (w.more()) {
            const CdShape& h = shape[b];
            CHECK(!ended, "a unit after the one marked as the CTA's last");
            CHECK(w.u >= u0 && w.u < u1, "position %lld outside the range", w.u);
            CHECK(w.sh.tiles == h.tiles && w.sh.first == h.first && w.sh.blocks == h.blocks, "another sequence's segments");
            CHECK(w.seg >= 0 && w.seg < heads * h.blocks && w.tile >= 0 && w.tile < h.tiles, "segment %d tile %d", w.seg, w.tile);
            CHECK(w.head() * h.blocks + w.block() == w.seg && w.head() < heads, "head %d block %d", w.head(), w.block());
            CHECK(w.u == base[b] + (long long)w.seg * (h.tiles + kCdSegmentCost) + kCdSegmentCost + w.tile, "position of a unit");
            const std::pair<int, int> key(b, w.seg);
            CHECK((int)did[key].size() == w.tile, "unit %d of a segment after %d", w.tile, (int)did[key].size());
            did[key].push_back(c);
            if (begins) part = w.part();
            CHECK(part == w.part(), "a part that changes its mind");
            if (w.tile == 0) info[key] = {c, cut.cta_before(w.seg0 + w.sh.tiles)};
            if (w.ends()) {
                if (w.part()) {
                    const int s = w.slot(c);
                    CHECK(s >= 0 && s < 2 * grid && !slots.count(s), "slot %d", s);
                    slots[s] = key;
                } else {
                    whole[key] = true;
                }
            }
            ended = w.last();
            begins = w.ends();
            if (w.advance(heads)) {
                CHECK(!ended, "a sequence after the unit marked as last");
                do { ++b; CHECK(b < (int)seqs.size(), "no sequence left"); } while (shape[b].tiles == 0);
                w.follow(shape[b]);
            }
        }
        // a range without a unit is the start of a segment only: the producer tells the consumers at once
        CHECK(ended || CdWalk(cut, c, base[b], shape[b]).more() == false, "the CTA's last unit is not marked");
    }
    size_t read = 0;
    for (size_t i = 0; i < seqs.size(); ++i)
        for (int s = 0; s < (shape[i].tiles ? heads * shape[i].blocks : 0); ++s) {
            const std::pair<int, int> key((int)i, s);
            CHECK((int)did[key].size() == shape[i].tiles, "units of a segment: %d of %d", (int)did[key].size(), shape[i].tiles);
            CHECK(info.count(key), "a segment whose CTAs are not noted");
            const int first = info[key].first, last = info[key].second;
            CHECK(did[key].front() == first && did[key].back() == last, "CTAs %d..%d, noted %d..%d", did[key].front(), did[key].back(), first, last);
            CHECK((last == first) == (whole.count(key) == 1), "written at once by CTA %d, parts to CTA %d", first, last);
            for (int c = 0; last > first && c <= last - first; ++c, ++read) {
                const int slot = cd_part_slot(first, c);
                CHECK(slots.count(slot) && slots[slot] == key, "slot %d is another segment's", slot);
            }
        }
    CHECK(read == slots.size(), "%d slots written, %d read", (int)slots.size(), (int)read);
}

static void check_decode() {
    std::mt19937 rng(1);
    auto pick = [&](std::vector<int> v) { return v[rng() % v.size()]; };
    for (int i = 0; i < 1500; ++i) {
        const int batch = pick({1, 1, 2, 7, 40, 333}), heads = pick({1, 2, 5, 8}), shared = pick({1, 2, 4, 7, 16});
        const int most = cd_max(1, 32 / shared), top = pick({1, 130, 2000, batch > 7 ? 3000 : 20000}), window = pick({0, 0, 1, 100, 1000, 5000});
        std::vector<Seq> seqs;
        for (int b = 0; b < batch; ++b) {
            const int all = (int)(rng() % (most + 2)), len = pick({0, 1 + (int)(rng() % top), top});
            seqs.push_back({all < most ? all : most, all, len});
        }
        for (int grid : {1, 5, 148, 444}) check_call("decode", seqs, heads, shared, window, grid);
    }
    // the longest sequences: where each CTA begins, without the walk
    const char* where = "long";
    for (int batch : {1, 3, 65535})
        for (int heads : {1, 8, 1024}) {
            const CdShape h = cd_shape(8, 4, 2147483647 - 1023, 2147483647 - 1031, 0);
            CHECK(h.tiles == (1 << 24) - 8 && h.first == 0, "units of the longest sequence: %d", h.tiles);
            const CdCut cut(h.cost(heads) * batch, 444);
            for (int c = 0; c < 444; ++c) {
                const __int128 want = (__int128)cut.total * c / cut.ctas;
                CHECK(cut.begin(c) == (long long)want, "begin of CTA %d", c);
                const long long b = cut.begin(c) / h.cost(heads);
                CdWalk w(cut, c, b * h.cost(heads), h);
                CHECK(w.seg >= 0 && w.seg < heads * h.blocks && w.tile >= 0 && w.tile < h.tiles && w.u >= cut.begin(c), "start of CTA %d", c);
                CHECK(cut.cta_before(cut.begin(c + 1)) == c, "CTA before its end: %d", c);
                ++g_cases;
            }
        }
}

static void check_plan(const char* where, const w4a16_cache& c, const w4a16_cache_attention_args& a, int sms) {
    ++g_cases;
    const AttentionPlan p = plan_attention(c, a, sms);
    const int64_t shared = a.q_heads / c.kv_heads, rows = a.max_q * shared;
    const int64_t tiles = ((int64_t)a.table_pages * c.page_size + kCpTile - 1) / kCpTile;
    CHECK(p.grid >= 1, "grid %d", p.grid);
    if (p.row_blocks) {
        CHECK(rows <= 32 && (int64_t)p.row_blocks * kCdRows >= rows && p.row_blocks <= 4, "%d blocks of rows", p.row_blocks);
        CHECK(p.grid <= kCdCtas * sms, "grid %d", p.grid);
        const int64_t segments = (int64_t)a.batch * c.kv_heads * p.row_blocks;
        CHECK(p.workspace >= (size_t)segments * 8 + 2 * (size_t)p.grid * kCdRows * (c.head_dim + 2) * 4, "workspace");
        CHECK(cd_info_bytes(segments) % 16 == 0 && cd_slot_floats(c.head_dim) * 4 % 16 == 0, "alignment of a slot");
        return;
    }
    CHECK(rows > 32, "%d rows", (int)rows);
    const int64_t block_rows = p.prompt.kv2 ? kCpRows : 2 * kCpRows;
    CHECK(!p.prompt.kv2 || rows <= kCpRows, "alternate tiles for %d rows", (int)rows);
    CHECK((int64_t)p.prompt.blocks * block_rows >= rows && (int64_t)(p.prompt.blocks - 1) * block_rows < rows, "%d blocks", p.prompt.blocks);
    CHECK(p.prompt.splits >= 1 && (p.prompt.splits == 1 || p.prompt.splits <= tiles / 4), "%d splits of %d tiles", p.prompt.splits, (int)tiles);
    CHECK((int64_t)p.grid == (int64_t)p.prompt.blocks * a.batch * c.kv_heads * p.prompt.splits, "grid %d", p.grid);
    // a part of a row is its D sums, maximum and sum of weights; nothing passes through memory where nothing is split
    const size_t part = (size_t)a.q_tokens * a.q_heads * (c.head_dim + 2) * 4;
    CHECK(p.workspace == (p.prompt.splits > 1 ? p.prompt.splits * part : 0), "workspace of %d parts", p.prompt.splits);
    CHECK(p.workspace <= (256u << 20), "workspace of %zu bytes", p.workspace);
}

static void check_plans() {
    std::mt19937 rng(2);
    auto log_pick = [&](double lo, double hi) { return (int64_t)(lo * std::pow(hi / lo, rng() / 4294967296.0) + 0.5); };
    for (int i = 0; i < 200000; ++i) {
        w4a16_cache c = {};
        w4a16_cache_attention_args a = {};
        c.num_pages = 1 << 20;
        c.head_dim = rng() % 2 ? 128 : 64;
        c.group_size = 64;
        c.page_size = 16 << rng() % 5;
        c.kv_heads = (int32_t)log_pick(1, rng() % 4 ? 16 : 1024);
        a.q_heads = c.kv_heads * (int32_t)log_pick(1, 16);
        a.batch = (int32_t)log_pick(1, 65535);
        a.max_q = (int32_t)log_pick(1, 100000);
        a.q_tokens = a.max_q + (int64_t)(rng() / 4294967296.0 * a.max_q * (a.batch - 1));
        a.table_pages = (int32_t)(log_pick(1, rng() % 4 ? 262144 : 2147482624.0) / c.page_size);
        a.causal = rng() % 4 != 0;
        a.window = rng() % 3 ? 0 : (int32_t)log_pick(1, 100000);
        // what the entry point accepts
        if (a.q_tokens * a.q_heads >= (1LL << 31) || (int64_t)a.table_pages * c.page_size > (1LL << 31) - 1024 || a.q_heads > 65536 ||
            (int64_t)a.batch * ((int64_t)a.max_q * a.q_heads / 128 + c.kv_heads) >= (1LL << 31))
            continue;
        check_plan("plan", c, a, rng() % 8 ? 148 : 1 + (int)(rng() % 300));
    }
}

int main() {
    check_decode();
    check_plans();
    if (g_fail) {
        std::printf("%d failures in %ld cases\n", g_fail, g_cases);
        return 1;
    }
    std::printf("ok %ld cases\n", g_cases);
    return 0;
}
