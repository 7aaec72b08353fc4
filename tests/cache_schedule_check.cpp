// Host-only check of the order in which the cache's prompt kernel issues its products
// (csrc/cache_schedule.h), built with g++ by tests/test_cache_schedule_cpu.py.  cp_products runs on a
// recorder that knows what tcgen05 promises: products of one accumulator and shape run in the
// order of their issue, any others in any order, and a commit's barrier completes when all
// products issued before it have.  For every product and every access of the softmax warps it checks that
// whatever touches the same TMEM columns (one of the two writing) has been waited for, and that a stage of shared
// memory is handed back after the last product that reads it, once a tile.
#include <cstdio>
#include <map>
#include <vector>

#include "cache_schedule.h"

using namespace w4a16;

static int g_fail = 0;

struct Span {
    int a, n;
    bool meets(const Span& o) const { return a < o.a + o.n && o.a < a + n; }
};

struct Product {
    Span out, in;         // TMEM columns written (and read, where it accumulates), operand columns
    int k_tile, v_tile;   // tile whose stage it reads, or -1
    const char* what;
};

template <int D>
struct Recorder {
    using T = CpTmem<D>;
    const CpWalk& w;
    std::vector<Product> done;                    // all issued, in order
    size_t known = 0;                             // the issuing warp knows that done[0 .. known) are complete
    std::vector<size_t> s_commit[2], o_commit[2]; // by step: products issued before the commit
    int scores_of[2] = {0, 0}, values_of[2] = {0, 0}, weights_of[2] = {0, 0};
    std::map<int, int> k_back, v_back;            // tile -> products before its stage was handed back
    int k_commits = 0, v_commits = 0;
    int known_o[2] = {0, 0};                      // commits of results that the issuing warp has waited for

    explicit Recorder(const CpWalk& walk) : w(walk) {}
    void fail(const char* msg, int x) {
        if (g_fail++ < 20) std::printf("FAIL D=%d n=%d two=%d kv2=%d: %s (%d)\n", D, w.n, w.two, w.kv2, msg, x);
    }
    int tile_of(int h, int step) const { return w.two ? (w.kv2 ? 2 * step + h : step) : step; }

    // The softmax of a half's step: knows what was committed before its scores.
    void softmax(int h, int step) {
        const size_t sure = s_commit[h][step];
        const Span s{T::S(h), kCpTile}, p{T::P(h), kCpTile / 2}, o{T::O(h), D};
        for (size_t j = sure; j < done.size(); ++j) {
            if (done[j].out.meets(s)) fail("a product writes scores while they are read", (int)j);
            if (done[j].out.meets(p) || done[j].in.meets(p)) fail("weights are written over columns of an unfinished product", (int)j);
            if (step > 0 && done[j].out.meets(o)) fail("a result is rescaled while a product adds to it", (int)j);
        }
    }
    bool wait_q(int) { return true; }
    bool wait_k(int st, int turn) {
        if (st < 0 || st >= kCpStages || turn < 0) fail("wait for keys", st);
        return true;
    }
    bool wait_v(int st, int turn) {
        if (st < 0 || st >= kCpStages || turn < 0) fail("wait for values", st);
        return true;
    }
    bool wait_p(int h, int step) {
        if ((size_t)step >= s_commit[h].size()) { fail("a wait for weights whose scores were not issued", step); return false; }
        if (step != weights_of[h]++) fail("weights out of order", step);
        softmax(h, step);
        if (s_commit[h][step] > known) known = s_commit[h][step];
        return true;
    }
    bool wait_o(int h, int step) {
        if ((size_t)step >= o_commit[h].size()) { fail("a wait for a result that was not issued", step); return false; }
        if (o_commit[h][step] > known) known = o_commit[h][step];
        known_o[h] = step + 1;
        return true;
    }
    void issue(const Product& p) {
        for (size_t j = known; j < done.size(); ++j) {
            const Product& q = done[j];
            const bool one_pipe = q.out.a == p.out.a && q.out.n == p.out.n;      // same accumulator and shape
            if (one_pipe) continue;
            if (p.out.meets(q.out) || p.out.meets(q.in) || p.in.meets(q.out)) {
                fail("a product meets columns of an unfinished one", (int)done.size());
                std::printf("    %s after %s\n", p.what, q.what);
            }
        }
        done.push_back(p);
    }
    void scores(int h, int st) {
        const int step = scores_of[h]++;
        if (step > 0 && weights_of[h] < step) fail("scores over scores that the softmax has not read", step);
        if (tile_of(h, step) % kCpStages != st) fail("stage of the keys", st);
        // a product of M = 128 rows; the unit of order is the accumulator, so one entry stands for its D / 16 pieces
        issue({{T::S(h), kCpTile}, {-1, 0}, tile_of(h, step), -1, "scores"});
    }
    void values(int h, int st, int step) {
        if (step != values_of[h]++) fail("values out of order", step);
        if (weights_of[h] != step + 1) fail("values before their weights", step);
        if (tile_of(h, step) % kCpStages != st) fail("stage of the values", st);
        issue({{T::O(h), D}, {T::P(h), kCpTile / 2}, -1, tile_of(h, step), "values"});
    }
    void commit_s(int h) { s_commit[h].push_back(done.size()); }
    void commit_o(int h) { o_commit[h].push_back(done.size()); }
    void commit_k(int st) {
        if (k_commits % kCpStages != st) fail("keys handed back out of order", st);
        k_back[k_commits++] = (int)done.size();
    }
    void commit_v(int st) {
        if (v_commits % kCpStages != st) fail("values handed back out of order", st);
        v_back[v_commits++] = (int)done.size();
    }
    void finish() {
        for (int h = 0; h < 2; ++h) {
            const int steps = w.steps(h);
            if (scores_of[h] != steps || values_of[h] != steps || weights_of[h] != steps) fail("steps of a half", h);
            if ((int)s_commit[h].size() != steps) fail("commits of a half", h);
            if (!steps) continue;
            // The softmax reads the result after the commit that last_o names: no later one, all of the half's products
            // before it.  Its wait is for a phase's parity: the one before must be known to be complete.
            const int last = w.template last_o<D>(h);
            if ((int)o_commit[h].size() != last + 1) { fail("commits of a result", h); continue; }
            for (size_t j = o_commit[h][last]; j < done.size(); ++j)
                if (done[j].out.meets({T::O(h), D})) fail("a product adds to a result after its last commit", (int)j);
            if (last > 0 && known_o[h] < last) fail("a result's phase is waited for while the one before may be open", h);
        }
        if (k_commits != w.n || v_commits != w.n) fail("stages handed back", k_commits);
        for (size_t j = 0; j < done.size(); ++j) {
            if (done[j].k_tile >= 0 && (int)j >= k_back[done[j].k_tile]) fail("keys handed back before their last product", (int)j);
            if (done[j].v_tile >= 0 && (int)j >= v_back[done[j].v_tile]) fail("values handed back before their last product", (int)j);
        }
    }
};

template <int D>
static void check(int n, bool two, bool kv2) {
    const CpWalk w{n, two, kv2};
    Recorder<D> r(w);
    if (n > 0) cp_products<D>(w, r);
    r.finish();
    using T = CpTmem<D>;
    const Span all[6] = {{T::S(0), kCpTile}, {T::S(1), kCpTile}, {T::O(0), D}, {T::O(1), D}, {T::P(0), kCpTile / 2}, {T::P(1), kCpTile / 2}};
    for (int i = 0; i < 6; ++i) {
        if (all[i].a < 0 || all[i].a + all[i].n > 512) r.fail("columns outside TMEM", i);
        for (int j = 0; j < i; ++j)
            if (all[i].meets(all[j]) && !(T::P_OVER_S && i == j + 4)) r.fail("columns shared", i);
    }
}

int main() {
    long cases = 0;
    for (int n = 0; n <= 40; ++n)
        for (int form = 0; form < 4; ++form) {
            const bool two = form & 1, kv2 = form & 2;
            if (kv2 && two != (n > 1)) continue;         // the kernel's own rule
            check<64>(n, two, kv2);
            check<128>(n, two, kv2);
            cases += 2;
        }
    if (g_fail) {
        std::printf("%d failures in %ld cases\n", g_fail, cases);
        return 1;
    }
    std::printf("ok %ld cases\n", cases);
    return 0;
}
