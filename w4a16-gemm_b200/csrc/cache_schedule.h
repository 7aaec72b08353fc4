// The order in which the cache's prompt kernel issues its tensor-core products, and the TMEM columns
// they use.  Plain C++ shared by the kernel and by a host-only checker that compiles it without nvcc.
//
// tcgen05 products run asynchronously.  Only products of one accumulator and shape are promised to
// run in the order of their issue; between any others a thread that needs an order commits the first
// to a barrier and waits for it.
#pragma once

#if defined(__CUDACC__)
#define W4A16_HD __host__ __device__
#else
#define W4A16_HD
#endif

namespace w4a16 {

constexpr int kCpRows = 128;        // rows of a half
constexpr int kCpTile = 128;        // cached tokens of a tile
constexpr int kCpStages = 2;        // shared-memory stages of keys and of values

// TMEM columns of a half: scores (fp32), weights (fp16, two a column), result (fp32).  With 128-wide heads
// scores and results take all 512 columns, and the weights lie over the first half of the scores that they
// come from; with 64-wide heads they have columns of their own.
template <int D>
struct CpTmem {
    static constexpr bool P_OVER_S = D == 128;
    W4A16_HD static constexpr int S(int h) { return h * kCpTile; }
    W4A16_HD static constexpr int O(int h) { return 2 * kCpTile + h * D; }
    W4A16_HD static constexpr int P(int h) { return P_OVER_S ? S(h) : 2 * kCpTile + 2 * D + h * (kCpTile / 2); }
    static_assert(2 * kCpTile + 2 * D + (P_OVER_S ? 0 : kCpTile) <= 512, "TMEM columns");
};

// The tiles of a CTA and how its halves take them: event e is one half's products with one tile, the halves
// in turn.  kv2: both halves hold the same rows and take alternate tiles; else every tile is for both.
struct CpWalk {
    int n;           // tiles
    bool two;        // the second half has work
    bool kv2;
    W4A16_HD int shift() const { return two && !kv2 ? 1 : 0; }
    W4A16_HD int events() const { return n << shift(); }
    W4A16_HD int tile_of(int e) const { return e >> shift(); }
    W4A16_HD int half_of(int e) const { return two ? e & 1 : 0; }
    W4A16_HD int step_of(int e) const { return two ? e >> 1 : e; }      // the event's number among its half's
    W4A16_HD bool ends_tile(int e) const { return shift() == 0 || (e & 1); }
    // Steps whose result is committed: those that are waited for.  Where that is not every one, there is one
    // only, so that a wait for a phase's parity cannot mistake one step for the one before the last.
    template <int D>
    W4A16_HD bool commits_o(int step, int h) const { return CpTmem<D>::P_OVER_S || step + 1 == steps(h); }
    // Which commit of the half's result says that its last step is done.
    template <int D>
    W4A16_HD int last_o(int h) const { return CpTmem<D>::P_OVER_S ? steps(h) - 1 : 0; }
    W4A16_HD int steps(int h) const { return two ? (kv2 ? (n + 1 - h) / 2 : n) : (h == 0 ? n : 0); }
};

// What the warp that issues the products does.  `op` issues them, commits and waits:
//     wait_q(h), wait_k(stage, turn), wait_v(stage, turn)    operands in shared memory; turn: use of the stage
//     wait_p(h, step)          the half's softmax has read its scores of this step and written its weights
//     wait_o(h, i)             the half's i-th committed PV is done (with all products issued before it)
//     scores(h, stage), values(h, stage, step)               S = Q K^T and O += P V (O = P V at step 0)
//     commit_s(h), commit_o(h), commit_k(stage), commit_v(stage)
// Waits return false when they run out; nothing is issued after that.
template <int D, typename Op>
W4A16_HD inline void cp_products(const CpWalk& w, Op& op) {
    auto issue_s = [&](int e) {
        const int h = w.half_of(e), tile = w.tile_of(e), st = tile % kCpStages;
        if (!op.wait_k(st, tile / kCpStages)) return false;
        // The half's next scores go over the weights that its last PV reads, another accumulator's product.  (512
        // queries of 64 heads over 32768 tokens: 650 us; 711 with the scores that do not go over the weights
        // issued before the wait, as products of 64 columns.)
        if (CpTmem<D>::P_OVER_S && w.step_of(e) > 0 && !op.wait_o(h, w.step_of(e) - 1)) return false;
        op.scores(h, st);
        op.commit_s(h);
        if (w.ends_tile(e)) op.commit_k(st);
        return true;
    };
    const int events = w.events(), ahead = w.two ? 2 : 1;
    if (!op.wait_q(0)) return;
    if (w.two && !w.kv2 && !op.wait_q(1)) return;
    for (int e = 0; e < ahead && e < events; ++e)
        if (!issue_s(e)) return;
    for (int e = 0; e < events; ++e) {
        const int h = w.half_of(e), tile = w.tile_of(e), st = tile % kCpStages, step = w.step_of(e);
        if (!op.wait_v(st, tile / kCpStages) || !op.wait_p(h, step)) return;
        op.values(h, st, step);
        if (w.commits_o<D>(step, h)) op.commit_o(h);
        if (w.ends_tile(e)) op.commit_v(st);
        if (e + ahead < events && !issue_s(e + ahead)) return;
    }
}

}  // namespace w4a16
