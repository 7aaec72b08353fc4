// Attention of few rows (query heads of a key head times queries of a sequence) over the 4-bit
// cache: rows in blocks of 8, one pass over the codes a block.  Included by cache.cu only.
//
// Work (cache_partition.h).  A segment is a (sequence, key head, block of rows), a unit 128 cached tokens of one.  All
// units of the call, segment by segment (a head's blocks after one another: from the second on
// the codes come from L2), are cut into equal contiguous ranges, one a CTA, so that ragged batches
// load every SM alike whatever the lengths; lengths are read on the device.  A range holds whole
// segments, whose results are written at once, and at most two parts of segments, whose sums go
// to the workspace for cache_decode_combine_kernel.
//
// A CTA is one producer warp, which walks the page table and fills a ring of stages with bulk
// copies (the runs of key codes, value codes and pairs of each page), and four consumer warps,
// each with 32 tokens of every stage and its own softmax state; the four states are merged at the
// end of a segment.
//
// What bounds it: the products' instructions.  64 sequences of up to 8192 tokens, 8 key heads of 128
// with 4 query heads each: 82 us, 4.0 TB/s; 79 with every read from L2, 60 without the products;
// masks and byte permutes keep the ALU at 51 %, HMMA is at 25 %.  With two groups a key, 128 registers are
// a few short (32 bytes of spills).  Measured there and not kept: 16 consumer
// warps an SM in place of 12 (each with a ring of its own 93 us; with 96 registers 90; with the
// queries in shared memory 85), the codes' shifts on the multiplier (90), blocks of 16 rows (a fifth
// slower from 16 rows on).
//
// Products on the tensor cores, with the codes as they are: a nibble masked in place is the
// fp16 subnormal c 2^-24 (bits 0-3) or c 2^-20 (bits 4-7), an exact operand, so eight codes cost
// one shift and four masks.  The odd power of two goes to where it is free: for q K^T into the
// query fragment, for P V into the result's row.  Scales and minima stay in fp32, outside the
// products:  q.K_t = s_t (q.c_t) + m_t sum(q),  out = sum_t (w_t s_t) c_t + sum_t w_t m_t.
// Queries become fp16 after their row is scaled by a power of two (nothing is lost from fp16
// or bf16 inputs within 2^-24 of the row's largest); w_t s_t becomes fp16 (2^-11 relative) after a
// power of two taken from the largest s_t seen keeps it within [2^-18, 2^14] for weights
// down to 2^-24 of the row's largest.  So that its rounding acts on the values' spread and not on
// their distance from the minimum, the same rounded weights are also multiplied with a constant
// 8, which is taken from the codes' product and put back in fp32:
//     out = sum_t fp16(w_t s_t) (c_t - 8) + sum_t w_t (m_t + 8 s_t).
//
// Order of the contraction index: lane t of a quad holds G / 4 neighbouring values of a key's
// group, in the order of the nibbles, and the query fragment follows it; token index i of an
// 8-token block is row (i >> 1) + 4 (i & 1), so that the value loads of a quad hit both halves
// of the banks.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "cache_attention.cuh"
#include "cache_partition.h"

namespace w4a16 {

constexpr int kCdWarps = 4;         // consumer warps
constexpr int kCdWarpTokens = kCdTile / kCdWarps;
constexpr int kCdThreads = (kCdWarps + 1) * 32;

// What the producer tells the consumers about a stage.
struct __align__(16) CdStage {
    int tok0;        // first token of the unit
    int row0, head;  // first row of the block, key head
    int flags;       // 1: first unit of this CTA's part of the segment, 2: last, 4: the part is not all of it,
                     // 8: last unit of this CTA; from bit 8 on: rows of the block
    int len, q0;
    int pos0;        // position of the sequence's first query
    int slot;        // workspace slot of the part
};

template <int D, int G>
struct CdCfg {
    using F = CacheFmt<D, G>;
    static constexpr int CODES = kCdTile * F::CODE;
    static constexpr int PAIRS = kCdTile * F::PAIR;
    static constexpr int STAGE = 2 * (CODES + PAIRS);
    static constexpr int ROWS = kCdRows;
    static constexpr int STAGES = D == 64 ? 5 : 3;
    static constexpr int LD = D + 4;                               // floats of a row in the merge buffer
    static constexpr int MERGE = kCdWarps * ROWS * LD * 4;         // [warp][row][LD]: sums, then maximum and sum of weights
    static constexpr int HDR = STAGES * (int)sizeof(CdStage);
    static constexpr int SMEM = STAGES * STAGE + MERGE + HDR + 256;
    static constexpr int CTAS = kCdCtas;
};

// The segments of one sequence.
__device__ __forceinline__ CdShape cd_shape(const AttentionParams& p, const SeqSpan& s) {
    return cd_shape(s.nq, p.shared, s.len, s.pos0, p.window);
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// D(16x8, f32) += A(16x16, f16, row) * B(16x8, f16, col); free to be scheduled.
__device__ __forceinline__ void hmma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void hmma_zero(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}

template <int D, int G>
__global__ void __launch_bounds__(kCdThreads, CdCfg<D, G>::CTAS)
cache_decode_kernel(const __grid_constant__ AttentionParams p) {
    using C = CdCfg<D, G>;
    using F = CacheFmt<D, G>;
    constexpr int NG = F::NG, ST = C::STAGES, ROWS = C::ROWS;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* merge_p = smem + ST * C::STAGE;
    CdStage* hdr = reinterpret_cast<CdStage*>(merge_p + C::MERGE);
    uint64_t* bars = reinterpret_cast<uint64_t*>(hdr + ST);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
    const uint32_t merge_bar = bar0 + 8u * (2 * ST);
    long long* found = reinterpret_cast<long long*>(bars + 2 * ST + 2);    // total units, first sequence's base, sequence
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kCdWarps);
        }
        mbar_init(merge_bar, kCdWarps * 32);
        fence_mbar_init();
    }
    // No early trigger: with one, the waiting combine CTAs get in the way of the next call's CTAs
    // (64 x 8192 tokens, calls back to back: 114 us a call; without 82 us).
    pdl_wait();

    // ---- this CTA's range of units: a scan over the sequences
    const int hk = p.c.kv_heads;
    {
        long long* warp_sum = found + 4;
        const int per = (p.batch + kCdThreads - 1) / kCdThreads;
        const int b0 = min((int)threadIdx.x * per, p.batch), b1 = min(b0 + per, p.batch);
        long long mine = 0;
        for (int b = b0; b < b1; ++b) mine += cd_shape(p, seq_span(p, b)).cost(hk);
        long long incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const long long o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        long long before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < kCdWarps + 1; ++w) {
            if (w < warp) before += warp_sum[w];
            total += warp_sum[w];
        }
        const long long u0 = CdCut(total, (int)gridDim.x).begin(blockIdx.x);
        long long base = before + incl - mine;
        if (threadIdx.x == 0) found[0] = total;
        if (u0 >= base && u0 < base + mine) {
            int b = b0;
            for (; b < b1; ++b) {
                const long long n = cd_shape(p, seq_span(p, b)).cost(hk);
                if (u0 < base + n) break;
                base += n;
            }
            found[1] = base;
            found[2] = b;
        }
        __syncthreads();
    }
    const CdCut cut(found[0], (int)gridDim.x);
    if (blockIdx.x >= cut.ctas) return;

    if (warp == kCdWarps) {
        // ------------------------------------------------------------ producer
        const int ps_log = p.c.page_shift;
        const int rows = min(1 << ps_log, kCdTile);             // tokens of a run
        const int part = lane & 3, run = lane >> 2;             // this lane's copy: K codes, V codes, K pairs, V pairs
        const uint32_t unit_b = part < 2 ? F::CODE : F::PAIR;
        const uint32_t run_bytes = (uint32_t)rows * unit_b;
        const uint32_t dst_off = (part < 2 ? part * C::CODES : 2 * C::CODES + (part - 2) * C::PAIRS) + run * run_bytes;
        const uint32_t src_part = part < 2 ? (uint32_t)(part * F::CODE) << ps_log
                                           : (uint32_t)(2 * F::CODE + (part - 2) * F::PAIR) << ps_log;
        int b = (int)found[2];
        SeqSpan s = seq_span(p, b);
        CdWalk w(cut, blockIdx.x, found[1], cd_shape(p, s));
        bool begins = true;
        int2* info = reinterpret_cast<int2*>(p.workspace);
        if (!w.more() && lane == 0) {                            // a start and no unit: nothing to do
            CdStage h = {};
            h.flags = 8;
            hdr[0] = h;
            mbar_arrive(full(0));
        }
        int st = 0, turn = 0, issued = 0;
        bool ok = true;
        while (w.more()) {
            const int tok0 = (w.sh.first + w.tile) * kCdTile;
            const int tok = tok0 + run * rows;
            const bool valid = run * rows < kCdTile && tok < s.len && tok + rows > seen_lo(p, s.pos0);
            const int64_t page = valid ? page_of(p, b, tok >> ps_log) : 0;
            const uint8_t* src = cache_block(p.c, page, w.head()) + src_part + (uint32_t)(tok & ((1 << ps_log) - 1)) * unit_b;
            const bool got = mbar_wait_sleep(empty(st), (uint32_t)turn ^ 1u, kDevTimeoutCache);
            if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
            const int runs = __popc(__ballot_sync(0xffffffffu, valid)) / 4;
            const bool ends = w.ends();
            if (lane == 0) {
                CdStage h;
                h.tok0 = tok0; h.row0 = w.block() * ROWS; h.head = w.head();
                const int block_rows = min(s.nq * p.shared - h.row0, ROWS);
                h.flags = (begins ? 1 : 0) | (ends ? 2 : 0) | (w.part() ? 4 : 0) | (w.last() ? 8 : 0) | block_rows << 8;
                h.len = s.len; h.pos0 = s.pos0; h.q0 = s.q0;
                h.slot = w.slot((int)blockIdx.x);
                hdr[st] = h;
                if (w.tile == 0)
                    info[((int64_t)b * hk + h.head) * p.row_blocks + w.block()] = make_int2((int)blockIdx.x, cut.cta_before(w.seg0 + w.sh.tiles));
                mbar_arrive_expect_tx(full(st), (uint32_t)(runs * rows * F::TOKEN));
            }
            __syncwarp();
            if (valid) bulk_load(smem_u32(smem + st * C::STAGE) + dst_off, src, run_bytes, full(st));
            ++issued;
            if (++st == ST) { st = 0; turn ^= 1; }
            begins = ends;
            if (w.advance(hk)) {
                CdShape next;
                do { s = seq_span(p, ++b); next = cd_shape(p, s); } while (next.tiles == 0);
                w.follow(next);
            }
        }
        if (!ok) {
            // Error path: the last stages that were issued may still be landing.
            for (int j = max(0, issued - ST); j < issued; ++j)
                mbar_wait(full(j % ST), (uint32_t)(j / ST) & 1u, kDevTimeoutDrain);
        }
        return;
    }

    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    const int krow = (g >> 1) + 4 * (g & 1);                     // cache row of token index g of an 8-token block
    constexpr uint32_t LO = 0x000F000Fu, HI = 0x00F000F0u;
    constexpr int KW = D / 32, VW = D / 64;                      // words of a key / value row that a lane holds
    float* merge = reinterpret_cast<float*>(merge_p);
    uint32_t merge_phase = 0;

    uint32_t qf[2 * KW][2];                                  // query fragments, contraction steps of 16
    float o[4 * VW][4];                                      // sums: (value 2j, rows 2t, 2t+1), (value 2j+1, ...)
    float oc[NG][4];                                         // the same weights times 8
    float m[2], thr[2], sum[2], msum[NG][2];                 // maximum followed, score above which it moves
    float r24[2], qs[NG][2];                             // score = r24 (s (q'.c) + m qs)
    int lo[2], hi[2];
    float vlim = 0.f, vmul = 1.f;                                // s_t <= vlim; w_t s_t vmul is what fp16 holds
    int lo_all = 0, lo_max = 0, hi_min = 0;
    bool wide = false;                                           // some row of the block has huge queries

    const int w0 = warp * kCdWarpTokens;                         // this warp's tokens of a unit
    int st = 0, turn = 0;
    while (true) {
        if (!__all_sync(0xffffffffu, mbar_wait(full(st), (uint32_t)turn, kDevTimeoutCache))) return;
        const CdStage h = hdr[st];
        if (h.flags & 1) {
            // ---- a new segment: queries, masks, empty state
            const int rows = h.flags >> 8;
            const int pos0 = h.pos0, pos_first = pos0 + h.row0 / p.shared;
            lo_all = seen_lo(p, pos_first);
            lo_max = seen_lo(p, pos0 + (h.row0 + rows - 1) / p.shared);
            hi_min = seen_hi(p, pos_first, h.len);
            const int row = g;
            uint4 raw[NG][G / 32];
            uint32_t amax = 0;
#pragma unroll
            for (int a = 0; a < NG; ++a)
#pragma unroll
                for (int j = 0; j < G / 32; ++j) {
                    raw[a][j] = make_uint4(0, 0, 0, 0);
                    if (row < rows)
                        raw[a][j] = __ldg(reinterpret_cast<const uint4*>(
                            p.q + (int64_t)(h.q0 + (h.row0 + row) / p.shared) * p.q_token +
                            (int64_t)(h.head * p.shared + (h.row0 + row) % p.shared) * p.q_head + a * G + t * (G / 4)) + j);
                }
            float f[NG][G / 4];
#pragma unroll
            for (int a = 0; a < NG; ++a)
#pragma unroll
                for (int j = 0; j < G / 32; ++j) {
                    float x[8];
                    if (p.bf16) unpack8<true>(raw[a][j], x);
                    else unpack8<false>(raw[a][j], x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        f[a][8 * j + e] = x[e];
                        amax = max(amax, __float_as_uint(x[e]) & 0x7FFFFFFFu);
                    }
                }
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // the row's power of two: its largest value comes to [2^13, 2^14)
            const int ex = min(max((int)(amax >> 23), 24), 253);
            const float down = __uint_as_float((uint32_t)(267 - ex) << 23 & 0x7F800000u);   // 2^(140 - ex)
            const float back = __uint_as_float((uint32_t)(ex - 13) << 23);                  // 2^(ex - 140)
            float total_q[NG];
#pragma unroll
            for (int a = 0; a < NG; ++a) {
                total_q[a] = 0.f;
#pragma unroll
                for (int e = 0; e < G / 4; ++e) {
                    f[a][e] *= down;
                    total_q[a] += __half2float(__float2half_rn(f[a][e]));
                }
                total_q[a] += __shfl_xor_sync(0xffffffffu, total_q[a], 1);
                total_q[a] += __shfl_xor_sync(0xffffffffu, total_q[a], 2);
#pragma unroll
                for (int w = 0; w < G / 32; ++w) {
                    const float* x = &f[a][8 * w];
                    const int c = 2 * (a * (G / 32) + w);
                    qf[c][0] = pack16(x[0], x[4], false);
                    qf[c][1] = pack16(x[1] * 0.0625f, x[5] * 0.0625f, false);
                    qf[c + 1][0] = pack16(x[2], x[6], false);
                    qf[c + 1][1] = pack16(x[3] * 0.0625f, x[7] * 0.0625f, false);
                }
            }
            // with queries of 2^94 and more 2^16 of the factor goes to the scores first: all of it may pass fp32
            wide = __any_sync(0xffffffffu, ex > 220);
            const float r = back * p.scale_log2 * (wide ? 256.f : 16777216.f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int from = 8 * t + 4 * e, mine = 2 * t + e;
                r24[e] = __shfl_sync(0xffffffffu, r, from);
#pragma unroll
                for (int a = 0; a < NG; ++a) qs[a][e] = __shfl_sync(0xffffffffu, total_q[a], from) * 5.9604644775390625e-8f;
                const int pos = pos0 + (h.row0 + mine) / p.shared;
                hi[e] = mine < rows ? seen_hi(p, pos, h.len) : h.len;
                lo[e] = mine < rows ? seen_lo(p, pos) : 0;
                m[e] = 0.f;
                thr[e] = -INFINITY;                       // nothing seen yet: any score sets the maximum
                sum[e] = 0.f;
#pragma unroll
                for (int a = 0; a < NG; ++a) msum[a][e] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4 * VW; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
#pragma unroll
            for (int a = 0; a < NG; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e) oc[a][e] = 0.f;
            vlim = 0.f;
            vmul = 1.f;
        }

        const int tok = h.tok0 + w0;                             // this warp's first token
        const uint8_t* sp = smem + st * C::STAGE;
        auto step = [&](auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
            uint32_t kw[2][2][KW];                               // [block][token g, g + 8][word]
            __half2 kp[2][2][NG], vp[2][2][NG];                  // (scale, minimum) of this lane's tokens
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = w0 + krow + blk * 16 + e * 8;
#pragma unroll
                    for (int a = 0; a < NG; ++a) {
                        const uint8_t* src = sp + row * F::CODE + t * (G / 8) + a * (G / 2);
                        if constexpr (G == 128) {
                            const uint4 v = *reinterpret_cast<const uint4*>(src);
                            kw[blk][e][0] = v.x; kw[blk][e][1] = v.y; kw[blk][e][2] = v.z; kw[blk][e][3] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(src);
                            kw[blk][e][2 * a] = v.x; kw[blk][e][2 * a + 1] = v.y;
                        }
                        const uint8_t* pr = sp + 2 * C::CODES + row * F::PAIR + a * 4;
                        kp[blk][e][a] = *reinterpret_cast<const __half2*>(pr);
                        vp[blk][e][a] = *reinterpret_cast<const __half2*>(pr + C::PAIRS);
                    }
                }
            // q . codes: four accumulators (two a block, by group or by step), so that few products wait for another
            constexpr int NA = 2 / NG;
            float acc[2][NG][NA][4];
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const int a = w / (G / 32);
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int blk = 0; blk < 2; ++blk) {
                        const uint32_t x0 = q ? kw[blk][0][w] >> 8 : kw[blk][0][w], x1 = q ? kw[blk][1][w] >> 8 : kw[blk][1][w];
                        const uint32_t af[4] = {x0 & LO, x1 & LO, x0 & HI, x1 & HI};
                        if (2 * (w % (G / 32)) + q < NA) hmma_zero(acc[blk][a][q % NA], af, qf[2 * w + q]);
                        else hmma(acc[blk][a][q % NA], af, qf[2 * w + q]);
                    }
            }
            float x[2][4];                                   // [block][..][token g rows 2t, 2t+1; token g+8]
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            float v = 0.f;
#pragma unroll
                            for (int a = 0; a < NG; ++a) {
                                const float c = NA == 2 ? acc[blk][a][0][2 * e + r] + acc[blk][a][NA - 1][2 * e + r] : acc[blk][a][0][2 * e + r];
                                const float sc = __low2float(kp[blk][e][a]), mn = __high2float(kp[blk][e][a]);
                                v = a ? fmaf(sc, c, v) : sc * c;
                                v = fmaf(mn, qs[a][r], v);
                            }
                            x[blk][2 * e + r] = v;
                        }
            // masks: tokens that a row does not see weigh nothing, and what lies past the sequence's
            // end (never written: any bits) must not reach a product
            uint32_t gone = 0;
            if constexpr (MASKED) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int tk = tok + blk * 16 + e * 8 + krow;
                        if (tk >= h.len || tk < lo_all)
#pragma unroll
                            for (int a = 0; a < NG; ++a) vp[blk][e][a] = __half2half2(__ushort_as_half(0));
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                if (tk >= hi[r] || tk < lo[r]) gone |= 1u << (4 * blk + 2 * e + r);
                    }
            }
            if (wide) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[blk][e] *= 65536.f;
            }
            // Scores, rounded to fp32 before the maximum is taken off: the maximum's own difference is then zero at any
            // size (fused, it is what the rounding left, 2^-25 of the score).
            float y[2][4], top[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = __fmul_rn(x[blk][2 * e + r], r24[r]);
                        if constexpr (MASKED)
                            if ((gone >> (4 * blk + 2 * e + r)) & 1u) v = -INFINITY;
                        y[blk][2 * e + r] = v;
                    }
                top[r] = fmaxf(fmaxf(y[0][r], y[0][2 + r]), fmaxf(y[1][r], y[1][2 + r]));
            }
            __half2 vtop = __half2half2(__ushort_as_half(0));
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int a = 0; a < NG; ++a) vtop = __hmax2(vtop, vp[blk][e][a]);
            float vmax = __low2float(vtop);
            bool move = vmax > vlim;
            move |= top[0] > thr[0] || top[1] > thr[1];
            // The maximum moves only when a score passes it by 2^8 (weights stay below 2^8): a few
            // times a segment, so the reductions over the warp and the rescaling are rare.
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, d));
                float vkeep = 1.f;
                if (vmax > vlim) {
                    // the power of two above vmax
                    const float lim = __uint_as_float((__float_as_uint(vmax) & 0x7F800000u) + 0x00800000u);
                    vkeep = vlim / lim;
                    vlim = lim;
                    vmul = 64.f / lim;
                }
                float keep[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float d = top[r];
#pragma unroll
                    for (int k = 4; k < 32; k *= 2) d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, k));
                    const bool fresh = thr[r] == -INFINITY;
                    keep[r] = 1.f;
                    if (d > (fresh ? -INFINITY : m[r])) {
                        keep[r] = fresh ? 0.f : exp2_fast(m[r] - d);
                        m[r] = d;
                        thr[r] = __fadd_rd(d, 8.f);
                    }
                    sum[r] *= keep[r];
#pragma unroll
                    for (int a = 0; a < NG; ++a) msum[a][r] *= keep[r];
                }
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                    oc[a][0] *= keep[0] * vkeep; oc[a][1] *= keep[1] * vkeep;
                    oc[a][2] = oc[a][0]; oc[a][3] = oc[a][1];
                }
#pragma unroll
                for (int j = 0; j < 4 * VW; ++j) {
                    o[j][0] *= keep[0] * vkeep; o[j][1] *= keep[1] * vkeep;
                    o[j][2] *= keep[0] * vkeep; o[j][3] *= keep[1] * vkeep;
                }
            }
            // weights, and their fp16 form in the layout of the product's right operand
            uint32_t pf[2][NG][2];
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float vs[NG], vm[NG];
#pragma unroll
                    for (int a = 0; a < NG; ++a) {
                        const float sv = __low2float(vp[blk][e][a]);
                        vs[a] = sv * vmul;
                        vm[a] = fmaf(8.f, sv, __high2float(vp[blk][e][a]));
                    }
                    const float p0 = exp2_fast(__fsub_rn(y[blk][2 * e], m[0])), p1 = exp2_fast(__fsub_rn(y[blk][2 * e + 1], m[1]));
                    sum[0] += p0;
                    sum[1] += p1;
#pragma unroll
                    for (int a = 0; a < NG; ++a) {
                        msum[a][0] = fmaf(p0, vm[a], msum[a][0]);
                        msum[a][1] = fmaf(p1, vm[a], msum[a][1]);
                        pf[blk][a][e] = movmatrix_trans(pack16(p0 * vs[a], p1 * vs[a], false));
                    }
                }
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                uint32_t vw[4][VW];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint8_t* src = sp + C::CODES + (w0 + t + blk * 16 + 4 * k) * F::CODE + g * (G / 16);
                    if constexpr (G == 128) {
                        const uint2 v = *reinterpret_cast<const uint2*>(src);
                        vw[k][0] = v.x; vw[k][1] = v.y;
                    } else {
#pragma unroll
                        for (int a = 0; a < NG; ++a) vw[k][a] = *reinterpret_cast<const uint32_t*>(src + a * (G / 2));
                    }
                }
                const uint32_t eight[4] = {0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u};   // 8 2^-24 each
#pragma unroll
                for (int a = 0; a < NG; ++a)
                    hmma(oc[a], eight, pf[blk][a]);
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    const int a = w / (G / 64);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t sel = half ? 0x7632u : 0x5410u;
                        uint32_t x01 = __byte_perm(vw[0][w], vw[1][w], sel), x23 = __byte_perm(vw[2][w], vw[3][w], sel);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const uint32_t af[4] = {x01 & LO, x01 & HI, x23 & LO, x23 & HI};
                            hmma(o[4 * w + 2 * half + q], af, pf[blk][a]);
                            x01 >>= 8;
                            x23 >>= 8;
                        }
                    }
                }
            }
        };
        if (tok < h.len && tok + kCdWarpTokens > lo_all) {
            if (tok >= lo_max && tok + kCdWarpTokens <= hi_min) step(std::false_type{});
            else step(std::true_type{});
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(st));
        if (++st == ST) { st = 0; turn ^= 1; }

        if (h.flags & 2) {
            // ---- the end of this CTA's part: the four warps' states become one
            const int rows = h.flags >> 8;
            float* mine = merge + warp * ROWS * C::LD;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = 2 * t + r;
                    float s = sum[r], a0 = msum[0][r], a1 = NG == 2 ? msum[NG - 1][r] : 0.f;
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) {
                        s += __shfl_xor_sync(0xffffffffu, s, d);
                        a0 += __shfl_xor_sync(0xffffffffu, a0, d);
                        if constexpr (NG == 2) a1 += __shfl_xor_sync(0xffffffffu, a1, d);
                    }
                    if (row < rows) {
                        const float up24 = 16777216.f / vmul, up20 = 1048576.f / vmul;
#pragma unroll
                        for (int j = 0; j < 4 * VW; ++j) {
                            const int w = j / 4, a = w / (G / 64);
                            const int d = a * G + g * (G / 8) + (w % (G / 64)) * 8 + 2 * (j % 4);
                            float2 v;
                            v.x = fmaf(o[j][r] - oc[a][r], up24, a ? a1 : a0);
                            v.y = fmaf(fmaf(-16.f, oc[a][r], o[j][2 + r]), up20, a ? a1 : a0);
                            *reinterpret_cast<float2*>(mine + row * C::LD + d) = v;
                        }
                        if (g == 0) {
                            mine[row * C::LD + D] = thr[r] == -INFINITY ? -INFINITY : m[r];
                            mine[row * C::LD + D + 1] = s;
                        }
                    }
                }
            mbar_arrive(merge_bar);
            if (!__all_sync(0xffffffffu, mbar_wait(merge_bar, merge_phase, kDevTimeoutCache))) return;
            merge_phase ^= 1;
            constexpr int V4 = D / 4;
            for (int i = threadIdx.x; i < rows * V4; i += kCdWarps * 32) {
                const int row = i / V4, d = i % V4 * 4;
                const float* src = merge + row * C::LD;
                float mm = -INFINITY, ss = 0.f;
#pragma unroll
                for (int w = 0; w < kCdWarps; ++w) mm = fmaxf(mm, src[w * ROWS * C::LD + D]);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kCdWarps; ++w) {
                    const float* sw = src + w * ROWS * C::LD;
                    // a warp that saw nothing has no maximum, and sums of zero (or NaN, which must stay)
                    const float k = sw[D] == -INFINITY ? 1.f : exp2_fast(sw[D] - mm);
                    const float4 x4 = *reinterpret_cast<const float4*>(sw + d);
                    v.x = fmaf(k, x4.x, v.x); v.y = fmaf(k, x4.y, v.y); v.z = fmaf(k, x4.z, v.z); v.w = fmaf(k, x4.w, v.w);
                    ss = fmaf(k, sw[D + 1], ss);
                }
                if (h.flags & 4) {
                    float* slot = reinterpret_cast<float*>(p.workspace + cd_info_bytes((int64_t)p.batch * hk * p.row_blocks)) +
                                  (size_t)h.slot * cd_slot_floats(D);
                    *reinterpret_cast<float4*>(slot + row * D + d) = v;
                    if (d == 0) {
                        slot[ROWS * D + row] = mm;
                        slot[ROWS * D + ROWS + row] = ss;
                    }
                } else {
                    const float inv = ss == 0.f ? 0.f : 1.f / ss;
                    const int64_t at = (int64_t)(h.q0 + (h.row0 + row) / p.shared) * (hk * p.shared) + h.head * p.shared +
                                       (h.row0 + row) % p.shared;
                    uint2 w2;
                    w2.x = pack16(v.x * inv, v.y * inv, p.bf16);
                    w2.y = pack16(v.z * inv, v.w * inv, p.bf16);
                    *reinterpret_cast<uint2*>(p.out + at * D + d) = w2;
                    if (p.lse && d == 0) p.lse[at] = ss == 0.f ? -INFINITY : (mm + log2f(ss)) * kLn2;
                }
            }
            // the buffer is free again once every warp has read it
            mbar_arrive(merge_bar);
            if (!__all_sync(0xffffffffu, mbar_wait(merge_bar, merge_phase, kDevTimeoutCache))) return;
            merge_phase ^= 1;
        }
        if (h.flags & 8) return;
    }
}

// Joins the parts of the segments that several CTAs held, and writes the zeros of sequences
// with nothing cached and of rows that are not answered.  SLICES groups of D / 4 threads hold a row's values and take every SLICES-th
// part; a block has several rows where few slices do (16 x 5 x 4096 with a block a row: 5.4 us of
// the call's 39).  `seg_rows`: rows of a segment that any sequence has.
template <int D, int SLICES>
__global__ void __launch_bounds__(SLICES == 1 ? 128 : D / 4 * SLICES)
cache_decode_combine_kernel(const __grid_constant__ AttentionParams p, int seg_rows, int64_t rows) {
    constexpr int V4 = D / 4;
    pdl_wait();
    pdl_launch_dependents();
    clear_outside<D>(p, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
    const int lane_d = threadIdx.x % V4, slice = SLICES == 1 ? 0 : threadIdx.x / V4;
    const int64_t r = SLICES == 1 ? (int64_t)blockIdx.x * (128 / V4) + threadIdx.x / V4 : (int64_t)blockIdx.x;
    if (r >= rows) return;
    const int64_t seg = r / seg_rows;
    const int row = (int)(r % seg_rows);
    const int hk = p.c.kv_heads, block = (int)(seg % p.row_blocks), bh = (int)(seg / p.row_blocks), b = bh / hk, head = bh % hk;
    // read along with the lengths: what it says of a segment without units is not used
    const int2 info = *(reinterpret_cast<const int2*>(p.workspace) + seg);
    const SeqSpan s = seq_span(p, b);
    const int whole = block * kCdRows + row;                  // the row among all of the sequence and head
    if (whole == 0 && head == 0) clear_past_max<D>(p, s, slice * V4 + lane_d, SLICES * V4);
    if (whole >= s.nq * p.shared) return;
    const int64_t at = (int64_t)(s.q0 + whole / p.shared) * (hk * p.shared) + head * p.shared + whole % p.shared;
    if (cd_shape(p, s).tiles == 0) {
        if (slice == 0) {
            *reinterpret_cast<uint2*>(p.out + at * D + lane_d * 4) = make_uint2(0u, 0u);
            if (p.lse && lane_d == 0) p.lse[at] = -INFINITY;
        }
        return;
    }
    const int n = info.y - info.x + 1;
    if (n == 1) return;                                    // one CTA had it all and has written it
    const float* slots = reinterpret_cast<const float*>(p.workspace + cd_info_bytes((int64_t)p.batch * hk * p.row_blocks));
    auto part_of = [&](int c) { return slots + (size_t)cd_part_slot(info.x, c) * cd_slot_floats(D); };
    // the row's maximum over the parts
    const uint32_t row_lanes = V4 == 32 ? 0xFFFFFFFFu : 0xFFFFu << (threadIdx.x & 16);
    float mm = -INFINITY;
    for (int c = lane_d; c < n; c += V4) mm = fmaxf(mm, part_of(c)[kCdRows * D + row]);
#pragma unroll
    for (int d = V4 / 2; d; d /= 2) mm = fmaxf(mm, __shfl_xor_sync(row_lanes, mm, d));
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float ss = 0.f;
#pragma unroll 4
    for (int c = slice; c < n; c += SLICES) {
        const float* x = part_of(c);
        const float mc = x[kCdRows * D + row], sc = x[kCdRows * D + kCdRows + row];
        const float4 y = *reinterpret_cast<const float4*>(x + row * D + lane_d * 4);
        const float k = mc == -INFINITY ? 1.f : exp2_fast(mc - mm);      // see the merge above
        v.x = fmaf(k, y.x, v.x); v.y = fmaf(k, y.y, v.y); v.z = fmaf(k, y.z, v.z); v.w = fmaf(k, y.w, v.w);
        ss = fmaf(k, sc, ss);
    }
    if constexpr (SLICES > 1) {
        __shared__ float4 part[V4 * SLICES];
        __shared__ float sums[SLICES];
        part[threadIdx.x] = v;
        if (lane_d == 0) sums[slice] = ss;
        __syncthreads();
        if (slice > 0) return;
        for (int j = 1; j < SLICES; ++j) {
            const float4 y = part[j * V4 + lane_d];
            v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
            ss += sums[j];
        }
    }
    const float inv = ss == 0.f ? 0.f : 1.f / ss;
    uint2 w2;
    w2.x = pack16(v.x * inv, v.y * inv, p.bf16);
    w2.y = pack16(v.z * inv, v.w * inv, p.bf16);
    *reinterpret_cast<uint2*>(p.out + at * D + lane_d * 4) = w2;
    if (p.lse && lane_d == 0) p.lse[at] = ss == 0.f ? -INFINITY : (mm + log2f(ss)) * kLn2;
}

}  // namespace w4a16
