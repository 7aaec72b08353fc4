// Attention of many rows (more than 32 a sequence and key head: prompts, chunks of prompts, long drafts) over the
// 4-bit cache on the tensor cores: tcgen05 products with accumulators in TMEM.  Included by
// cache.cu only.
//
// A CTA takes up to 256 rows (query heads of a key head times queries, in that order) of one
// sequence and key head as two tiles of 128, and walks the 128-token tiles of the cache that
// any of its rows sees:
//     S = Q K^T   (128 x 128, TMEM)  ->  P = 2^(r S - m), fp16, TMEM
//     O += P V    (128 x D, TMEM)
// While the tensor cores work on one half's products, the other half's softmax runs.  With 128
// rows or fewer the halves take alternate tiles of the cache instead, for the same rows; the first
// one's warps join the two results from TMEM.
//
// Warps: 0 issues the products; 1 fetches codes and pairs (bulk copies); 2 clears rows that are not
// answered; 4-7 turn codes and pairs into fp16 operands in shared memory (keys [token][value], values
// transposed [value][token], both K-major with 128-byte swizzle); 8-11 and 12-15 hold one half each, a
// thread a row: they load the queries, run the softmax and write the result.
//
// What bounds it: the chain of a half's step, some 4800 cycles for a 128-token tile of both halves
// where the products alone take 2048 and the exponentials (16 a cycle and SM) as many: scores
// read 180, maximum 370, weights 1800, then 1800 for PV, the next S and the hand-overs between
// warps (100 to 200 each), and the wait for PV before that S (128-wide heads).  512 queries of 64 heads
// over 32768 tokens: 630 to 660 us, 840 TFLOP/s, at the GPU's power limit; a prompt of 4096 (32/8 heads) 189 us.
//
// Measured on those 512 queries and not kept, when this kernel took 660 us: two threads a row (680), a warp
// of its own for the products of each half (765), a PV and the next S issued in one go after all their
// waits (758), a quarter of the exponentials as polynomials on the FMA pipe (792), a second read of the
// scores from TMEM in place of 128 registers (1160); and with no difference: weights handed over in two
// parts, a third S buffer with 64-wide heads, queries and results moved in coalesced rows.
//
// Rounding.  A cached value code * scale + minimum is rounded once to fp16 (2^-11), as a 16-bit
// cache would hold it, which for keys moves a score by some 2^-12 of what its largest channels add.  With
// fp16 outputs and outlier channels the result is 5.5e-4 from 64 bits (1e-3 on other inputs), where the
// decode kernel's is 2.5e-4 and the output's own rounding 2.1e-4; with bf16 outputs 1.8e-3 to 2.0e-3, of
// which their rounding is 1.7e-3.  Measured and not kept: codes as operands, with scales and minima in fp32
// on the scores, give 3.3e-4 but take 223 us where this took 188 (a prompt of 4096), and 951 where it took
// 640 with two groups a key (their scores in two parts); the scores in fragment order, for fewer loads of
// the scales, 232 and 1316.
//
// Queries become fp16 after a power of two (exact within 2^-24 of the row's largest).  Weights are fp16 up to 2^14: the maximum is followed only when a score passes
// it by 2^8, and 2^6 is put on top, so weights down to 2^-20 of the row's largest keep all
// bits.  Sums, maxima and accumulators are fp32.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "cache_attention.cuh"
#include "cache_plan.h"
#include "cache_schedule.h"

namespace w4a16 {

__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// Two fp32 operations in one instruction, on register pairs.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void split2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float v;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}

// Products issued by a whole warp with its values uniform and one elected lane (677 us with a
// branch for one lane where this takes 660).  Descriptors are given by their low words; the high
// word is the same for every operand here: 8-row groups 1024 bytes apart, 128-byte swizzle.
constexpr uint32_t kCpDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t cp_desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | (1u << 16); }

// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
        :: "r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kCpDescHi) : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
        :: "r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kCpDescHi) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        :: "r"(bar) : "memory");
}

template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

// One arrival for a warp whose lanes have all come here.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

constexpr int kCpThreads = 512;

template <int D, int G>
struct CpCfg {
    using F = CacheFmt<D, G>;
    static constexpr int Q_BYTES = kCpRows * D * 2;
    static constexpr int K_BYTES = kCpTile * D * 2;
    static constexpr int V_BYTES = D * kCpTile * 2;
    static constexpr int ST = kCpStages;
    // Codes and pairs as they come from the cache: a slot for the keys or the values of a tile.  Values
    // lie in chunks of 8 tokens with 16 bytes between them: a warp reads 8 chunks at once, and stores
    // 16-byte columns of 8 tokens without conflicts either.  (Unpadded, with 8-way conflicts of the
    // loads, 665 us in the case above; with those of the stores instead, 762 us.)
    static constexpr int RAW_CHUNK = 8 * F::CODE, RAW_PAD = RAW_CHUNK + 16;
    static constexpr int RAW_PAIRS = (kCpTile / 8) * RAW_PAD;      // offset of the pairs
    static constexpr int RAW = RAW_PAIRS + kCpTile * F::PAIR;
    static constexpr int RAWS = 3;
    static constexpr int USED = 1024 + 2 * Q_BYTES + ST * (K_BYTES + V_BYTES) + RAWS * RAW + 256;
    // more than half of the SM's shared memory: one CTA, which owns all of TMEM, on an SM
    static constexpr int SMEM = USED > 116 * 1024 ? USED : 116 * 1024;
    static constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(kCpTile >> 3) << 17) | ((uint32_t)(kCpRows >> 4) << 24);
    static constexpr uint32_t IDESC_O = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kCpRows >> 4) << 24);
};

// The CTA's barriers, 8 bytes each from `base` on, then the word for TMEM's address.
template <int RAWS>
struct CpBars {
    uint32_t base;
    static constexpr int ST = kCpStages;
    __device__ __forceinline__ uint32_t k_full(int s) const { return base + 8u * s; }
    __device__ __forceinline__ uint32_t k_empty(int s) const { return base + 8u * (ST + s); }
    __device__ __forceinline__ uint32_t v_full(int s) const { return base + 8u * (2 * ST + s); }
    __device__ __forceinline__ uint32_t v_empty(int s) const { return base + 8u * (3 * ST + s); }
    __device__ __forceinline__ uint32_t q_full(int h) const { return base + 8u * (4 * ST + h); }
    __device__ __forceinline__ uint32_t s_full(int h) const { return base + 8u * (4 * ST + 2 + h); }
    __device__ __forceinline__ uint32_t p_full(int h) const { return base + 8u * (4 * ST + 4 + h); }
    __device__ __forceinline__ uint32_t o_done(int h) const { return base + 8u * (4 * ST + 6 + h); }
    __device__ __forceinline__ uint32_t r_full(int i) const { return base + 8u * (4 * ST + 8 + i); }
    __device__ __forceinline__ uint32_t r_empty(int i) const { return base + 8u * (4 * ST + 8 + RAWS + i); }
    __device__ __forceinline__ uint32_t done() const { return base + 8u * (4 * ST + 8 + 2 * RAWS); }
    __device__ __forceinline__ uint32_t tmem_slot() const { return done() + 8; }
};

// What cp_products asks for, by a whole warp.
template <int D, int G>
struct CpIssue {
    using C = CpCfg<D, G>;
    const CpBars<C::RAWS> bar;
    const uint32_t tmem, q_lo, k_lo, v_lo;       // operands as descriptors' low words
    const bool kv2;
    __device__ __forceinline__ bool wait(uint32_t b, int turn) const {
        return __all_sync(0xffffffffu, mbar_wait(b, (uint32_t)turn & 1u, kDevTimeoutCache));
    }
    __device__ __forceinline__ bool wait_q(int h) const { return wait(bar.q_full(h), 0); }
    __device__ __forceinline__ bool wait_k(int st, int turn) const { return wait(bar.k_full(st), turn); }
    __device__ __forceinline__ bool wait_v(int st, int turn) const { return wait(bar.v_full(st), turn); }
    __device__ __forceinline__ bool wait_p(int h, int step) const { return wait(bar.p_full(h), step); }
    __device__ __forceinline__ bool wait_o(int h, int step) const { return wait(bar.o_done(h), step); }
    __device__ __forceinline__ void scores(int h, int st) const {
        tc_fence_after();
        const uint32_t qa = q_lo + (kv2 ? 0 : h) * (C::Q_BYTES >> 4), kb = k_lo + st * (C::K_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
            mma_ss(tmem + CpTmem<D>::S(h), qa + (k / 4) * (kCpRows * 128 >> 4) + (k % 4) * 2,
                   kb + (k / 4) * (kCpTile * 128 >> 4) + (k % 4) * 2, C::IDESC_S, k != 0);
    }
    __device__ __forceinline__ void values(int h, int st, int step) const {
        tc_fence_after();
        const uint32_t vb = v_lo + st * (C::V_BYTES >> 4), pt = tmem + CpTmem<D>::P(h);
#pragma unroll
        for (int k = 0; k < kCpTile / 16; ++k)
            mma_ts(tmem + CpTmem<D>::O(h), pt + k * 8, vb + (k / 4) * (D * 128 >> 4) + (k % 4) * 2, C::IDESC_O, k ? 1 : step);
    }
    __device__ __forceinline__ void commit_s(int h) const { mma_commit(bar.s_full(h)); }
    __device__ __forceinline__ void commit_o(int h) const { mma_commit(bar.o_done(h)); }
    __device__ __forceinline__ void commit_k(int st) const { mma_commit(bar.k_empty(st)); }
    __device__ __forceinline__ void commit_v(int st) const { mma_commit(bar.v_empty(st)); }
};

__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// Two codes as fp16 times scale plus minimum, one rounding: w holds them in the low nibbles of
// its halves (high: in bits 4-7).  1024 + c, or 1024 + 16 c, is the half 0x6400 | bits.
__device__ __forceinline__ uint32_t value_lo(uint32_t w, __half2 sc, __half2 mn) {
    const __half2 c = __hadd2(as_half2((w & 0x000F000Fu) | 0x64006400u), __half2half2(__ushort_as_half(0xE400)));
    return as_u32(__hfma2(c, sc, mn));
}
__device__ __forceinline__ uint32_t value_hi(uint32_t w, __half2 sc, __half2 mn) {
    const __half2 c = __hfma2(as_half2((w & 0x00F000F0u) | 0x64006400u), __half2half2(__ushort_as_half(0x2C00)),
                              __half2half2(__ushort_as_half(0xD400)));
    return as_u32(__hfma2(c, sc, mn));
}

template <int D, int G>
__global__ void __launch_bounds__(kCpThreads, 1)
cache_prompt_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ CpGrid gr) {
    using C = CpCfg<D, G>;
    using F = CacheFmt<D, G>;
    constexpr int ST = C::ST;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t qs = base, ks = qs + 2 * C::Q_BYTES, vs = ks + ST * C::K_BYTES, raws = vs + ST * C::V_BYTES,
                   bar0 = raws + C::RAWS * C::RAW;
    const CpBars<C::RAWS> bar{bar0};

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(bar.k_full(s), 4);
            mbar_init(bar.k_empty(s), 1);
            mbar_init(bar.v_full(s), 4);
            mbar_init(bar.v_empty(s), 1);
        }
        for (int h = 0; h < 2; ++h) {
            mbar_init(bar.q_full(h), 4);
            mbar_init(bar.s_full(h), 1);
            mbar_init(bar.p_full(h), 4);
            mbar_init(bar.o_done(h), 1);
        }
        for (int i = 0; i < C::RAWS; ++i) {
            mbar_init(bar.r_full(i), 1);
            mbar_init(bar.r_empty(i), 4);
        }
        mbar_init(bar.done(), 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(bar.tmem_slot(), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (bar.tmem_slot() - raw));
    // No early trigger: the next kernel's waiting CTAs slow this one's down (prompt 4096, calls back to
    // back: 188 us with it, 183 without).
    pdl_wait();

    // ---- this CTA's rows and tiles; the row blocks that see most come first
    const int hk = p.c.kv_heads, heads = hk * p.shared;
    int idx = blockIdx.x;
    const int split = idx % gr.splits; idx /= gr.splits;
    const int head = idx % hk; idx /= hk;
    const int b = idx % p.batch;
    const int block = gr.blocks - 1 - idx / p.batch;
    const SeqSpan s = seq_span(p, b);
    const int block_rows = gr.kv2 ? kCpRows : 2 * kCpRows;
    const int row0 = block * block_rows, rows = min(s.nq * p.shared - row0, block_rows);   // rows <= 0: nothing here
    const int pos_first = s.pos0 + row0 / p.shared, pos_last = s.pos0 + (row0 + max(rows, 1) - 1) / p.shared;
    const int tok_lo = seen_lo(p, pos_first), tok_hi = seen_hi(p, pos_last, s.len);
    int t0 = tok_lo / kCpTile, n = rows > 0 ? max((tok_hi + kCpTile - 1) / kCpTile - t0, 0) : 0;
    {
        const int a = (int)((long long)n * split / gr.splits), e = (int)((long long)n * (split + 1) / gr.splits);
        t0 += a;
        n = e - a;
    }
    const CpWalk walk{n, gr.kv2 ? n > 1 : rows > kCpRows, gr.kv2 != 0};

    if (warp < 4) {
        reg_dec<48>();
        if (warp == 0 && n > 0) {
            // -------------------------------------------------------- products
            CpIssue<D, G> issue{bar, tmem, cp_desc_lo(qs), cp_desc_lo(ks), cp_desc_lo(vs), gr.kv2 != 0};
            cp_products<D>(walk, issue);
            mma_commit(bar.done());         // every product retired before TMEM is released
            mbar_wait(bar.done(), 0, kDevTimeoutDrain);
        } else if (warp == 1) {
            // -------------------------------------------------------- codes and pairs into shared memory
            // Lanes 0-7: the codes of the keys of a run (the part of a page that is in the tile); 8-15: its
            // pairs; 16-31: the codes of the values of a chunk.  Few copies: issuing one takes some 40 cycles.
            const int ps_log = p.c.page_shift, run_rows = min(1 << ps_log, kCpTile);
            const int kind = lane < 8 ? 0 : lane < 16 ? 1 : 2;
            const int rows_c = kind == 2 ? 8 : run_rows, unit = kind == 2 ? lane - 16 : lane & 7;
            const uint32_t row_b = kind == 1 ? F::PAIR : F::CODE, bytes = (uint32_t)rows_c * row_b;
            const uint32_t dst_off = kind == 0 ? unit * bytes : kind == 1 ? C::RAW_PAIRS + unit * bytes : unit * C::RAW_PAD;
            const uint32_t src_off = kind == 0 ? 0u : kind == 1 ? (uint32_t)(2 * F::CODE) << ps_log : (uint32_t)F::CODE << ps_log;
            auto token_of = [&](int tile) {
                const int tok = (t0 + tile) * kCpTile + unit * rows_c;
                return unit * rows_c < kCpTile && tok < s.len && tok + rows_c > tok_lo ? tok : -1;
            };
            bool ok = true;
            int i = 0, slot = 0, turn = 1;
            int tok = n > 0 ? token_of(0) : -1;
            int64_t page = tok >= 0 ? page_of(p, b, tok >> ps_log) : 0;
            for (int tile = 0; tile < n && ok; ++tile) {
                const uint32_t valid = __ballot_sync(0xffffffffu, tok >= 0);
                const bool mine = tok >= 0;
                const uint8_t* src = cache_block(p.c, page, head) + src_off + (uint32_t)(tok & ((1 << ps_log) - 1)) * row_b;
                tok = tile + 1 < n ? token_of(tile + 1) : -1;
                page = tok >= 0 ? page_of(p, b, tok >> ps_log) : 0;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++i) {
                    ok = __all_sync(0xffffffffu, mbar_wait_sleep(bar.r_empty(slot), (uint32_t)turn, kDevTimeoutCache));
                    if (!ok) break;
                    const uint32_t codes = kv ? __popc(valid >> 16) * 8u * F::CODE : __popc(valid & 0xFFu) * (uint32_t)run_rows * F::CODE;
                    const uint32_t pairs = __popc(valid & 0xFF00u) * (uint32_t)run_rows * F::PAIR;
                    if (lane == 0) mbar_arrive_expect_tx(bar.r_full(slot), codes + pairs);
                    __syncwarp();
                    if (mine && kind != (kv ? 0 : 2))
                        bulk_load(raws + slot * C::RAW + dst_off, src + (kv && kind == 1 ? (uint32_t)F::PAIR << ps_log : 0u), bytes,
                                  bar.r_full(slot));
                    if (++slot == C::RAWS) { slot = 0; turn ^= 1; }
                }
            }
            if (!ok)       // what was issued may still be landing
                for (int j = max(0, i - C::RAWS); j < i; ++j) mbar_wait(bar.r_full(j % C::RAWS), (uint32_t)(j / C::RAWS) & 1u, kDevTimeoutDrain);
        } else if (warp == 2) {
            // -------------------------------------------------------- rows that are not answered
            clear_outside<D>(p, (int64_t)blockIdx.x * 32 + lane, (int64_t)gridDim.x * 32);
            if (block == 0 && head == 0 && split == 0) clear_past_max<D>(p, s, lane, 32);
        }
    } else if (warp < 8) {
        // ------------------------------------------------------------ codes -> operands
        reg_dec<80>();
        const int w = warp - 4;
        const int g = lane >> 2, t = lane & 3;
        constexpr int KB = D / 8;                     // bytes of a key that a thread takes: D / 4 values
        constexpr int KWD = KB / 4;                   // in words
        constexpr int DV = D / 8, VWD = DV / 8;       // values of each of 8 tokens that it takes, in words
        const int chunk = lane & 7, dg = (lane >> 3) + 4 * (w >> 1), vtok = (w & 1) * 64 + chunk * 8;
        const int ka = t * (D / 4) / G, va = dg * DV / G;               // groups
        bool ok = true;
        int slot = 0, turn = 0;
        for (int tile = 0; tile < n; ++tile) {
            const int st = tile % ST;
            ok = __all_sync(0xffffffffu, mbar_wait(bar.r_full(slot), (uint32_t)turn, kDevTimeoutCache) &&
                                             mbar_wait(bar.k_empty(st), ((tile / ST) & 1) ^ 1, kDevTimeoutCache));
            if (!ok) break;
            const uint8_t* src = smem_raw + (raws - raw) + slot * C::RAW;
            uint32_t kw[4][KWD], kp[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * 32 + w * 8 + g;
                if constexpr (KWD == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(src + row * F::CODE + t * KB);
                    kw[i][0] = v.x; kw[i][1] = v.y; kw[i][2] = v.z; kw[i][3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2*>(src + row * F::CODE + t * KB);
                    kw[i][0] = v.x; kw[i][1] = v.y;
                }
                kp[i] = *reinterpret_cast<const uint32_t*>(src + C::RAW_PAIRS + row * F::PAIR + ka * 4);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = i * 32 + w * 8 + g;
                const __half2 pr = as_half2(kp[i]);
                const __half2 sc = __low2half2(pr), mn = __high2half2(pr);
                uint8_t* dst = smem_raw + (ks - raw) + st * C::K_BYTES + row * 128;
#pragma unroll
                for (int j = 0; j < KWD; ++j) {
                    const uint32_t x = kw[i][j], z = x >> 8;
                    uint4 o;
                    o.x = value_lo(x, sc, mn); o.y = value_hi(x, sc, mn);
                    o.z = value_lo(z, sc, mn); o.w = value_hi(z, sc, mn);
                    const int c = t * KWD + j;                           // 16-byte chunk of the token's row
                    *reinterpret_cast<uint4*>(dst + (c / 8) * (kCpTile * 128) + (((c % 8) ^ (row & 7)) * 16)) = o;
                }
            }
            fence_proxy_async_smem();
            warp_arrive(bar.k_full(st));
            warp_arrive(bar.r_empty(slot));
            if (++slot == C::RAWS) { slot = 0; turn ^= 1; }
            ok = __all_sync(0xffffffffu, mbar_wait(bar.r_full(slot), (uint32_t)turn, kDevTimeoutCache) &&
                                             mbar_wait(bar.v_empty(st), ((tile / ST) & 1) ^ 1, kDevTimeoutCache));
            if (!ok) break;
            src = smem_raw + (raws - raw) + slot * C::RAW;
            uint32_t vw[8][VWD], vp[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint8_t* at = src + (vtok / 8) * C::RAW_PAD + k * F::CODE + dg * (DV / 2);
                if constexpr (VWD == 2) {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    vw[k][0] = v.x; vw[k][1] = v.y;
                } else {
                    vw[k][0] = *reinterpret_cast<const uint32_t*>(at);
                }
            }
            {
                const uint4* at = reinterpret_cast<const uint4*>(src + C::RAW_PAIRS + vtok * F::PAIR);
                if constexpr (F::NG == 1) {
                    const uint4 v0 = at[0], v1 = at[1];
                    vp[0] = v0.x; vp[1] = v0.y; vp[2] = v0.z; vp[3] = v0.w;
                    vp[4] = v1.x; vp[5] = v1.y; vp[6] = v1.z; vp[7] = v1.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint4 v = at[k];
                        vp[2 * k] = va ? v.y : v.x;
                        vp[2 * k + 1] = va ? v.w : v.z;
                    }
                }
            }
            const int tok = (t0 + tile) * kCpTile + vtok;
            if (tok < tok_lo || tok + 8 > s.len) {
                // a row past the end, or below what is seen, may never have been written
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (tok + k >= s.len || tok + k < tok_lo) vp[k] = 0u;
            }
            {
                __half2 sc[4], mn[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sc[k] = as_half2(__byte_perm(vp[2 * k], vp[2 * k + 1], 0x5410));
                    mn[k] = as_half2(__byte_perm(vp[2 * k], vp[2 * k + 1], 0x7632));
                }
                uint8_t* dst = smem_raw + (vs - raw) + st * C::V_BYTES + (vtok / 64) * (D * 128);
#pragma unroll
                for (int j = 0; j < VWD; ++j)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = __byte_perm(vw[2 * k][j], vw[2 * k + 1][j], hf ? 0x7632 : 0x5410);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int d = dg * DV + j * 8 + hf * 4 + q;
                            uint32_t o[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t y = q >= 2 ? x[k] >> 8 : x[k];
                                o[k] = q & 1 ? value_hi(y, sc[k], mn[k]) : value_lo(y, sc[k], mn[k]);
                            }
                            *reinterpret_cast<uint4*>(dst + d * 128 + ((chunk ^ (d & 7)) * 16)) = make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
            }
            fence_proxy_async_smem();
            warp_arrive(bar.v_full(st));
            warp_arrive(bar.r_empty(slot));
            if (++slot == C::RAWS) { slot = 0; turn ^= 1; }
        }
    } else {
        // ------------------------------------------------------------ softmax: a thread a row
        reg_inc<192>();
        const int h = (warp - 8) >> 2;
        const int r_in = (warp & 3) * 32 + lane;                       // row of the half = TMEM lane
        const int row = row0 + (gr.kv2 ? 0 : h * kCpRows) + r_in;      // row of the (sequence, key head)
        const bool live = row < row0 + rows;
        const int token = live ? row / p.shared : 0, qh = live ? head * p.shared + row % p.shared : 0;
        const int64_t at = (int64_t)(s.q0 + token) * heads + qh;       // row of out
        const bool warp_live = row - lane < row0 + rows;               // some row of the warp is real
        const int steps = walk.steps(h);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_t = tmem + lanes + CpTmem<D>::S(h), p_t = tmem + lanes + CpTmem<D>::P(h), o_t = tmem + lanes + CpTmem<D>::O(h);
        float r = 1.f;
        if (steps > 0 && (h == 0 || !gr.kv2)) {
            // the row's queries, scaled by a power of two: the largest comes to [2^13, 2^14).  Values of a
            // group of eight go in the order in which the keys' nibbles come out: 0 4 1 5 2 6 3 7.
            const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(s.q0 + token) * p.q_token + (int64_t)qh * p.q_head);
            uint4 v[D / 8];
            uint32_t amax = 0;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) v[j] = live ? __ldg(src + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
                float x[8];
                if (p.bf16) unpack8<true>(v[j], x);
                else unpack8<false>(v[j], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7FFFFFFFu);
            }
            const int ex = min(max((int)(amax >> 23), 24), 253);
            float down = __uint_as_float((uint32_t)(267 - ex) << 23);                  // 2^(140 - ex)
            r = __uint_as_float((uint32_t)(ex - 13) << 23) * fabsf(p.scale_log2);      // 2^(ex - 140) ...
            if (p.scale_log2 < 0.f) down = -down;
            uint8_t* dst = smem_raw + (qs - raw) + h * C::Q_BYTES + r_in * 128;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
                float x[8];
                if (p.bf16) unpack8<true>(v[j], x);
                else unpack8<false>(v[j], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= down;
                const uint4 o = make_uint4(pack16(x[0], x[4], false), pack16(x[1], x[5], false), pack16(x[2], x[6], false),
                                           pack16(x[3], x[7], false));
                *reinterpret_cast<uint4*>(dst + (j / 8) * (kCpRows * 128) + (((j % 8) ^ (r_in & 7)) * 16)) = o;
            }
            fence_proxy_async_smem();
            warp_arrive(bar.q_full(h));
        }
        if (gr.kv2) {
            // both halves hold the same rows: the second takes the first's factors
            float* fac = reinterpret_cast<float*>(smem_raw + (qs - raw) + C::Q_BYTES);    // the second half's queries are not used
            if (h == 0) fac[r_in] = r;
            bar_sync_named(1, 256);
            r = fac[r_in];
        }
        r = fmaxf(r, 1e-37f);                                          // never zero: a masked score is -inf * r
        const int pos = s.pos0 + token;
        const int hi = live ? seen_hi(p, pos, s.len) : s.len, lo = live ? seen_lo(p, pos) : 0;
        float m = 0.f, l = 0.f;
        bool fresh = true;                                             // no score seen yet
        bool large = false;                                            // some row's maximum of the warp is
        const int row_a = row - r_in, row_e = min(row_a + kCpRows, row0 + rows) - 1;
        const int in_hi = seen_hi(p, s.pos0 + row_a / p.shared, s.len);      // every row of the half sees [in_lo, in_hi)
        const int in_lo = seen_lo(p, s.pos0 + max(row_e, 0) / p.shared);
        bool ok = true;
        for (int step = 0; step < steps; ++step) {
            const int tile = t0 + (gr.kv2 && walk.two ? 2 * step + h : step);
            ok = __all_sync(0xffffffffu, mbar_wait(bar.s_full(h), step & 1, kDevTimeoutCache));
            if (!ok) break;
            tc_fence_after();
            const int k0 = tile * kCpTile;
            // The tile's weights; false, with nothing changed, where the plain form does not do.
            auto weights = [&](auto careful) {
                constexpr bool CAREFUL = decltype(careful)::value;         // masks, and scores of any size
                uint32_t x[kCpTile];
#pragma unroll
                for (int c = 0; c < kCpTile; c += 32) tmem_ld_x32(s_t + c, x + c);
                tc_wait_ld();
                if constexpr (CAREFUL) {
                    // One comparison a score and side that needs one (12 heads, window 700, with both sides
                    // compared in every tile at an end: 61 us against 57).
                    const int from = lo - k0, to = hi - k0;
                    if (k0 + kCpTile > in_hi) {
#pragma unroll
                        for (int c = 0; c < kCpTile; ++c)
                            if (c >= to) x[c] = 0xFF800000u;
                    }
                    if (k0 < in_lo) {
#pragma unroll
                        for (int c = 0; c < kCpTile; ++c)
                            if (c < from) x[c] = 0xFF800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kCpTile; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1]));
                const float top = __fmul_rn(fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), r);
                const bool move = fresh ? top > -INFINITY : top > __fadd_rd(m, 8.f);
                if (__any_sync(0xffffffffu, move)) {
                    // a large maximum: see below
                    large = __any_sync(0xffffffffu, fabsf(move ? top : m) > 1048576.f);
                    if (!CAREFUL && large) return false;
                    float keep = 1.f;
                    if (move) {
                        keep = fresh ? 0.f : exp2_fast(m - top);
                        m = top;
                        fresh = false;
                    }
                    l *= keep;
                    if (step > 0) {             // this S was committed after the last step's PV: O is at rest
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld_x32(o_t + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st_x32(o_t + c, o);
                        }
                    }
                }
                uint64_t r2 = pair2(r, r), off2 = pair2(6.f - m, 6.f - m);
                if (CAREFUL && large) {
                    // Scores are rounded before the maximum is taken off, as the maximum was: fused, the maximum's own difference
                    // is what the rounding left, 2^-25 of the score.
#pragma unroll
                    for (int c = 0; c < kCpTile; ++c) x[c] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(x[c]), r), m));
                    r2 = pair2(1.f, 1.f);
                    off2 = pair2(6.f, 6.f);
                }
                uint64_t sum2[2] = {pair2(0.f, 0.f), pair2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float p0, p1;
                        split2(fma2(pair2(__uint_as_float(x[32 * c + 2 * e]), __uint_as_float(x[32 * c + 2 * e + 1])), r2, off2), p0, p1);
                        p0 = exp2_fast(p0);
                        p1 = exp2_fast(p1);
                        sum2[e & 1] = add2(sum2[e & 1], pair2(p0, p1));
                        pk[e] = pack16(p0, p1, false);
                    }
                    tmem_st_x16(p_t + 16 * c, pk);
                }
                tc_wait_st();
                tc_fence_before();
                warp_arrive(bar.p_full(h));
                float a0, a1, b0, b1;
                split2(sum2[0], a0, a1);
                split2(sum2[1], b0, b1);
                l += (a0 + a1) + (b0 + b1);
                return true;
            };
            if (warp_live) {
                if (large || k0 < in_lo || k0 + kCpTile > in_hi || !weights(std::false_type{})) weights(std::true_type{});
            } else {
                warp_arrive(bar.p_full(h));
            }
        }
        if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(bar.o_done(h), walk.last_o<D>(h) & 1, kDevTimeoutCache));
        // ---- results
        float keep = 1.f, other = 0.f;                                 // factors of this half's result and of the second's
        if (gr.kv2) {
            float* ml = reinterpret_cast<float*>(smem_raw + (qs - raw) + C::Q_BYTES) + kCpRows;    // behind the factors
            if (h == 1) { ml[r_in] = fresh ? -INFINITY : m; ml[kCpRows + r_in] = l; }
            bar_sync_named(1, 256);
            if (h == 0 && walk.steps(1) > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar.o_done(1), walk.last_o<D>(1) & 1, kDevTimeoutCache)) && ok;
                const float m1 = ml[r_in], top = fresh ? m1 : fmaxf(m, m1);
                // a half that saw nothing has sums of zero (or NaN, which must stay)
                keep = fresh ? 1.f : exp2_fast(m - top);
                other = m1 == -INFINITY ? 1.f : exp2_fast(m1 - top);
                l = fmaf(l, keep, ml[kCpRows + r_in] * other);
                fresh = top == -INFINITY;
                m = top;
            }
        }
        if (ok && warp_live && rows > 0 && !(gr.kv2 && h == 1)) {
            tc_fence_after();
            const int64_t all = p.q_tokens * heads;
            float* po = reinterpret_cast<float*>(p.workspace) + ((int64_t)split * all + at) * D;
            float* pm = reinterpret_cast<float*>(p.workspace) + (int64_t)gr.splits * all * D + ((int64_t)split * all + at) * 2;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const bool joined = gr.kv2 && walk.steps(1) > 0;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (steps > 0) {
                    tmem_ld_x32(o_t + c, o);
                    tc_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (joined) {
                    uint32_t o1[32];
                    tmem_ld_x32(tmem + lanes + CpTmem<D>::O(1) + c, o1);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        o[e] = __float_as_uint(fmaf(__uint_as_float(o[e]), keep, __uint_as_float(o1[e]) * other));
                }
                if (live && gr.splits == 1) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float f[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(o[e + k]) * inv;
                        *reinterpret_cast<uint4*>(p.out + at * D + c + e) = p.bf16 ? pack8<true>(f) : pack8<false>(f);
                    }
                } else if (live) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(po + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (live && gr.splits == 1) {
                if (p.lse) p.lse[at] = l == 0.f ? -INFINITY : (m - 6.f + log2f(l)) * kLn2;
            } else if (live) {
                pm[0] = fresh ? -INFINITY : m;
                pm[1] = l;
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

// Joins the parts of each row.  Grid (rows of the longest sequence, sequence); D / 4 threads a row.
template <int D>
__global__ void __launch_bounds__(128) cache_prompt_combine_kernel(const __grid_constant__ AttentionParams p, int parts) {
    constexpr int V4 = D / 4;
    pdl_wait();
    pdl_launch_dependents();
    const int heads = p.c.kv_heads * p.shared;
    const SeqSpan s = seq_span(p, blockIdx.y);
    const int64_t i = (int64_t)blockIdx.x * (128 / V4) + threadIdx.x / V4;
    if (i >= (int64_t)s.nq * heads) return;
    const int64_t all = p.q_tokens * heads, at = (int64_t)s.q0 * heads + i;
    const int d = threadIdx.x % V4 * 4;
    const float* po = reinterpret_cast<const float*>(p.workspace) + at * D + d;
    const float* pm = reinterpret_cast<const float*>(p.workspace) + (int64_t)parts * all * D + at * 2;
    float mm = -INFINITY;
    for (int c = 0; c < parts; ++c) mm = fmaxf(mm, pm[c * all * 2]);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float ss = 0.f;
#pragma unroll 4
    for (int c = 0; c < parts; ++c) {
        const float2 ml = *reinterpret_cast<const float2*>(pm + c * all * 2);
        const float4 y = *reinterpret_cast<const float4*>(po + c * all * D);
        const float k = ml.x == -INFINITY ? 1.f : exp2_fast(ml.x - mm);        // nothing seen: zeros (or NaN, which must stay)
        v.x = fmaf(k, y.x, v.x); v.y = fmaf(k, y.y, v.y); v.z = fmaf(k, y.z, v.z); v.w = fmaf(k, y.w, v.w);
        ss = fmaf(k, ml.y, ss);
    }
    const float inv = ss == 0.f ? 0.f : 1.f / ss;
    uint2 w2;
    w2.x = pack16(v.x * inv, v.y * inv, p.bf16);
    w2.y = pack16(v.z * inv, v.w * inv, p.bf16);
    *reinterpret_cast<uint2*>(p.out + at * D + d) = w2;
    if (p.lse && d == 0) p.lse[at] = ss == 0.f ? -INFINITY : (mm - 6.f + log2f(ss)) * kLn2;
}

}  // namespace w4a16
