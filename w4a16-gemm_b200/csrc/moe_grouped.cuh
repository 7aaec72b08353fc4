// The products of an expert layer with many entries an expert: rows sorted by expert, each multiplied by its expert's
// 4-bit weight on the fifth-generation tensor cores.  Included by kernels.cu only.
//
//     D_g[n, row] (TMEM, fp32) = sum over group g's k of (q[n, k] - 8) (A, TMEM, fp16, exact) * x[row, k] (B, shared memory)
//     sum[n, row] (registers, fp32) += scale[g, n] * D_g[n, row]
//
// The shape of prefill.cuh's kernel (its warp roles and rings are described there) with one difference: the weights are
// not rounded.  A group's products are made of the exact integers q - 8 in one of two accumulators, and the warps
// that drain it multiply by the group's scale, one number a lane, while the tensor cores fill the other: the scale costs one
// FMA for 64 or 128 products, the dequantising warps 9 instructions a word instead of 13, and what a tile leaves in
// registers needs no accumulator, so that the next tile's products run through its epilogue.
//
// Tiles of 64 rows and 128 channels, two CTAs an SM, each with half of TMEM (two accumulators, two slots of A) and its own
// chain of copies, operands, products and sums: a stage of one chain takes about 0.8 us whatever its tile, so two chains
// were worth more than tiles of twice the rows (16 entries an expert: 64 experts of 2048 x 1408 165 us where one CTA with
// 128 rows took 242; 192 entries: the same).  A tile's rows come from a list; a tile of fewer rows is multiplied as the
// narrowest product that holds them.  A stage is two 64-wide K chunks in two copies, rows and words.
//
// Bound by the hand-overs of a chain, not by the tensor cores (leaving out three products of four: 518 -> 444 us, and the
// drains: 463).  With groups of 128 by the issuing warp (2100 clocks a stage when one lane polled its barriers one after
// the other; three lanes at once, one commit less and one descriptor: 192 entries an expert 517 -> 462 us, 441 today), with
// groups of 64 by the drain, 630 clocks of its warps' own for each 64 K (571 us).  The other shapes, one CTA of 128 rows and one chain of
// 64 rows and 256 channels (582), were timed before the issuing warp was shortened, which they have more of a tile for, and
// not since.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "dequant.cuh"
#include "epilogue.cuh"
#include "internal.h"
#include "launch.cuh"
#include "prefill.cuh"
#include "ptx.cuh"

namespace w4a16 {

constexpr int kMgDqWarps = 4;                                      // each two n16 blocks of the tile
constexpr int kMgEpiWarp0 = 2 + kMgDqWarps, kMgEpiWarps = 8;       // each 32 channels, half of the rows
constexpr int kMgThreads = (kMgEpiWarp0 + kMgEpiWarps) * 32;

struct MgCfg {
    static constexpr int TOK = kMoeGroupedRows;                    // rows of a tile, at most
    static constexpr int KCH = 2;                                  // 64-wide K chunks of a stage
    static constexpr int X_BYTES = KCH * TOK * 128;                // [chunk][row][128 B], 128-byte swizzle
    static constexpr int W_BYTES = KCH * kPfWBytes;                // [n16 block][chunk][512 B]
    static constexpr int STAGE = X_BYTES + W_BYTES;
    static constexpr int STAGES = 4;
    static constexpr int TMEM = 256;                               // columns: half of an SM's
    static constexpr int A_COL0 = 2 * TOK, A_COLS = 32 * KCH;      // two accumulators, then the A ring
    static constexpr int A_STAGES = (TMEM - A_COL0) / A_COLS;
    static constexpr int SMEM = 1024 + STAGES * STAGE + 1024;
    static_assert(STAGE % 1024 == 0 && SMEM <= 113 * 1024 && SMEM > 76 * 1024, "two CTAs an SM, no third");
    static_assert(TOK == 64 && A_STAGES == 2, "TMEM");
};

struct MgTile {
    int expert, row0, rows, tn;
};
__device__ __forceinline__ MgTile mg_tile(int tile, int n_tiles, const MoeGroups& g) {
    const int4 v = __ldcg(reinterpret_cast<const int4*>(g.tiles) + tile / n_tiles);
    return {v.x, v.y, v.z, tile % n_tiles};
}

template <int G, bool GATED>
__global__ void __launch_bounds__(kMgThreads, 2)
moe_grouped_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const __half* __restrict__ scales, void* __restrict__ yv, int N, int K,
                   int activation, MoeGroups groups)
{
    using C = MgCfg;
    constexpr int ST = C::STAGES, NA = C::A_STAGES, TOK = C::TOK;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const uint32_t bar0 = base + ST * C::STAGE;
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
    auto afull = [&](int a) { return bar0 + 8u * (2 * ST + a); };
    auto aempty = [&](int a) { return bar0 + 8u * (2 * ST + NA + a); };
    auto accfull = [&](int b) { return bar0 + 8u * (2 * ST + 2 * NA + b); };
    auto accempty = [&](int b) { return bar0 + 8u * (2 * ST + 2 * NA + 2 + b); };
    const uint32_t done_bar = bar0 + 8u * (2 * ST + 2 * NA + 4);
    const uint32_t tmem_slot = done_bar + 8u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kMgDqWarps);       // the dequantising warps, for the MMAs too
        }
        for (int a = 0; a < NA; ++a) {
            mbar_init(afull(a), kMgDqWarps);
            mbar_init(aempty(a), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(accfull(b), 1);
            mbar_init(accempty(b), kMgEpiWarps);
        }
        mbar_init(done_bar, 1);
        fence_mbar_init();
        prefetch_tmap(&tm_x);
        prefetch_tmap(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - raw));

    pdl_wait();
    pdl_launch_dependents();

    const int n_tiles = (N + kPfRows - 1) / kPfRows;
    const int total = n_tiles * __ldcg(&groups.head->tiles);
    const int KC = K >> 6, KB = KC < C::KCH ? KC : C::KCH, KT = (KC + C::KCH - 1) / C::KCH;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                const MgTile t = mg_tile(tile, n_tiles, groups);
                for (int kt = 0; kt < KT; ++kt, ++it) {
                    const int s = it % ST;
                    if (!mbar_wait(empty(s), ((it / ST) & 1) ^ 1, kDevTimeoutExperts)) { ok = false; break; }
                    const uint32_t sb = base + s * C::STAGE;
                    mbar_arrive_expect_tx(full(s), (uint32_t)(KB * (TOK * 128 + kPfWBytes)));
                    tma_load_3d(sb, &tm_x, 0, t.row0, kt * C::KCH, full(s));
                    tma_load_3d(sb + C::X_BYTES, &tm_w, 0, kt * C::KCH, t.expert * groups.blocks + t.tn * 8, full(s));
                }
            }
            if (!ok)      // the last stages that were issued may still be landing
                for (int j = max(0, it - ST); j < it; ++j) mbar_wait(full(j % ST), (j / ST) & 1, kDevTimeoutExperts);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        // This warp's instructions are what a stage waits for, so they are few: a stage's three barriers are polled by three
        // lanes at once, and one descriptor is counted up (its 14 address bits never carry).
        int it = 0, gi = 0;
        bool ok = true;
        const uint64_t desc0 = pf_sw128_desc(base);
        const auto products = [&](int s, int a, int j, uint32_t idesc, bool first) {      // of one chunk
            const uint32_t d = tmem + (uint32_t)((gi & 1) * TOK), at = tmem + (uint32_t)(C::A_COL0 + a * C::A_COLS + j * 32);
            const uint64_t x = desc0 + (uint32_t)((s * C::STAGE + j * TOK * 128) >> 4);
#pragma unroll
            for (int k16 = 0; k16 < 4; ++k16) tc_mma_ts(d, at + k16 * 8, x + k16 * 2, idesc, !(first && k16 == 0));
        };
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
            const MgTile t = mg_tile(tile, n_tiles, groups);
            const uint32_t idesc = (pf_idesc<TOK>() & ~(63u << 17)) | ((uint32_t)((t.rows + 15) / 16 * 2) << 17);
            for (int kt = 0; kt < KT; ++kt, ++it) {
                const int s = it % ST, a = it % NA;
                const bool both = kt * C::KCH + 1 < KC;
                const uint32_t bar = lane == 0 ? full(s) : lane == 1 ? afull(a) : accempty(gi & 1);
                const uint32_t parity = lane == 0 ? (it / ST) & 1 : lane == 1 ? (it / NA) & 1 : ((gi >> 1) & 1) ^ 1;
                ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, kDevTimeoutExperts));
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    products(s, a, 0, idesc, true);
                    if (G == 128) products(s, a, 1, idesc, false);      // K has whole groups
                    tc_commit(accfull(gi & 1));
                }
                ++gi;
                if (G == 64 && both) {
                    ok = __all_sync(0xffffffffu, mbar_wait(accempty(gi & 1), ((gi >> 1) & 1) ^ 1, kDevTimeoutExperts));
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        products(s, a, 1, idesc, true);
                        tc_commit(accfull(gi & 1));
                    }
                    ++gi;
                }
                if (lane == 0) tc_commit(aempty(a));
            }
        }
        if (lane == 0) {
            tc_commit(done_bar);   // every MMA of this CTA retired before TMEM is released
            mbar_wait(done_bar, 0, kDevTimeoutExperts);
        }
    } else if (warp < kMgEpiWarp0) {
        // ------------------------------------------------------------ codes -> TMEM A ring (q - 8, exact)
        const int nbl = 2 * (warp & 3);                             // first n16 block inside the tile
        const uint32_t lane_field = (uint32_t)(16 * nbl) << 16;
        int it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
            for (int kt = 0; kt < KT; ++kt, ++it) {
                const int s = it % ST, a = it % NA;
                bool w_ok = mbar_wait(full(s), (it / ST) & 1, kDevTimeoutExperts);
                w_ok = w_ok && mbar_wait(aempty(a), ((it / NA) & 1) ^ 1, kDevTimeoutExperts);
                if (!__all_sync(0xffffffffu, w_ok)) { ok = false; break; }
                tc_fence_after();
                const int nch = KC - kt * C::KCH < C::KCH ? KC - kt * C::KCH : C::KCH;
                const uint32_t sbw = base + s * C::STAGE + C::X_BYTES;
                uint4 w[2][C::KCH];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < C::KCH; ++j)
                        if (j < nch) w[b][j] = lds128(sbw + (uint32_t)(((nbl + b) * KB + j) * 512 + lane * 16));
                // the products of the stage whose A slot this is are done, and so is everyone with that stage
                __syncwarp();
                if (lane == 0 && it >= NA) mbar_arrive(empty((it - NA) % ST));
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < C::KCH; ++j)
                        if (j < nch) {
                            uint32_t r[16];
                            unscaled_word(w[b][j].x, *reinterpret_cast<uint32_t(*)[4]>(&r[0]));
                            unscaled_word(w[b][j].y, *reinterpret_cast<uint32_t(*)[4]>(&r[4]));
                            unscaled_word(w[b][j].z, *reinterpret_cast<uint32_t(*)[4]>(&r[8]));
                            unscaled_word(w[b][j].w, *reinterpret_cast<uint32_t(*)[4]>(&r[12]));
                            tmem_st_16x128b_x8(tmem + lane_field + ((uint32_t)(16 * b) << 16) +
                                                   (uint32_t)(C::A_COL0 + a * C::A_COLS + j * 32), r);
                        }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(afull(a));
            }
        }
    } else {
        // ------------------------------------------------------------ scaled sums, epilogue
        // warp (quarter q, part h) owns output channels 32q .. 32q + 31 of the tile (TMEM lanes) and rows 32h .. 32h + 31
        constexpr int CW = TOK / (kMgEpiWarps / 4);
        const int q = warp & 3, h = (warp - kMgEpiWarp0) >> 2;
        const uint32_t tcol = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(h * CW);
        const int scale_groups = K / G;
        int gi = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
            const MgTile t = mg_tile(tile, n_tiles, groups);
            const int n = t.tn * kPfRows + 32 * q + lane;
            const bool rows_here = h * CW < t.rows;
            const __half* const s_at = scales + (int64_t)t.expert * groups.scale_rows * N + min(n, N - 1);
            float sum[CW];
#pragma unroll
            for (int i = 0; i < CW; ++i) sum[i] = 0.f;
            // scales two groups ahead: a group takes less time than a load from L2
            __half next = __ldg(s_at), after = scale_groups > 1 ? __ldg(s_at + N) : next;
            for (int g = 0; g < scale_groups; ++g, ++gi) {
                const float scale = __half2float(next);
                next = after;
                if (g + 2 < scale_groups) after = __ldg(s_at + (int64_t)(g + 2) * N);
                ok = __all_sync(0xffffffffu, mbar_wait(accfull(gi & 1), (gi >> 1) & 1, kDevTimeoutExperts));
                if (!ok) break;
                tc_fence_after();
                if (rows_here) {
                    const uint32_t at = tcol + (uint32_t)((gi & 1) * TOK);
                    uint32_t r[CW];       // all of the warp's columns in one wait
                    tmem_ld_cols<16>(at, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
                    tmem_ld_cols<16>(at + 16, *reinterpret_cast<uint32_t(*)[16]>(&r[16]));
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < CW; ++i) sum[i] = fmaf(scale, __uint_as_float(r[i]), sum[i]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(accempty(gi & 1));
            }
            if (!ok || !rows_here) continue;
            const int row = t.row0 + h * CW, end = t.row0 + t.rows;
            if constexpr (GATED) {
                // lanes l and l + 8 of a half warp hold the two factors: of each pair of rows the gate's lane makes the
                // first one's result, the other lane the second one's (see prefill.cuh).  Which activation it is is asked
                // once, not for every value (2048 tokens of 6 of 64: groups of 64 588 -> 571 us, of 128 456 -> 441).
                const bool up = lane >> 3 & 1;
                uint32_t hv[CW / 4];
#pragma unroll
                for (int i = 0; i < CW / 2; ++i) {
                    const float z0 = sum[2 * i], z1 = sum[2 * i + 1];
                    const float got = __shfl_xor_sync(0xffffffffu, up ? z0 : z1, 8);
                    sum[2 * i] = up ? got : z0;
                    sum[2 * i + 1] = up ? z1 : got;
                }
                if (activation == W4A16_ACTIVATION_SILU) {
#pragma unroll
                    for (int i = 0; i < CW / 2; ++i) sum[2 * i] = times_sigmoid(sum[2 * i], sum[2 * i]);
                } else {
#pragma unroll
                    for (int i = 0; i < CW / 2; ++i) sum[2 * i] = activate(sum[2 * i], activation);
                }
#pragma unroll
                for (int i = 0; i < CW / 4; ++i) {
                    const __half2 p = __floats2half2_rn(sum[4 * i] * sum[4 * i + 1], sum[4 * i + 2] * sum[4 * i + 3]);
                    hv[i] = *reinterpret_cast<const uint32_t*>(&p);
                }
                store_gated<CW>(hv, static_cast<__half*>(yv), row, end, n, N);
            } else if (n < N) {
                float* const y = static_cast<float*>(yv) + (size_t)row * N + n;
#pragma unroll
                for (int i = 0; i < CW; ++i)
                    if (row + i < end) __stcg(y + (size_t)i * N, sum[i]);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, C::TMEM);
}

// ------------------------------------------------------------------ host side
// x [K/64][rows][64] in boxes of a stage's chunks and a tile's rows; the experts' words as one tall weight [experts * N /
// 16][K/64][128] in boxes of 8 blocks.
cudaError_t make_grouped_tensor_maps(const GroupedArgs& a, CUtensorMap* tx, CUtensorMap* tw);

template <int G, bool GATED>
static cudaError_t launch_grouped_t(const GroupedArgs& a, int grid) {
    CUtensorMap tx, tw;
    cudaError_t err = make_grouped_tensor_maps(a, &tx, &tw);
    if (err != cudaSuccess) return err;
    auto kern = moe_grouped_kernel<G, GATED>;
    err = ensure_max_dynamic_smem(reinterpret_cast<const void*>(kern));
    if (err != cudaSuccess) return err;
    return launch(kern, dim3(2 * grid), kMgThreads, MgCfg::SMEM, a.stream, a.pdl, tx, tw, static_cast<const __half*>(a.scales), a.y,
                  a.N, a.K, a.activation, a.groups);
}

cudaError_t launch_grouped(const GroupedArgs& a, const DeviceInfo& dev) {
    if (a.gated) return a.G == 64 ? launch_grouped_t<64, true>(a, dev.num_sms) : launch_grouped_t<128, true>(a, dev.num_sms);
    return a.G == 64 ? launch_grouped_t<64, false>(a, dev.num_sms) : launch_grouped_t<128, false>(a, dev.num_sms);
}

}  // namespace w4a16
