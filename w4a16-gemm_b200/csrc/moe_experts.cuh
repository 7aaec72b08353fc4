// A mixture-of-experts layer from 4-bit experts:
//
//     h_tj = act(x_t Wg_e^T) * (x_t Wu_e^T),   e = experts[t][j]
//     y_t  = residual_t + sum_j weights[t][j] (h_tj Wd_e^T)
//
// Few entries an expert: three kernels, each launched behind the one before with programmatic dependent launch: the
// gated product, the second product, the weighted sum.  The products stream the weights of the experts that
// were chosen, each once a tile.  Which entries make which tile every CTA works out for itself, from up to 1024
// entries (about 1 us, where a kernel in front takes 4); above that a kernel does it once, in front.
//
// Many entries an expert (more than 14 on average, 10 with groups of 128): the products of moe_grouped.cuh, over rows of x that a kernel puts
// into sorted order first.
//
// The second product's CTAs start where the first one's leave, and fetch their first weights before the first
// one has ended: what that reads was written before the call, or by the kernel in front, and the gated product lets
// its successor start only after its own wait for whatever ran before it.
//
// One CTA an SM takes a range of the (tile, n16 block of output channels) sequence and walks it in batches
// of up to 10 blocks of one tile.  A batch runs over K in stages of 8 chunks of 64, filled by bulk copies onto
// one mbarrier: a block's 8 chunks are one run of 4 KB; the chunks' scales; 1 KB of each of the tile's rows.
// Issuing a bulk copy takes about 30 ns whatever its size, and a turn of one warp with all of a stage's copies longer than
// their bytes, so the three kinds have a warp each (32 tokens of 6 of 64 experts 108 -> 87 us).  Consumer
// warp w of 8 takes chunk w of a stage for all of the batch's blocks, so that K is summed over 8 warps, through
// shared memory, once a batch: sums are whole where they are made, and the gate needs no second pass.  Few warps with
// many independent chains each: what a warp does once a stage (waits, rows, the ones' product) counts
// for 10 blocks; two warps a chunk with half of the blocks each took 5 % longer, three 12 %.
//
// The codes enter mma.m16n8k16 where they lie in their words, masked: four bits at the bottom of a half are the fp16
// subnormal q 2^-24, the next four q 2^-20 (the first are rows 0-7 of a block, the others rows 8-15).  That
// takes 5 instructions a word where making the fp16 numbers q - 8 takes 9.  The 8 is taken off a chunk's sums
// with the sum of its x (a product with ones, shared by the blocks), the powers of two when a batch's sums are
// joined.  A chunk's sums are multiplied by its scale in fp32: the weight (q - 8) * s is never rounded.  The gated
// product's results are rounded to fp16 once, being operands of the second product, whose results stay fp32
// until the weighted sum.  That rounding is what a product with a gate returns on its own, its range with it (beyond 65504
// an inner result is infinite); it is the only one before y's, and takes the error against 64 bits from 2.1e-4, what
// y's rounding makes alone, to 2.9e-4.  Two fp16 numbers for every inner result keep fp32's bits (built, in both forms: 2.1e-4) for
// twice the second weight's products and twice the bytes of its rows, and the same range: one token of 2 of 8 experts 47.0 ->
// 50.7 us, 32 of 6 of 64 78.7 -> 86.7, 2048 of 6 of 64 560 -> 618 with groups of 64 and 440 -> 530 with groups of 128.  Not kept.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "epilogue.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace w4a16 {

constexpr int kMoeConsumers = kMoeChunks;                 // warps: one for each chunk of a stage
constexpr int kMoeProducers = 3;                          // warps: packed words, scales, rows
constexpr int kMoeThreads = (kMoeConsumers + kMoeProducers) * 32;
constexpr int kMoePlanThreads = 1024;

struct MoeCfg {
    static constexpr int BLOCKS = 10;                                 // n16 blocks of a batch, at most
    static constexpr int X_PITCH = kMoeChunks * 128 + 16;             // rows 16 bytes apart in banks: ldmatrix without conflicts
    static constexpr int W_BYTES = BLOCKS * kMoeChunks * 512;     // [block][chunk][32 lanes x 16 B]
    static constexpr int X_BYTES = kMoeRows * X_PITCH;
    static constexpr int S_ROW = BLOCKS * 32;                     // scales of one group of K: [block][16]
    static constexpr int S_BYTES = kMoeChunks * S_ROW;
    static constexpr int STAGE = W_BYTES + X_BYTES + S_BYTES;
    static constexpr int STAGES = 3;
    static constexpr int RED_BYTES = BLOCKS * kMoeChunks * 512;        // [block][chunk warp][lane] float4
    static constexpr int BARS = STAGES * STAGE + RED_BYTES;
    static constexpr int PLAN = BARS + 2 * STAGES * 8;                     // tiles of few entries, their order
    static constexpr int SMEM = 128 + PLAN + kMoeFewEntries * (8 + 2);
    static_assert(RED_BYTES >= kMoeMaxExperts * 8 + kMoeFewEntries * 6, "the sort's scratch");
    static_assert(BLOCKS == 10 && STAGE % 16 == 0 && SMEM <= 227 * 1024, "shared memory");
};

struct MoeParams {
    const __half* x;             // [tokens][hidden]
    const int32_t* words[2];     // of the two products: [experts][n * k / 8]
    const __half* scales[2];     // [experts][k / G][n]
    const int32_t* experts;      // [tokens][k]
    const float* weights;        // [tokens][k]
    const __half* residual;      // [tokens][hidden] or NULL
    __half* y;
    char* workspace;
    MoePlan plan;
    int32_t entries, k, num_experts, hidden, inner, activation;
};

__device__ __forceinline__ MoeHead* moe_head(const MoeParams& p) { return reinterpret_cast<MoeHead*>(p.workspace); }
__device__ __forceinline__ int4* moe_tiles(const MoeParams& p) { return reinterpret_cast<int4*>(p.workspace + p.plan.tiles_at); }
__device__ __forceinline__ int32_t* moe_order(const MoeParams& p) { return reinterpret_cast<int32_t*>(p.workspace + p.plan.order_at); }
__device__ __forceinline__ int32_t* moe_place(const MoeParams& p) { return reinterpret_cast<int32_t*>(p.workspace + p.plan.place_at); }
__device__ __forceinline__ __half* moe_inner(const MoeParams& p) { return reinterpret_cast<__half*>(p.workspace + p.plan.inner_at); }
__device__ __forceinline__ float* moe_out(const MoeParams& p) { return reinterpret_cast<float*>(p.workspace + p.plan.out_at); }

// Inclusive sum over the CTA's threads, in their order.
__device__ __forceinline__ int scan_threads(int v, int* shared) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) shared[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int w = shared[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        shared[lane] = w;
    }
    __syncthreads();
    if (warp > 0) v += shared[warp - 1];
    __syncthreads();
    return v;
}

// One CTA: counts the experts' entries, lays their tiles out, sorts the entries.  The order of one expert's entries is
// the order in which they arrive; no result depends on it, since every entry's row is summed by itself.
static __global__ void __launch_bounds__(kMoePlanThreads) moe_plan_kernel(const __grid_constant__ MoeParams p) {
    __shared__ int count[kMoeMaxExperts], cursor[kMoeMaxExperts], warps[32];
    const int t = threadIdx.x;
    count[t] = 0;
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    const auto expert_of = [&](int i) {
        const int e = i < p.entries ? __ldg(p.experts + i) : -1;
        return e >= 0 && e < p.num_experts ? e : -1;
    };
    constexpr int AHEAD = 8;                              // loads in flight
    for (int i0 = t; i0 < p.entries; i0 += AHEAD * kMoePlanThreads) {
        int e[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) e[j] = expert_of(i0 + j * kMoePlanThreads);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (e[j] >= 0) atomicAdd(&count[e[j]], 1);
    }
    __syncthreads();
    const int mine = count[t], rows = p.plan.rows, tiles = (mine + rows - 1) / rows;
    const int end = scan_threads(mine, warps), tile_end = scan_threads(tiles, warps);
    cursor[t] = end - mine;
    int4* const out = moe_tiles(p) + (tile_end - tiles);
    for (int i = 0; i < tiles; ++i) out[i] = make_int4(t, end - mine + i * rows, min(rows, mine - i * rows), 0);
    if (t == kMoePlanThreads - 1) {
        moe_head(p)->tiles = tile_end;
        moe_head(p)->entries = end;
    }
    __syncthreads();
    int32_t* const order = moe_order(p);
    for (int i0 = t; i0 < p.entries; i0 += AHEAD * kMoePlanThreads) {
        int e[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) e[j] = expert_of(i0 + j * kMoePlanThreads);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (e[j] >= 0) {
                const int i = i0 + j * kMoePlanThreads, at = atomicAdd(&cursor[e[j]], 1);
                order[at] = i;
                if (p.plan.grouped) moe_place(p)[i] = at;
            }
    }
}

// Rows of x in sorted order: a warp a row.
constexpr int kMoeGatherThreads = 256;
static __global__ void __launch_bounds__(kMoeGatherThreads) moe_gather_kernel(const __grid_constant__ MoeParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t row = (int64_t)blockIdx.x * (kMoeGatherThreads / 32) + threadIdx.x / 32;
    if (row >= __ldcg(&moe_head(p)->entries)) return;
    const int64_t token = __ldcg(moe_order(p) + row) / p.k;
    const uint4* const from = reinterpret_cast<const uint4*>(p.x + token * p.hidden);
    uint4* const to = reinterpret_cast<uint4*>(p.workspace + p.plan.rows_at) + row * (p.hidden / 8);
    const int units = p.hidden / 8;
    for (int i = threadIdx.x & 31; i < units; i += 8 * 32) {      // eight loads in flight
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * 32 < units) v[j] = from[i + j * 32];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * 32 < units) to[i + j * 32] = v[j];
    }
}

// One tile, packed: its expert and count, its first sorted entry.
struct MoeSmallTile {
    uint16_t expert, count;
    uint32_t start;
};

// The same for up to kMoeFewEntries entries, by every CTA in its shared memory, in one order: expert by expert, the
// entries of one as they are numbered (the CTAs of a call have to agree).  scratch: two words an expert, six bytes an entry.  Returns the number of tiles.
template <int THREADS>
__device__ __forceinline__ int moe_sort_few(const MoeParams& p, MoeSmallTile* tiles, uint16_t* order, char* scratch) {
    constexpr int PER = (kMoeMaxExperts + THREADS - 1) / THREADS;
    constexpr int WARPS = THREADS / 32;
    __shared__ uint32_t sums[32];
    int32_t* const count = reinterpret_cast<int32_t*>(scratch);
    int32_t* const first = count + kMoeMaxExperts;
    int32_t* const expert = first + kMoeMaxExperts;
    uint16_t* const rank = reinterpret_cast<uint16_t*>(expert + kMoeFewEntries);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (p.entries <= 32) {               // one warp, in registers: experts by their first entry
        if (warp == 0) {
            const int raw = lane < p.entries ? __ldg(p.experts + lane) : -1;
            const int e = raw >= 0 && raw < p.num_experts ? raw : -1;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const int n = __popc(same), leader = __ffs(same) - 1;
            const bool leads = e >= 0 && leader == lane;
            const uint32_t mine = leads ? (uint32_t)n | (uint32_t)((n + p.plan.rows - 1) / p.plan.rows) << 16 : 0u;
            uint32_t end = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, end, o);
                if (lane >= o) end += u;
            }
            const uint32_t before = end - mine;
            const int start = __shfl_sync(0xffffffffu, before, leader) & 0xffff;
            if (e >= 0) order[start + __popc(same & ((1u << lane) - 1))] = (uint16_t)lane;
            if (leads)
                for (int i = 0; i * p.plan.rows < n; ++i)
                    tiles[(before >> 16) + i] = {(uint16_t)e, (uint16_t)min(p.plan.rows, n - i * p.plan.rows), (uint32_t)(start + i * p.plan.rows)};
            if (lane == 31) sums[0] = end;
        }
        __syncthreads();
        return (int)(sums[0] >> 16);
    }
    for (int i = t; i < kMoeMaxExperts; i += THREADS) count[i] = 0;
    for (int i = t; i < p.entries; i += THREADS) {
        const int e = __ldg(p.experts + i);
        expert[i] = e >= 0 && e < p.num_experts ? e : -1;
    }
    __syncthreads();
    if (warp == 0) {                     // ranks among the entries of one expert, 32 entries at a time
        for (int i0 = 0; i0 < p.entries; i0 += 32) {
            const int i = i0 + lane, e = i < p.entries ? expert[i] : -1;
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            const int before = __popc(same & ((1u << lane) - 1));
            if (e >= 0) {
                const int r = count[e] + before;
                rank[i] = (uint16_t)r;
            }
            __syncwarp();
            if (e >= 0 && before == 0) count[e] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    // entries and tiles before each expert, 16 bits each, PER experts a thread
    uint32_t mine[PER], v = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = PER * t + j, n = e < kMoeMaxExperts ? count[e] : 0;
        mine[j] = (uint32_t)n | (uint32_t)((n + p.plan.rows - 1) / p.plan.rows) << 16;
        v += mine[j];
    }
    uint32_t end = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += u;
    }
    if (lane == 31) sums[warp] = end;
    __syncthreads();
    uint32_t before = end - v, all = 0;
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? sums[w] : 0u;
        all += sums[w];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int n = mine[j] & 0xffff, start = before & 0xffff, tile = before >> 16, e = PER * t + j;
        if (e < kMoeMaxExperts) first[e] = start;
        for (int i = 0; i * p.plan.rows < n; ++i)
            tiles[tile + i] = {(uint16_t)e, (uint16_t)min(p.plan.rows, n - i * p.plan.rows), (uint32_t)(start + i * p.plan.rows)};
        before += mine[j];
    }
    __syncthreads();
    for (int i = t; i < p.entries; i += THREADS)
        if (expert[i] >= 0) order[first[expert[i]] + rank[i]] = (uint16_t)i;
    __syncthreads();
    return (int)(all >> 16);
}

// Untiled bulk copy into this CTA's shared memory (16-byte aligned addresses and size).
__device__ __forceinline__ void moe_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// The codes of one packed word as an A fragment of subnormals: rows g at 2^-24, rows g + 8 at 2^-20.
__device__ __forceinline__ void code_word(uint32_t q, uint32_t (&a)[4]) {
    const uint32_t q8 = q >> 8;
    a[0] = q & 0x000F000Fu;
    a[1] = q & 0x00F000F0u;
    a[2] = q8 & 0x000F000Fu;
    a[3] = q8 & 0x00F000F0u;
}

// c += a * b, or c = a * b.  Not volatile: chains of different blocks may be put between one another.
__device__ __forceinline__ void moe_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool fresh) {
    if (fresh)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a warp takes out of a stage: its chunk's rows, the N blocks' words and scales.
template <int N>
struct MoeFragments {
    uint32_t b[8];
    uint4 w[N];
    uint16_t scale[N][2];
    // x_at, w_at, s_at: this lane's shared-memory addresses
    __device__ __forceinline__ void load(uint32_t x_at, uint32_t w_at, uint32_t s_at) {
        ldmatrix_x4(*reinterpret_cast<uint32_t(*)[4]>(&b[0]), x_at);
        ldmatrix_x4(*reinterpret_cast<uint32_t(*)[4]>(&b[4]), x_at + 64);
#pragma unroll
        for (int blk = 0; blk < N; ++blk) {
            w[blk] = lds128(w_at + blk * (kMoeChunks * 512));
            scale[blk][0] = lds_u16(s_at + blk * 32);
            scale[blk][1] = lds_u16(s_at + blk * 32 + 16);
        }
    }
    // Products of the chunk, added to the blocks' sums.
    __device__ __forceinline__ void multiply(float (&acc)[N][4]) const {
        float c[N][4], sum[4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const uint32_t ones[4] = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
            moe_mma(sum, ones, b[2 * ks], b[2 * ks + 1], ks == 0);
#pragma unroll
            for (int blk = 0; blk < N; ++blk) {
                uint32_t a[4];
                code_word(ks == 0 ? w[blk].x : ks == 1 ? w[blk].y : ks == 2 ? w[blk].z : w[blk].w, a);
                moe_mma(c[blk], a, b[2 * ks], b[2 * ks + 1], ks == 0);
            }
        }
        // less 8 for every code, in the units of the rows
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float eight = sum[i] * (i < 2 ? -0x1p-21f : -0x1p-17f);
#pragma unroll
            for (int blk = 0; blk < N; ++blk)
                acc[blk][i] = fmaf(__half2float(__ushort_as_half(scale[blk][i >> 1])), c[blk][i] + eight, acc[blk][i]);
        }
    }
};

// A place in the ring of stages.
template <int STAGES>
struct MoeRing {
    int stage;
    uint32_t phase;
    __device__ __forceinline__ void next() {
        if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
        }
    }
};

// One consumer warp's share of a batch of N blocks: its chunk of `stages` stages, the last of which holds `last` chunks.
// A stage is given back as soon as it is in registers.  Leaves the sums in `red` (this lane's address of the first
// block's).  False once a wait has run out; the ring is walked to the batch's end all the same.
template <int N>
__device__ __forceinline__ bool moe_batch(uint32_t base, MoeRing<MoeCfg::STAGES>& ring, int stages, int last, int chunk,
                                          uint32_t x_lane, uint32_t w_lane, uint32_t s_lane, uint32_t red, bool ok) {
    using C = MoeCfg;
    float acc[N][4];
#pragma unroll
    for (int blk = 0; blk < N; ++blk)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[blk][i] = 0.f;
#pragma unroll 1
    for (int st = 0; st < stages; ++st) {
        const uint32_t sb = base + (uint32_t)(ring.stage * C::STAGE);
        const bool there = st + 1 < stages || chunk < last;
        ok = ok && __all_sync(0xffffffffu, mbar_wait_sleep(base + (uint32_t)(C::BARS + ring.stage * 8), ring.phase, kDevTimeoutExperts));
        const uint32_t empty = base + (uint32_t)(C::BARS + (C::STAGES + ring.stage) * 8);
        ring.next();
        // one straight run, with the fragments alive in it alone: they and the sums take 130 registers
        if (ok && there) {
            MoeFragments<N> f;
            f.load(sb + x_lane, sb + w_lane, sb + s_lane);
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(empty);
            f.multiply(acc);
        } else {
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(empty);
        }
    }
    bar_sync_named(1, kMoeConsumers * 32);           // the last batch's sums have been read
#pragma unroll
    for (int blk = 0; blk < N; ++blk)
        sts128(red + blk * kMoeChunks * 512, make_float4(acc[blk][0], acc[blk][1], acc[blk][2], acc[blk][3]));
    return ok;
}

// A CTA's walk: batches of up to BLOCKS blocks of one (tile, K range), over its range of units.  Unit u is block u % blocks
// of K range u / blocks % splits of tile u / blocks / splits.  Batches of one range are of one size to within a block: a
// short last one would take as many turns as a full one (25 blocks by 8, as 8 + 8 + 8 + 1 instead of 7 + 6 + 6 + 6, made
// the slowest CTA 36 us late where the others took 29).
template <int BLOCKS>
struct MoeWalk {
    int unit, end, blocks, splits;
    int tile, split, block, n;         // of the current batch
    __device__ __forceinline__ bool next() {
        unit += n;
        if (unit >= end) return false;
        const int line = unit / blocks;
        block = unit - line * blocks;
        tile = line / splits;
        split = line - tile * splits;
        const int left = min(blocks - block, end - unit), batches = (left + BLOCKS - 1) / BLOCKS;
        n = (left + batches - 1) / batches;
        return true;
    }
};

// GATED: the first product (rows of x, gated, into the workspace in sorted order); else the second (rows of the
// first's results, into the workspace by entry and K range).
template <int G, bool GATED>
static __global__ void __launch_bounds__(kMoeThreads, 1) moe_product_kernel(const __grid_constant__ MoeParams p) {
    using C = MoeCfg;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto stage = [&](int s) { return base + (uint32_t)(s * C::STAGE); };
    auto full = [&](int s) { return base + (uint32_t)(C::BARS + s * 8); };
    auto empty = [&](int s) { return base + (uint32_t)(C::BARS + (C::STAGES + s) * 8); };
    const uint32_t red = base + C::STAGES * C::STAGE;

    if (GATED) {
        pdl_wait();
        pdl_launch_dependents();
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(full(s), kMoeProducers);
            mbar_init(empty(s), kMoeConsumers);
        }
        fence_mbar_init();
    }
    char* const smem = reinterpret_cast<char*>(smem_raw) + (base - smem_u32(smem_raw));
    MoeSmallTile* const small = reinterpret_cast<MoeSmallTile*>(smem + C::PLAN);
    uint16_t* const small_order = reinterpret_cast<uint16_t*>(small + kMoeFewEntries);
    int tiles;
    if (p.plan.few) {
        tiles = moe_sort_few<kMoeThreads>(p, small, small_order, smem + C::STAGES * C::STAGE);
    } else {
        __syncthreads();
        tiles = __ldcg(&moe_head(p)->tiles);
    }
    const auto tile_at = [&](int i) {
        if (!p.plan.few) return __ldcg(moe_tiles(p) + i);
        const MoeSmallTile t = small[i];
        return make_int4(t.expert, (int)t.start, t.count, 0);
    };
    const auto entry_at = [&](int i) { return p.plan.few ? (int)small_order[i] : __ldcg(moe_order(p) + i); };

    const int K = GATED ? p.hidden : p.inner, N = GATED ? 2 * p.inner : p.hidden;
    const int chunks = K >> 6, all_stages = (chunks + kMoeChunks - 1) / kMoeChunks;
    MoeWalk<C::BLOCKS> walk;
    walk.blocks = N >> 4;
    walk.splits = GATED ? 1 : p.plan.splits;
    const long long units = (long long)tiles * walk.splits * walk.blocks;
    walk.unit = (int)(units * blockIdx.x / gridDim.x);
    walk.end = (int)(units * (blockIdx.x + 1) / gridDim.x);
    walk.n = 0;
    int it = 0;

    if (warp >= kMoeConsumers) {
        // ------------------------------------------------ producers: one copy a lane
        const int role = warp - kMoeConsumers;           // 0 the blocks' packed words, 1 the groups' scales, 2 the tile's rows
        bool ok = true;
        if (!GATED && role == 2) pdl_wait();             // the rows are the first product's results
        while (ok && walk.next()) {
            const int4 tile = tile_at(walk.tile);
            const char* src;                             // of this lane at chunk 0
            uint32_t dst;
            int64_t step;                                // bytes from chunk to chunk (scales: from group to group)
            int have;                                    // lanes with a copy (scales: by the stage)
            if (role == 0) {
                src = reinterpret_cast<const char*>(p.words[GATED ? 0 : 1]) +
                      ((int64_t)tile.x * walk.blocks + walk.block + lane) * chunks * 512;
                dst = lane * (kMoeChunks * 512);
                step = 512;
                have = walk.n;
            } else if (role == 1) {
                src = reinterpret_cast<const char*>(p.scales[GATED ? 0 : 1] + ((int64_t)tile.x * (K / G) + lane) * N + walk.block * 16);
                dst = C::W_BYTES + C::X_BYTES + lane * C::S_ROW;
                step = (int64_t)N * 2;
                have = 0;
            } else {
                have = tile.z;
                const int at = tile.y + min(lane, have - 1);
                src = reinterpret_cast<const char*>(GATED ? p.x + (int64_t)(entry_at(at) / p.k) * K
                                                          : moe_inner(p) + (int64_t)at * K);
                dst = C::W_BYTES + lane * C::X_PITCH;
                step = 128;
            }
            const int s1 = all_stages * (walk.split + 1) / walk.splits;
            for (int st = all_stages * walk.split / walk.splits; st < s1; ++st, ++it) {
                const int s = it % C::STAGES, c0 = st * kMoeChunks, n = min(kMoeChunks, chunks - c0);
                if (it >= C::STAGES) {
                    ok = __all_sync(0xffffffffu, mbar_wait_sleep(empty(s), (it / C::STAGES - 1) & 1, kDevTimeoutExperts));
                    if (!ok) break;
                }
                const int copies = role == 1 ? (n * 64 + G - 1) / G : have;
                const uint32_t bytes = role == 0 ? n * 512 : role == 1 ? walk.n * 32 : n * 128;
                if (lane == 0) mbar_arrive_expect_tx(full(s), copies * bytes);
                __syncwarp();
                if (lane < copies) moe_copy(stage(s) + dst, src + (role == 1 ? c0 * 64 / G : c0) * step, bytes, full(s));
            }
        }
        // copies still in flight must land before the CTA may exit (they have, unless a wait ran out)
        for (int j = it - 1; j >= 0 && j >= it - C::STAGES; --j) mbar_wait(full(j % C::STAGES), (j / C::STAGES) & 1, kDevTimeoutExperts);
        return;
    }

    // ---------------------------------------------------- consumers
    // After a wait that ran out a warp computes nothing more but keeps every barrier, so that none waits for it.
    const int chunk = warp, g8 = lane >> 2, t4 = lane & 3;
    const uint32_t x_lane = C::W_BYTES + (lane & 7) * C::X_PITCH + chunk * 128 + (lane >> 3) * 16;
    const uint32_t w_lane = chunk * 512 + lane * 16;
    const uint32_t s_lane = C::W_BYTES + C::X_BYTES + (chunk * 64 / G) * C::S_ROW + g8 * 2;
    const uint32_t red_lane = red + chunk * 512 + lane * 16;
    if (!GATED) {
        pdl_wait();                                      // the call before may still read what this one writes
        pdl_launch_dependents();
    }
    bool ok = true;
    MoeRing<C::STAGES> ring = {0, 0};
    while (walk.next()) {
        const int s0 = all_stages * walk.split / walk.splits, stages = all_stages * (walk.split + 1) / walk.splits - s0;
        const int last = min(kMoeChunks, chunks - (s0 + stages - 1) * kMoeChunks);
        switch (walk.n) {
#define W4A16_MOE_BATCH(N) \
            case N: \
                ok = moe_batch<N>(base, ring, stages, last, chunk, x_lane, w_lane, s_lane, red_lane, ok); \
                break;
            W4A16_MOE_BATCH(1) W4A16_MOE_BATCH(2) W4A16_MOE_BATCH(3) W4A16_MOE_BATCH(4) W4A16_MOE_BATCH(5)
            W4A16_MOE_BATCH(6) W4A16_MOE_BATCH(7) W4A16_MOE_BATCH(8) W4A16_MOE_BATCH(9) W4A16_MOE_BATCH(10)
#undef W4A16_MOE_BATCH
        }
        bar_sync_named(2, kMoeConsumers * 32);
        const int4 tile = tile_at(walk.tile);
        for (int blk = warp; blk < walk.n; blk += kMoeConsumers) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kMoeChunks; ++c) {
                const float4 f = lds128f(red + ((blk * kMoeChunks + c) * 32 + lane) * 16);
                v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
            }
            v[0] *= 0x1p24f; v[1] *= 0x1p24f; v[2] *= 0x1p20f; v[3] *= 0x1p20f;
            // elements 0, 1: row g8 of the block for rows 2 t4, 2 t4 + 1 of the tile; 2, 3: row g8 + 8
            const int nb = walk.block + blk;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = 2 * t4 + j;
                if (row >= tile.z) continue;
                if (GATED) {
                    moe_inner(p)[(int64_t)(tile.y + row) * p.inner + nb * 8 + g8] =
                        __float2half_rn(activate(v[j], p.activation) * v[2 + j]);
                } else {
                    const int64_t entry = entry_at(tile.y + row);
                    float* const o = moe_out(p) + ((int64_t)walk.split * p.entries + entry) * p.hidden + nb * 16 + g8;
                    __stcg(o, v[j]);
                    __stcg(o + 8, v[2 + j]);
                }
            }
        }
    }
}

constexpr int kMoeFinishThreads = 128;

// y = residual + the entries' results, weighted, in the order of the choices and their K ranges: four columns a thread, and
// SLICES threads (of different warps) to share those columns' parts, whose sums are added in order.  Bound by the
// latency of its loads: each thread has 8 in flight.
template <int SLICES>
static __global__ void __launch_bounds__(kMoeFinishThreads) moe_finish_kernel(const __grid_constant__ MoeParams p) {
    constexpr int QUADS = kMoeFinishThreads / SLICES;
    __shared__ float4 shared[SLICES > 1 ? kMoeFinishThreads : 1];
    const int64_t token = blockIdx.x;
    const int slice = threadIdx.x / QUADS, col = (blockIdx.y * QUADS + threadIdx.x % QUADS) * 4;
    const bool in_row = col < p.hidden;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.residual && in_row && slice == 0) {          // an input of the call: there before the products began
        const uint2 r = *reinterpret_cast<const uint2*>(p.residual + token * p.hidden + col);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
    const int parts = p.k * p.plan.splits, per = (parts + SLICES - 1) / SLICES;
    const int end = min(parts, (slice + 1) * per);
    pdl_wait();
    pdl_launch_dependents();
    // what an expert outside the layer would have left is loaded too, and dropped
    for (int i0 = slice * per; i0 < end && in_row; i0 += 8) {
        float4 d[8];
        float w[8];
        bool in[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int part = min(i0 + i, end - 1), j = part / p.plan.splits, range = part - j * p.plan.splits;
            const int64_t entry = token * p.k + j;
            d[i] = __ldcg(reinterpret_cast<const float4*>(moe_out(p) + (range * (int64_t)p.entries + entry) * p.hidden + col));
            const int e = __ldg(p.experts + entry);
            w[i] = __ldg(p.weights + entry);
            in[i] = i0 + i < end && e >= 0 && e < p.num_experts;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in[i]) {
                v[0] = fmaf(w[i], d[i].x, v[0]);
                v[1] = fmaf(w[i], d[i].y, v[1]);
                v[2] = fmaf(w[i], d[i].z, v[2]);
                v[3] = fmaf(w[i], d[i].w, v[3]);
            }
    }
    if constexpr (SLICES > 1) {
        shared[threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (slice > 0) return;
#pragma unroll
        for (int i = 1; i < SLICES; ++i) {
            const float4 f = shared[i * QUADS + threadIdx.x];
            v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        }
    }
    if (!in_row) return;
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p.y + token * p.hidden + col) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// The same over the grouped products' results (in sorted order): a CTA a token, four columns a thread and turn.  Its
// choices' rows and weights are looked up once; bound by the memory's bandwidth.
static __global__ void __launch_bounds__(kMoeFinishThreads) moe_grouped_finish_kernel(const __grid_constant__ MoeParams p) {
    __shared__ int32_t row[32];
    __shared__ float weight[32];
    const int64_t token = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    if ((int)threadIdx.x < p.k) {
        const int64_t entry = token * p.k + threadIdx.x;
        const int e = __ldg(p.experts + entry);
        const bool in = e >= 0 && e < p.num_experts;
        row[threadIdx.x] = in ? __ldcg(moe_place(p) + entry) : -1;
        weight[threadIdx.x] = in ? __ldg(p.weights + entry) : 0.f;
    }
    __syncthreads();
    const float4* const out = reinterpret_cast<const float4*>(moe_out(p));
    const int quads = p.hidden / 4;
    for (int c = threadIdx.x; c < quads; c += kMoeFinishThreads) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (p.residual) {
            const uint2 r = reinterpret_cast<const uint2*>(p.residual + token * p.hidden)[c];
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        }
        for (int j0 = 0; j0 < p.k; j0 += 8) {
            float4 d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < p.k && row[j0 + j] >= 0) d[j] = __ldcg(out + (int64_t)row[j0 + j] * quads + c);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < p.k && row[j0 + j] >= 0) {
                    const float w = weight[j0 + j];
                    v[0] = fmaf(w, d[j].x, v[0]);
                    v[1] = fmaf(w, d[j].y, v[1]);
                    v[2] = fmaf(w, d[j].z, v[2]);
                    v[3] = fmaf(w, d[j].w, v[3]);
                }
        }
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        reinterpret_cast<uint2*>(p.y + token * p.hidden)[c] =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

}  // namespace w4a16
