// Device code of the 4-bit key/value cache: append, read back, attention.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "ptx.cuh"
#include "cache_format.cuh"
#include "cache_attention.cuh"
#include "cache_decode.cuh"
#include "cache_prompt.cuh"

namespace w4a16 {

cudaError_t read_cache_device_status(int* code, bool reset) {
    cudaError_t err = cudaMemcpyFromSymbol(code, w4a16_device_status, sizeof(int));
    if (err != cudaSuccess || !reset) return err;
    const int zero = 0;
    return cudaMemcpyToSymbol(w4a16_device_status, &zero, sizeof(int));
}

cudaError_t run_cache_wait_limit_check() {
    wait_limit_kernel<<<1, 32>>>(1, kDevTimeoutCache);
    const cudaError_t err = cudaGetLastError();
    return err != cudaSuccess ? err : cudaDeviceSynchronize();
}

static CacheView cache_view(const w4a16_cache& c) {
    CacheView v;
    v.data = static_cast<uint8_t*>(c.data);
    v.num_pages = c.num_pages;
    v.page_shift = 0;
    while ((1 << v.page_shift) < c.page_size) ++v.page_shift;
    v.kv_heads = c.kv_heads;
    v.block_bytes = cache_block_bytes(c.page_size, c.head_dim, c.group_size);
    return v;
}

// Calls f with the cache's (D, G) as integral constants.
template <typename Fn>
static cudaError_t with_format(const w4a16_cache& c, Fn&& f) {
    using std::integral_constant;
    if (c.head_dim == 64) return f(integral_constant<int, 64>{}, integral_constant<int, 64>{});
    if (c.group_size == 64) return f(integral_constant<int, 128>{}, integral_constant<int, 64>{});
    return f(integral_constant<int, 128>{}, integral_constant<int, 128>{});
}

template <typename Fn>
static cudaError_t with_bool(bool b, Fn&& f) {
    return b ? f(std::integral_constant<bool, true>{}) : f(std::integral_constant<bool, false>{});
}

template <typename... KArgs, typename... Args>
static cudaError_t launch(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, bool pdl,
                          Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

cudaError_t launch_cache_append(const CacheAppendArgs& a) {
    AppendParams p = {};
    p.c = cache_view(a.c);
    p.k = static_cast<const uint16_t*>(a.k);
    p.v = static_cast<const uint16_t*>(a.v);
    p.k_token = a.k_token_stride; p.k_head = a.k_head_stride;
    p.v_token = a.v_token_stride; p.v_head = a.v_head_stride;
    p.slots = a.slots;
    p.tokens = a.tokens;
    int vecs = 2 * a.c.kv_heads;
    if (a.rotate) {
        p.q = static_cast<const uint16_t*>(a.r.q);
        p.q_out = static_cast<uint16_t*>(a.r.q_out);
        p.q_token = a.r.q_token_stride; p.q_head = a.r.q_head_stride;
        p.positions = a.r.positions;
        p.axis_stride = a.r.positions_axis_stride;
        p.cos_sin = a.r.cos_sin;
        p.max_pos = a.r.max_pos;
        p.q_heads = a.r.q ? a.r.q_heads : 0;
        p.axes = a.r.axes;
        p.end0 = a.r.sections[0];
        p.end1 = a.r.sections[0] + a.r.sections[1];
        p.rotary_dim = a.r.rotary_dim;
        p.interleaved = a.r.interleaved;
        vecs += p.q_heads;
    }
    // lane groups a token: as many as it has vectors, up to those of one CTA
    const int lanes = a.c.head_dim / 8;
    while ((2 << p.log_par) <= vecs && (2 << p.log_par) <= kAppendThreads / lanes) ++p.log_par;
    // With threads enough for every SM (148 of 1024) a token's lanes take several vectors with the same
    // cosines and sines: 8192 tokens of 64 and 8 heads 86 us with 16 groups a token, 64 with 4 or
    // 2, 75 with 1; 1157 tokens of 28 and 4 heads on three axes 11 us with 16, 8 with 8.
    while (p.log_par > 2 && (a.tokens << p.log_par) * lanes > 160000) --p.log_par;
    const int64_t threads = (a.tokens << p.log_par) * lanes;
    const dim3 grid((unsigned)((threads + kAppendThreads - 1) / kAppendThreads));
    return with_format(a.c, [&](auto d, auto g) {
        return with_bool(a.bf16, [&](auto bf) {
            return with_bool(a.rotate, [&](auto rot) {
                return launch(cache_append_kernel<d.value, g.value, bf.value, rot.value>, grid, kAppendThreads, 0,
                              a.stream, a.pdl, p);
            });
        });
    });
}

cudaError_t launch_cache_read(const w4a16_cache& c, const int64_t* slots, int64_t tokens, void* k, void* v, bool bf16,
                              cudaStream_t stream, bool pdl) {
    const int64_t per = kReadVecs * (kReadThreads / (c.head_dim / 8));
    const dim3 grid((unsigned)((tokens * c.kv_heads + per - 1) / per));
    return with_format(c, [&](auto d, auto g) {
        return with_bool(bf16, [&](auto bf) {
            return launch(cache_read_kernel<d.value, g.value, bf.value>, grid, kReadThreads, 0, stream, pdl,
                          cache_view(c), slots, tokens, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v));
        });
    });
}

static AttentionParams attention_params(const w4a16_cache& c, const w4a16_cache_attention_args& a) {
    AttentionParams p = {};
    p.c = cache_view(c);
    p.q = static_cast<const uint16_t*>(a.q);
    p.out = static_cast<uint16_t*>(a.out);
    p.lse = a.lse;
    p.q_token = a.q_token_stride; p.q_head = a.q_head_stride;
    p.q_tokens = a.q_tokens;
    p.table = a.page_table;
    p.table_stride = a.page_table_stride;
    p.table_pages = a.table_pages;
    p.seq_lens = a.seq_lens;
    p.cu_q = a.cu_q;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.batch = a.batch;
    p.max_q = a.max_q;
    p.shared = a.q_heads / c.kv_heads;
    p.causal = a.causal != 0;
    p.window = a.window > 0 ? a.window : 0;
    p.bf16 = a.dtype == W4A16_ACT_BF16;
    return p;
}

// How an attention call is run: by rows (query heads of a key head times queries).
struct AttentionPlan {
    int row_blocks;      // blocks of 8 rows of the decode kernel; 0: the prompt kernel
    int grid;
    CpGrid prompt;
    size_t workspace;
};

template <int D, int G>
static AttentionPlan plan_decode_t(const w4a16_cache& c, const w4a16_cache_attention_args& a, const DeviceInfo& dev) {
    using C = CdCfg<D, G>;
    const int64_t rows = (int64_t)a.max_q * (a.q_heads / c.kv_heads);
    const int64_t blocks = (rows + C::ROWS - 1) / C::ROWS, segments = (int64_t)a.batch * c.kv_heads * blocks;
    const int64_t tiles = ((int64_t)a.table_pages * c.page_size + kCdTile - 1) / kCdTile;
    AttentionPlan p = {};
    p.row_blocks = (int)blocks;
    p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(segments * tiles, (int64_t)C::CTAS * dev.num_sms));
    p.workspace = cd_info_bytes(segments) + 2 * (size_t)p.grid * cd_slot_floats(C::ROWS, D) * sizeof(float);
    return p;
}

// Row blocks of 256 (128, with the halves on alternate tiles, if no sequence has more rows).  A
// block's tiles are split over as many CTAs as an estimate says is shortest: a tile 2.4 us, a CTA's
// start and end 7 us (measured); the work spread over the SMs, and for the last wave, as far as it is not
// full, a CTA of the block with fewest tiles (heavy blocks come first); and the parts written and
// joined.  Lengths are not known here:
// the page table's width stands for them.  Measured, 32/8 heads, unsplit / as chosen: 800 queries over
// 16384 tokens (104 blocks) 305 / 269 us, 1200 (152) 543 / 429; a prompt of 1500 (192, unsplit) 43.
// Results of split blocks pass through the workspace, which is kept below 256 MB.
static AttentionPlan plan_prompt(const w4a16_cache& c, const w4a16_cache_attention_args& a, const DeviceInfo& dev) {
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
        const double waves = (double)(busy * s) / dev.num_sms, idle = std::ceil(waves) - waves;
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

static AttentionPlan plan_attention(const w4a16_cache& c, const w4a16_cache_attention_args& a, const DeviceInfo& dev) {
    const int64_t rows = (int64_t)a.max_q * (a.q_heads / c.kv_heads);
    if (rows > kDecodeRows) return plan_prompt(c, a, dev);
    AttentionPlan p = {};
    with_format(c, [&](auto d, auto g) {
        p = plan_decode_t<d.value, g.value>(c, a, dev);
        return cudaSuccess;
    });
    return p;
}

size_t cache_attention_workspace(const w4a16_cache& c, const w4a16_cache_attention_args& a, const DeviceInfo& dev) {
    return plan_attention(c, a, dev).workspace;
}

template <int D, int G>
static cudaError_t launch_decode_t(const AttentionParams& ap, const AttentionPlan& plan, cudaStream_t stream, bool pdl) {
    using C = CdCfg<D, G>;
    auto kern = cache_decode_kernel<D, G>;
    cudaError_t err = ensure_max_dynamic_smem(reinterpret_cast<const void*>(kern));
    if (err != cudaSuccess) return err;
    err = launch(kern, dim3(plan.grid), kCdThreads, C::SMEM, stream, pdl, ap);
    if (err != cudaSuccess) return err;
    // slices of a row's parts: by how many CTAs a segment may be spread over
    const int64_t segments = (int64_t)ap.batch * ap.c.kv_heads * ap.row_blocks;
    const int64_t spread = plan.grid / segments;
    const int seg_rows = std::min(C::ROWS, ap.max_q * ap.shared);
    const int64_t rows = segments * seg_rows, per = 128 / (D / 4);
    if (spread < 8)
        return launch(cache_decode_combine_kernel<D, 1>, dim3((unsigned)((rows + per - 1) / per)), 128, 0, stream, pdl, ap, seg_rows, rows);
    if (spread < 64)
        return launch(cache_decode_combine_kernel<D, 4>, dim3((unsigned)rows), D, 0, stream, pdl, ap, seg_rows, rows);
    return launch(cache_decode_combine_kernel<D, 16>, dim3((unsigned)rows), 4 * D, 0, stream, pdl, ap, seg_rows, rows);
}

template <int D, int G>
static cudaError_t launch_prompt_t(const AttentionParams& ap, const AttentionPlan& plan, cudaStream_t stream, bool pdl) {
    using C = CpCfg<D, G>;
    auto kern = cache_prompt_kernel<D, G>;
    cudaError_t err = ensure_max_dynamic_smem(reinterpret_cast<const void*>(kern));
    if (err != cudaSuccess) return err;
    err = launch(kern, dim3((unsigned)plan.grid), kCpThreads, C::SMEM, stream, pdl, ap, plan.prompt);
    if (err != cudaSuccess || plan.prompt.splits == 1) return err;
    const int64_t rows = (int64_t)ap.max_q * ap.shared * ap.c.kv_heads, per = 128 / (D / 4);
    return launch(cache_prompt_combine_kernel<D>, dim3((unsigned)((rows + per - 1) / per), (unsigned)ap.batch), 128, 0, stream,
                  pdl, ap, plan.prompt.splits);
}

cudaError_t launch_cache_attention(const w4a16_cache& c, const w4a16_cache_attention_args& a, const DeviceInfo& dev,
                                   void* workspace, cudaStream_t stream, bool pdl) {
    AttentionParams p = attention_params(c, a);
    p.workspace = static_cast<char*>(workspace);
    const AttentionPlan plan = plan_attention(c, a, dev);
    p.row_blocks = plan.row_blocks;
    return with_format(c, [&](auto d, auto g) {
        if (plan.row_blocks > 0) return launch_decode_t<d.value, g.value>(p, plan, stream, pdl);
        return launch_prompt_t<d.value, g.value>(p, plan, stream, pdl);
    });
}

}  // namespace w4a16
