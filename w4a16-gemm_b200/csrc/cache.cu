// Device code of the 4-bit key/value cache: append, read back, attention.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "ptx.cuh"
#include "cache_format.cuh"
#include "cache_plan.h"
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

size_t cache_attention_workspace(const w4a16_cache& c, const w4a16_cache_attention_args& a, const DeviceInfo& dev) {
    return plan_attention(c, a, dev.num_sms).workspace;
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
    const int seg_rows = std::min(kCdRows, ap.max_q * ap.shared);
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
    const AttentionPlan plan = plan_attention(c, a, dev.num_sms);
    p.row_blocks = plan.row_blocks;
    return with_format(c, [&](auto d, auto g) {
        if (plan.row_blocks > 0) return launch_decode_t<d.value, g.value>(p, plan, stream, pdl);
        return launch_prompt_t<d.value, g.value>(p, plan, stream, pdl);
    });
}

}  // namespace w4a16
