// Device code of the expert layer.
#include <cuda_runtime.h>

#include "internal.h"
#include "launch.cuh"
#include "moe_experts.cuh"

namespace w4a16 {

cudaError_t read_moe_device_status(int* code, bool reset) {
    cudaError_t err = cudaMemcpyFromSymbol(code, w4a16_device_status, sizeof(int));
    if (err != cudaSuccess || !reset) return err;
    const int zero = 0;
    return cudaMemcpyToSymbol(w4a16_device_status, &zero, sizeof(int));
}

cudaError_t run_moe_wait_limit_check() {
    wait_limit_kernel<<<1, 32>>>(1, kDevTimeoutExperts);
    const cudaError_t err = cudaGetLastError();
    return err != cudaSuccess ? err : cudaDeviceSynchronize();
}

static MoePlan plan_of(const w4a16_moe_args& a, const DeviceInfo& dev) {
    return moe_plan(a.tokens, a.k, a.num_experts, a.hidden, a.inner, dev.num_sms, a.gate_up_group == 128 && a.down_group == 128);
}

size_t moe_workspace(const w4a16_moe_args& a, const DeviceInfo& dev) { return plan_of(a, dev).bytes; }

template <int G, bool GATED>
static cudaError_t launch_product_t(const MoeParams& p, int grid, cudaStream_t stream, bool pdl) {
    auto kern = moe_product_kernel<G, GATED>;
    const cudaError_t err = ensure_max_dynamic_smem(reinterpret_cast<const void*>(kern));
    if (err != cudaSuccess) return err;
    return launch(kern, dim3(grid), kMoeThreads, MoeCfg::SMEM, stream, pdl, p);
}

template <bool GATED>
static cudaError_t launch_product(const MoeParams& p, int G, int grid, cudaStream_t stream, bool pdl) {
    return G == 64 ? launch_product_t<64, GATED>(p, grid, stream, pdl) : launch_product_t<128, GATED>(p, grid, stream, pdl);
}

cudaError_t launch_moe_experts(const w4a16_moe_args& a, const DeviceInfo& dev, void* workspace, cudaStream_t stream, bool pdl) {
    MoeParams p = {};
    p.x = static_cast<const __half*>(a.x);
    p.words[0] = a.gate_up_wp;
    p.words[1] = a.down_wp;
    p.scales[0] = static_cast<const __half*>(a.gate_up_scales);
    p.scales[1] = static_cast<const __half*>(a.down_scales);
    p.experts = a.experts;
    p.weights = a.weights;
    p.residual = static_cast<const __half*>(a.residual);
    p.y = static_cast<__half*>(a.y);
    p.workspace = static_cast<char*>(workspace);
    p.plan = plan_of(a, dev);
    p.entries = (int32_t)(a.tokens * a.k);
    p.k = a.k;
    p.num_experts = a.num_experts;
    p.hidden = a.hidden;
    p.inner = a.inner;
    p.activation = a.activation;
    cudaError_t err = p.plan.few ? cudaSuccess : launch(moe_plan_kernel, dim3(1), kMoePlanThreads, 0, stream, pdl, p);
    if (p.plan.grouped) {
        constexpr int rows = kMoeGatherThreads / 32;
        if (err == cudaSuccess)
            err = launch(moe_gather_kernel, dim3((unsigned)((p.entries + rows - 1) / rows)), kMoeGatherThreads, 0, stream, pdl, p);
        GroupedArgs g = {a.gate_up_wp, p.workspace + p.plan.rows_at, a.gate_up_scales, p.workspace + p.plan.inner_at, p.entries,
                         a.num_experts, 2 * a.inner, a.hidden, a.gate_up_group, true, a.activation,
                         {reinterpret_cast<MoeHead*>(p.workspace), reinterpret_cast<MoeTile*>(p.workspace + p.plan.tiles_at),
                          2 * a.inner / 16, a.hidden / a.gate_up_group}, stream, pdl};
        if (err == cudaSuccess) err = launch_grouped(g, dev);
        g.wp = a.down_wp;
        g.x = p.workspace + p.plan.inner_at;
        g.scales = a.down_scales;
        g.y = p.workspace + p.plan.out_at;
        g.N = a.hidden;
        g.K = a.inner;
        g.G = a.down_group;
        g.gated = false;
        g.groups.blocks = a.hidden / 16;
        g.groups.scale_rows = a.inner / a.down_group;
        if (err == cudaSuccess) err = launch_grouped(g, dev);
    } else {
        if (err == cudaSuccess) err = launch_product<true>(p, a.gate_up_group, dev.num_sms, stream, pdl);
        if (err == cudaSuccess) err = launch_product<false>(p, a.down_group, dev.num_sms, stream, pdl);
    }
    if (err != cudaSuccess) return err;
    if (p.plan.grouped) return launch(moe_grouped_finish_kernel, dim3((unsigned)a.tokens), kMoeFinishThreads, 0, stream, pdl, p);
    const auto finish = [&](auto kern, int slices) {
        const int cols = 4 * kMoeFinishThreads / slices;
        return launch(kern, dim3((unsigned)a.tokens, (unsigned)((a.hidden + cols - 1) / cols)), kMoeFinishThreads, 0, stream, pdl, p);
    };
    // a few tokens' parts are spread over threads, a prompt's fill the machine as they are
    return a.tokens <= 64 ? finish(moe_finish_kernel<4>, 4) : finish(moe_finish_kernel<1>, 1);
}

}  // namespace w4a16
