// Device code of a decoder layer's small operators: the norm with the residual's addition, the router of
// a mixture of experts.
#include <cuda_runtime.h>

#include "internal.h"
#include "launch.cuh"
#include "norm.cuh"
#include "moe_route.cuh"

namespace w4a16 {

// Widths by who owns a row: up to a warp for 256 values, then as few threads as hold it in two vectors each, since
// fewer threads a row are more rows in flight.
template <typename T, typename R>
static cudaError_t launch_norm_t(const NormArgs& a, cudaStream_t stream, bool pdl) {
    const int vecs = a.dim / 8;
    const auto grid = [&](int rows) { return dim3((unsigned)((a.rows + rows - 1) / rows)); };
    if (vecs <= 8) return launch(rms_norm_kernel<T, R, 8, 1, 32>, grid(32), 256, 0, stream, pdl, a);
    if (vecs <= 16) return launch(rms_norm_kernel<T, R, 16, 1, 16>, grid(16), 256, 0, stream, pdl, a);
    if (vecs <= 32) return launch(rms_norm_kernel<T, R, 32, 1, 8>, grid(8), 256, 0, stream, pdl, a);
    if (vecs <= 128) return launch(rms_norm_kernel<T, R, 64, 2, 1>, grid(1), 64, 0, stream, pdl, a);
    if (vecs <= 256) return launch(rms_norm_kernel<T, R, 128, 2, 1>, grid(1), 128, 0, stream, pdl, a);
    if (vecs <= 512) return launch(rms_norm_kernel<T, R, 256, 2, 1>, grid(1), 256, 0, stream, pdl, a);
    if (vecs <= 1024) return launch(rms_norm_kernel<T, R, 512, 2, 1>, grid(1), 512, 0, stream, pdl, a);
    if (vecs <= 2048) return launch(rms_norm_kernel<T, R, 1024, 2, 1>, grid(1), 1024, 0, stream, pdl, a);
    return launch(rms_norm_kernel<T, R, 1024, 4, 1>, grid(1), 1024, 0, stream, pdl, a);
}

template <typename T>
static cudaError_t launch_norm_r(const NormArgs& a, bool residual_f32, cudaStream_t stream, bool pdl) {
    if (!a.residual) return launch_norm_t<T, void>(a, stream, pdl);
    return residual_f32 ? launch_norm_t<T, float>(a, stream, pdl) : launch_norm_t<T, T>(a, stream, pdl);
}

cudaError_t launch_rms_norm(const w4a16_norm_args& n, cudaStream_t stream, bool pdl) {
    NormArgs a = {n.x, n.weight, n.residual, n.y, n.residual_out, n.tokens * n.heads, n.heads, n.dim,
                  n.x_token_stride, n.x_head_stride, n.residual_token_stride, n.residual_head_stride,
                  n.y_token_stride, n.y_head_stride, n.residual_out_token_stride, n.residual_out_head_stride, n.eps};
    return n.dtype == W4A16_ACT_BF16 ? launch_norm_r<__nv_bfloat16>(a, n.residual_f32 != 0, stream, pdl)
                                     : launch_norm_r<__half>(a, n.residual_f32 != 0, stream, pdl);
}

template <typename T>
static cudaError_t launch_route_t(const RouteArgs& a, cudaStream_t stream, bool pdl) {
    const dim3 grid((unsigned)((a.tokens + kRouteWarps - 1) / kRouteWarps));
    const int threads = kRouteWarps * 32;
    if (a.num_experts <= 64) return launch(moe_route_kernel<T, 2>, grid, threads, 0, stream, pdl, a);
    if (a.num_experts <= 256) return launch(moe_route_kernel<T, 8>, grid, threads, 0, stream, pdl, a);
    return launch(moe_route_kernel<T, 32>, grid, threads, 0, stream, pdl, a);
}

cudaError_t launch_moe_route(const void* logits, int32_t dtype, int64_t row_stride, int64_t tokens, int32_t num_experts,
                             int32_t k, bool renormalize, float* weights, int32_t* experts, cudaStream_t stream, bool pdl) {
    const RouteArgs a = {logits, row_stride, weights, experts, tokens, num_experts, k, renormalize};
    if (dtype == W4A16_LOGITS_F32) return launch_route_t<float>(a, stream, pdl);
    return dtype == W4A16_ACT_BF16 ? launch_route_t<__nv_bfloat16>(a, stream, pdl) : launch_route_t<__half>(a, stream, pdl);
}

}  // namespace w4a16
