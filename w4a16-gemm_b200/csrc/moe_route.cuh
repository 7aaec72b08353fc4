// The router of a mixture of experts: softmax of a token's logits over its experts, and the k largest.
//
//     p_e = exp(l_e - max) / sum,   sum over all experts, or over the chosen ones (renormalize)
//
// Experts come in falling order of their logits, equal ones by index.  What is -inf or NaN is no candidate:
// where fewer than k remain, the rest of the row is expert -1 with weight 0.  One warp a token; its
// logits stay in registers (VALUES a lane) as integers of the same order, so that a choice is two warp
// reductions: the largest, then the lowest index that has it.  A decode step is bound by the launch, a
// prompt by the latency of a warp's 2 k reductions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "internal.h"
#include "ptx.cuh"

namespace w4a16 {

constexpr int kRouteWarps = 4;

struct RouteArgs {
    const void* logits;
    int64_t row_stride;
    float* weights;            // dense [tokens][k]
    int32_t* experts;          // dense [tokens][k]
    int64_t tokens;
    int32_t num_experts, k;
    bool renormalize;
};

// Integers that order as the floats do; 0 for NaN and -inf (no float maps to 0).  -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float f) {
    if (!(f > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(f + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// exp(l - max) for l <= max, both above -inf; 1 where they are equal, infinities included.
__device__ __forceinline__ float exp_below(float l, float max) { return l == max ? 1.f : expf(l - max); }

__device__ __forceinline__ float logit_at(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float logit_at(const __half* p, int64_t i) { return __half2float(p[i]); }
__device__ __forceinline__ float logit_at(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }

template <typename T, int VALUES>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_kernel(RouteArgs a) {
    pdl_wait();
    pdl_launch_dependents();      // after the wait: the next kernel may read ahead what the one before this wrote
    const int lane = threadIdx.x & 31;
    const int64_t token = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    const T* const row = static_cast<const T*>(a.logits) + token * a.row_stride;
    uint32_t v[VALUES];
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
        const int e = i * 32 + lane;
        v[i] = e < a.num_experts ? ordered(logit_at(row, e)) : 0u;
    }
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) best = max(best, v[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    const float largest = unordered(best);
    float all = 0.f;
    if (!a.renormalize) {
#pragma unroll
        for (int i = 0; i < VALUES; ++i) all += v[i] ? exp_below(unordered(v[i]), largest) : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    // lane j keeps choice j (k is at most a warp)
    float mine = 0.f, chosen = 0.f;
    int32_t expert = -1;
    for (int j = 0; j < a.k && best; ++j) {
        uint32_t first = 0xffffffffu;
#pragma unroll
        for (int i = VALUES - 1; i >= 0; --i)
            if (v[i] == best) first = (uint32_t)(i * 32 + lane);
        first = __reduce_min_sync(0xffffffffu, first);
        const float w = exp_below(unordered(best), largest);
        chosen += w;
        if (lane == j) {
            mine = w;
            expert = (int32_t)first;
        }
        best = 0;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) {
            if ((uint32_t)(i * 32 + lane) == first) v[i] = 0u;
            best = max(best, v[i]);
        }
        best = __reduce_max_sync(0xffffffffu, best);
    }
    if (lane < a.k) {
        a.weights[token * a.k + lane] = expert < 0 ? 0.f : mine / (a.renormalize ? chosen : all);
        a.experts[token * a.k + lane] = expert;
    }
}

}  // namespace w4a16
