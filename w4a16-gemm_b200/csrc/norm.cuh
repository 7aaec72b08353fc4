// Root-mean-square norm of rows, with the residual's addition:
//
//     h = x + residual,   y = h * weight / sqrt(mean(h^2) + eps)
//
// Everything between the inputs and the roundings of y and of the stored h is fp32; y comes from the
// unrounded h.  Bound by the memory's bandwidth: a row is read once and stays in registers between its
// sum and its scaling.  8 values (16 bytes) a load; THREADS threads own a row, each VPT such vectors.  What a
// row takes is its latency (loads, two barriers, stores), so the rows in flight count: 32 registers a thread, 2048
// threads an SM, a few bytes of spills included (8192 rows of 8192 with a residual, bf16: 118 -> 91 us; in a graph 85, 6.3 TB/s).
// The sum x + residual is stored as soon as it is made, so that what is kept of it may be scaled.  Rows of up to 256 values go to one
// warp or to a part of one (8 lanes a row of 64 values, 16 of 128): no shared memory, no barrier.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "internal.h"
#include "ptx.cuh"

namespace w4a16 {

template <typename T>
__device__ __forceinline__ float2 pair_to_float(uint32_t v) {
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

template <typename T>
__device__ __forceinline__ uint32_t float_to_pair(float a, float b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Eight values from p on (16-byte aligned), of a 16-bit type or of fp32.
template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&f)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
        const float4 a = p[0], b = p[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = pair_to_float<T>(u[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&f)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
            make_uint4(float_to_pair<T>(f[0], f[1]), float_to_pair<T>(f[2], f[3]), float_to_pair<T>(f[4], f[5]),
                       float_to_pair<T>(f[6], f[7]));
    }
}

// Sum over aligned groups of LANES lanes of a warp.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The row's sum over THREADS threads (all of them get it, added in the same order every time).
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* shared) {
    v = lane_sum<THREADS < 32 ? THREADS : 32>(v);
    if constexpr (THREADS > 32) {
        constexpr int W = THREADS / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) shared[warp] = v;
        __syncthreads();
        v = lane_sum<32>(lane < W ? shared[lane] : 0.f);
        __syncthreads();
    }
    return v;
}

struct NormArgs {
    const void* x;
    const void* weight;
    const void* residual;     // NULL: none
    void* y;
    void* residual_out;       // where h goes, if there is a residual
    int64_t rows;
    int32_t heads, dim;       // row r is head r % heads of token r / heads
    int64_t x_token, x_head, residual_token, residual_head, y_token, y_head, out_token, out_head;   // strides
    float eps;
};

// T: x, weight and y.  R: the residual's type, or void without one.
template <typename T, typename R, int THREADS, int VPT, int ROWS>
__global__ void __launch_bounds__(THREADS * ROWS, VPT <= 2 ? 2048 / (THREADS * ROWS) : 1) rms_norm_kernel(NormArgs a) {
    constexpr bool ADD = !std::is_same_v<R, void>;
    __shared__ float shared[THREADS > 32 ? THREADS / 32 : 1];
    pdl_wait();
    pdl_launch_dependents();      // after the wait: the next kernel may read ahead what the one before this wrote
    const int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
    const int dim = row < a.rows ? a.dim : 0;     // past the last row: nothing is read or written
    const int64_t token = row / a.heads, head = row - token * a.heads;
    const int64_t xo = token * a.x_token + head * a.x_head, yo = token * a.y_token + head * a.y_head;
    const int t = threadIdx.x % THREADS;
    float h[VPT][8], w[VPT][8];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int at = (i * THREADS + t) * 8;
        if (at < dim) {
            load8<T>(a.x, xo + at, h[i]);
            if constexpr (ADD) {
                float r[8];
                load8<R>(a.residual, token * a.residual_token + head * a.residual_head + at, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] += r[j];
                store8<R>(a.residual_out, token * a.out_token + head * a.out_head + at, h[i]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j], h[i][j], sum);
    sum = row_sum<THREADS>(sum, shared);
    const float n = (float)a.dim;
    // squares of large finite values (bf16 and fp32 reach 3e38) pass fp32, and those of values below 2^-60 or so, which count
    // where eps is as small, fall out of it: then the row is scaled by 2^-80 or 2^80 for its sum.  The first keeps every square of
    // 2^127 finite and loses none that counts beside it; with the second, for means below 2^-64, a row's squares stay
    // below 2^111, and full down to values of 2^-143.  Rows that share a warp share its shuffles, so a warp sums again if one of its
    // rows has to, and the others keep their first sum.
    const float mean = sum / n + a.eps;
    float scale = rsqrtf(mean);
    const bool again = !(mean >= 0x1p-64f && mean < INFINITY);
    if (THREADS < 32 ? __any_sync(0xffffffffu, again) : again) {
        const float s = mean < 1.f ? 0x1p80f : 0x1p-80f;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(h[i][j] * s, h[i][j] * s, sum);
        sum = row_sum<THREADS>(sum, shared);
        if (again) {
            scale = rsqrtf(sum / n + a.eps * s * s);
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] *= s;
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int at = (i * THREADS + t) * 8;
        if (at < dim) {
            load8<T>(a.weight, at, w[i]);      // the same for every row: there in L1
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * scale * w[i][j];
            store8<T>(a.y, yo + at, h[i]);
        }
    }
}

}  // namespace w4a16
