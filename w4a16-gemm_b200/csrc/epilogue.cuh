// What a product does with its sums before they are stored (w4a16_linear), and the activations that the
// experts' products share with it.
//
//     plain:  y = act(z + bias) + residual
//     gated:  y_j = act(z_g + bias_g) * (z_u + bias_u) + residual_j
//
// z are the fp32 sums; everything up to the one rounding to fp16 is fp32.  Rows of a gated weight
// alternate in runs of eight: rows 16i .. 16i + 7 are rows 8i .. 8i + 7 of the gate, the eight after
// them those of the other factor.  An n16 block of weights then holds both factors of eight results:
// in an m16n8k16 accumulator they are elements i and i + 2 of one lane, in TMEM lanes l and l + 8 of
// one warp, so that no sum leaves its warp to meet its partner.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "internal.h"

namespace w4a16 {

// The activations in fp32.  erf is CUDA's: below z = -3, where 1 + erf cancels, gelu is off by up to |z| 2^-24, a step or
// two of fp16's smallest.
//
// z * sigmoid(t).  exp and the division are the fast ones: a few fp32 ulps for |t| up to 88 (where the
// result has vanished in 16 bits), against the 2^-11 of the rounding that follows.
__device__ __forceinline__ float times_sigmoid(float z, float t) {
    return __fdividef(z, 1.f + __expf(-t));
}

__device__ __forceinline__ float activate(float z, int activation) {
    switch (activation) {
        case W4A16_ACTIVATION_RELU: return z < 0.f ? 0.f : z;          // NaN stays
        case W4A16_ACTIVATION_SILU: return times_sigmoid(z, z);
        case W4A16_ACTIVATION_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
        case W4A16_ACTIVATION_GELU_TANH:                               // (1 + tanh u) / 2 = sigmoid(2u)
            return times_sigmoid(z, 1.5957691f * (z + 0.044715f * z * z * z));
        default: return z;
    }
}

__device__ __forceinline__ float half_at(const void* p, size_t i) {
    return __half2float(static_cast<const __half*>(p)[i]);
}

// One finished sum (gated: both factors') of token tok, at column col of the product's N, into y.
template <int EPI>
__device__ __forceinline__ void store_epilogue(__half* __restrict__ y, const Epilogue& e, int tok, int N, int col, float z,
                                               float zu) {
    if (e.bias) {
        z += half_at(e.bias, col);
        if (EPI == kEpiGated) zu += half_at(e.bias, col + 8);
    }
    float v = activate(z, e.activation);
    size_t o = (size_t)tok * N + col;
    if (EPI == kEpiGated) {
        v *= zu;
        o = (size_t)tok * (N / 2) + 8 * (col / 16) + col % 8;
    }
    if (e.residual) v += half_at(e.residual, o);
    y[o] = __float2half_rn(v);
}

}  // namespace w4a16
