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

// The activations in fp32, each good to 2^-16 or so of its own value down to z = -9: with a gate the other factor may be large
// where the activation is small.  exp and the division are the fast ones; exp's error grows with its argument t, 2 + 1.2 |t|
// fp32 ulps (26 at 20, where the factor is 2e-9), against the 2^-11 of the rounding that follows.
//
// z * sigmoid(t).
__device__ __forceinline__ float times_sigmoid(float z, float t) {
    return __fdividef(z, 1.f + __expf(-t));
}

// The normal distribution's Phi(z).  1 + erf(z / sqrt 2) would cancel below -3 (7 % off at -5, all of it from -5.5 on), so the
// smaller tail is made, Phi(-a) = exp(-a^2 / 2) r(a) at a = |z|: r falls from 1/2 as 1 / (a sqrt(2 pi)), and r / t is a polynomial of
// t = 1 / (1 + 0.3625 a), of degree 6 for a relative error of 7.7e-7 up to a = 14 (a weighted least-squares fit, the weights
// repeated until the error was level; 2.7e-6 in fp32).  erfcf is as good but longer:
// a prompt's plain product with bias and gelu, 2048 x 14336 x 4096, takes 341 us with it, 289 with erff, 260 with this.
__device__ __forceinline__ float normal_below(float z) {
    const float a = fabsf(z), t = __fdividef(1.f, fmaf(a, 0.3625f, 1.f));
    float q = 0.0480628535f;
    q = fmaf(q, t, -0.179742277f);
    q = fmaf(q, t, 0.175103799f);
    q = fmaf(q, t, 0.029682558f);
    q = fmaf(q, t, 0.139256671f);
    q = fmaf(q, t, 0.142936394f);
    q = fmaf(q, t, 0.144700378f);
    q *= t * __expf(-0.5f * a * a);
    return z < 0.f ? q : 1.f - q;
}

__device__ __forceinline__ float activate(float z, int activation) {
    switch (activation) {
        case W4A16_ACTIVATION_RELU: return z < 0.f ? 0.f : z;          // NaN stays
        case W4A16_ACTIVATION_SILU: return times_sigmoid(z, z);
        case W4A16_ACTIVATION_GELU: return z * normal_below(z);
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
