// The 4-bit key/value cache's format, and the kernels that write it (quantising, with
// rotary positions) and read it back.  Included by cache.cu only.
//
// One (page, head) block: key codes [ps][D/2] | value codes [ps][D/2] | key pairs
// [ps][D/G] | value pairs, a pair being fp16 (scale, minimum).  Codes stay in the order of
// the values (low nibble first): a token's codes are one run of D/2 bytes, whole bytes belong to
// one token (tokens are written by independent threads), and both attention kernels take
// any order of the contraction index as long as the other operand follows it.
//
//     minimum = fp16(min x), scale = fp16(max(max x - minimum, 0) / 15)
//     code    = clamp(round_half_even((x - minimum) / scale), 0, 15)     (0 where scale is 0)
//     value   = code * scale + minimum
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "internal.h"
#include "ptx.cuh"

namespace w4a16 {

// A cache as the kernels see it.
struct CacheView {
    uint8_t* data;
    int64_t num_pages;
    int32_t page_shift;      // log2(page_size)
    int32_t kv_heads;
    uint32_t block_bytes;    // one (page, head) block
};

template <int D, int G>
struct CacheFmt {
    static_assert((D == 64 || D == 128) && (G == 64 || G == 128) && G <= D, "cache format");
    static constexpr int CODE = D / 2;          // bytes of codes of one token, one of K / V
    static constexpr int NG = D / G;            // groups of a token
    static constexpr int PAIR = 4 * NG;         // bytes of its (scale, minimum) pairs
    static constexpr int TOKEN = 2 * (CODE + PAIR);
};

__host__ __device__ __forceinline__ uint32_t cache_block_bytes(int page_size, int D, int G) {
    return (uint32_t)page_size * (uint32_t)(D + 8 * (D / G));
}

__device__ __forceinline__ uint8_t* cache_block(const CacheView& c, int64_t page, int head) {
    return c.data + (page * c.kv_heads + head) * (int64_t)c.block_bytes;
}

// ------------------------------------------------------------------ 16-bit activations
__device__ __forceinline__ void unpack16(uint32_t w, bool bf16, float& a, float& b) {
    if (bf16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const __half2 h = *reinterpret_cast<const __half2*>(&w);
        a = __low2float(h);
        b = __high2float(h);
    }
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
    unpack16(w.x, BF16, f[0], f[1]);
    unpack16(w.y, BF16, f[2], f[3]);
    unpack16(w.z, BF16, f[4], f[5]);
    unpack16(w.w, BF16, f[6], f[7]);
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack16(f[0], f[1], BF16), pack16(f[2], f[3], BF16), pack16(f[4], f[5], BF16),
                      pack16(f[6], f[7], BF16));
}

// ------------------------------------------------------------------ append
struct AppendParams {
    CacheView c;
    const uint16_t *k, *v, *q;
    uint16_t* q_out;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head;    // strides in elements
    const int64_t* slots;
    const int64_t* positions;
    const float* cos_sin;
    int64_t axis_stride, max_pos;
    int64_t tokens;
    int32_t q_heads;         // 0: no queries
    int32_t axes;
    int32_t end0, end1;      // angles below end0 are axis 0's, below end1 axis 1's
    int32_t rotary_dim;
    int32_t interleaved;
    int32_t log_par;         // log2 of the lane groups that share a token's vectors
};

constexpr int kAppendThreads = 256;

// 8 values -> 8 codes (one word), with the group's (scale, minimum).
template <int G>
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], uint32_t& pair) {
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -W4A16_CACHE_LIMIT), W4A16_CACHE_LIMIT) : 0.f;
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
    }
#pragma unroll
    for (int d = 1; d < G / 8; d *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    const __half mn_h = __float2half_rn(lo);
    const float mn = __half2float(mn_h);
    const __half sc_h = __float2half_rn(__fdiv_rn(fmaxf(__fsub_rn(hi, mn), 0.f), 15.f));
    const float sc = __half2float(sc_h);
    pair = (uint32_t)__half_as_ushort(sc_h) | ((uint32_t)__half_as_ushort(mn_h) << 16);
    uint32_t w = 0;
    if (sc > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float r = rintf(__fdiv_rn(__fsub_rn(x[j], mn), sc));
            w |= (uint32_t)(int)fminf(fmaxf(r, 0.f), 15.f) << (4 * j);
        }
    }
    return w;
}

// D / 8 lanes hold one vector (a key, value or query of one token and head), 8 values a
// lane.  2^log_par such lane groups share a token: its cosines and sines are loaded once a
// lane and serve every vector that the lane takes.  Bound by memory: see DESIGN for figures.
template <int D, int G, bool BF16, bool ROT>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int L = D / 8;
    using F = CacheFmt<D, G>;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t group = ((int64_t)blockIdx.x * kAppendThreads + threadIdx.x) / L;
    const int l = threadIdx.x % L, par = 1 << p.log_par;
    const int64_t token_raw = group >> p.log_par;
    const int sub = (int)(group & (par - 1));
    const bool live = token_raw < p.tokens;               // lanes of a warp stay together for the shuffles
    const int64_t token = live ? token_raw : p.tokens - 1;
    const int hk = p.c.kv_heads, vecs = 2 * hk + (ROT ? p.q_heads : 0);

    const int64_t slot = __ldg(p.slots + token);
    const int64_t page = slot >> p.c.page_shift;
    const bool store = live && slot >= 0 && page < p.c.num_pages;
    const int row = (int)(slot & ((1 << p.c.page_shift) - 1));

    float cs[8], sn[8];
    const int half = p.rotary_dim >> 1;
    const int span = p.rotary_dim >> 4;                   // lanes between the two halves of a pair
    const bool turned = ROT && l * 8 < p.rotary_dim;
    if constexpr (ROT) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { cs[j] = 1.f; sn[j] = 0.f; }
        if (turned) {
            int64_t pos[3];
#pragma unroll
            for (int a = 0; a < 3; ++a)
                pos[a] = a < p.axes ? min(max(__ldg(p.positions + a * p.axis_stride + token), (int64_t)0), p.max_pos - 1) : 0;
            const int n = p.interleaved ? 4 : 8;          // angles of this lane
            const int i0 = p.interleaved ? l * 4 : (l < span ? l : l - span) * 8;
            if (p.axes == 1) {
                const float* t = p.cos_sin + pos[0] * p.rotary_dim + i0;
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    if (j < n) {
                        const float4 a = __ldg(reinterpret_cast<const float4*>(t + j));
                        const float4 b = __ldg(reinterpret_cast<const float4*>(t + half + j));
                        cs[j] = a.x; cs[j + 1] = a.y; cs[j + 2] = a.z; cs[j + 3] = a.w;
                        sn[j] = b.x; sn[j + 1] = b.y; sn[j + 2] = b.z; sn[j + 3] = b.w;
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) {
                        const int i = i0 + j;
                        const float* t = p.cos_sin + (i < p.end0 ? pos[0] : i < p.end1 ? pos[1] : pos[2]) * p.rotary_dim + i;
                        cs[j] = __ldg(t);
                        sn[j] = __ldg(t + half);
                    }
            }
        }
    }

    auto source = [&](int vec) -> const uint16_t* {
        if (vec < hk) return p.k + token * p.k_token + vec * p.k_head;
        if (vec < 2 * hk) return p.v + token * p.v_token + (vec - hk) * p.v_head;
        return p.q + token * p.q_token + (int64_t)(vec - 2 * hk) * p.q_head;
    };
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int rounds = (vecs + par - 1) >> p.log_par;
    uint4 next = live && sub < vecs ? __ldg(reinterpret_cast<const uint4*>(source(sub)) + l) : zero;
    for (int it = 0; it < rounds; ++it) {
        const int vec = sub + (it << p.log_par);
        const uint4 raw = next;
        if (it + 1 < rounds) {
            const int nv = vec + par;
            next = live && nv < vecs ? __ldg(reinterpret_cast<const uint4*>(source(nv)) + l) : zero;
        }
        float x[8];
        unpack8<BF16>(raw, x);
        const bool is_v = vec >= hk && vec < 2 * hk;
        if constexpr (ROT) {
            if (p.interleaved) {
                if (turned && !is_v) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = x[2 * j], b = x[2 * j + 1];
                        x[2 * j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
                        x[2 * j + 1] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float o = __shfl_xor_sync(0xffffffffu, x[j], span);
                    const float xc = __fmul_rn(x[j], cs[j]), os = __fmul_rn(o, sn[j]);
                    if (turned && !is_v) x[j] = l < span ? __fsub_rn(xc, os) : __fadd_rn(xc, os);
                }
            }
        }
        uint32_t pair;
        if (ROT && vec >= 2 * hk) {
            if (live && vec < vecs)
                reinterpret_cast<uint4*>(p.q_out + (token * p.q_heads + (vec - 2 * hk)) * D)[l] = pack8<BF16>(x);
        }
        // every lane of the warp takes part in the shuffles of the group's minimum and maximum
        const uint32_t codes = quantise8<G>(x, pair);
        if (store && vec < 2 * hk) {
            const int which = is_v ? 1 : 0;
            uint8_t* b = cache_block(p.c, page, vec - which * hk);
            const uint32_t ps = 1u << p.c.page_shift;
            *reinterpret_cast<uint32_t*>(b + which * ps * F::CODE + row * F::CODE + l * 4) = codes;
            if (l % (G / 8) == 0)
                *reinterpret_cast<uint32_t*>(b + 2 * ps * F::CODE + which * ps * F::PAIR + row * F::PAIR + (l / (G / 8)) * 4) = pair;
        }
    }
}

// ------------------------------------------------------------------ read back
constexpr int kReadThreads = 256;

// Value j (0..7) of a word of codes as fp32: code * scale + minimum, the product exact (4 by
// 11 bits), the sum rounded once.
__device__ __forceinline__ float cached_value(uint32_t w, int j, float sc, float mn) {
    // 2^23 + code, less 2^23
    const float c = __uint_as_float(0x4B000000u | ((w >> (4 * j)) & 15u)) - 8388608.f;
    return fmaf(c, sc, mn);
}

// D / 16 lanes hold one token and head, 16 keys and 16 values a lane.
template <int D, int G, bool BF16>
__global__ void __launch_bounds__(kReadThreads)
cache_read_kernel(const __grid_constant__ CacheView c, const int64_t* __restrict__ slots, int64_t tokens,
                  uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    constexpr int L = D / 16;
    using F = CacheFmt<D, G>;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t i = (int64_t)blockIdx.x * kReadThreads + threadIdx.x;
    const int64_t vec = i / L;
    const int l = (int)(i % L);
    const int64_t token = vec / c.kv_heads;
    if (token >= tokens) return;
    const int head = (int)(vec % c.kv_heads);
    const int64_t slot = __ldg(slots + token);
    const int64_t page = slot >> c.page_shift;
    uint2 w[2] = {};
    uint32_t pair[2] = {};
    if (slot >= 0 && page < c.num_pages) {
        const uint32_t ps = 1u << c.page_shift, row = (uint32_t)slot & (ps - 1);
        const uint8_t* b = cache_block(c, page, head);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            w[t] = *reinterpret_cast<const uint2*>(b + t * ps * F::CODE + row * F::CODE + l * 8);
            pair[t] = *reinterpret_cast<const uint32_t*>(b + 2 * ps * F::CODE + t * ps * F::PAIR + row * F::PAIR + (l * 16 / G) * 4);
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const __half2 ph = *reinterpret_cast<const __half2*>(&pair[t]);
        const float sc = __low2float(ph), mn = __high2float(ph);
        float f[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[j] = cached_value(w[t].x, j, sc, mn);
            g[j] = cached_value(w[t].y, j, sc, mn);
        }
        uint4* out = reinterpret_cast<uint4*>((t ? v : k) + vec * D + l * 16);
        out[0] = pack8<BF16>(f);
        out[1] = pack8<BF16>(g);
    }
}

}  // namespace w4a16
