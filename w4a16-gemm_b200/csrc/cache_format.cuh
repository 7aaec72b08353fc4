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

// Neither kernel here lets the next one start early: its waiting CTAs take the place of CTAs that
// have work (reads of 8192 tokens of 8 heads back to back: 8.8 us a call with a trigger, 7.7 without).
constexpr int kAppendThreads = 256;

// 8 values -> 8 codes (one word), with the group's (scale, minimum).
//
// The quotient is a product with the reciprocal, at most 2^-18 off for quotients up to 16; only where
// it comes within 10^-4 of the middle between two codes (one warp in 20) is the division done, so
// that codes are those of the IEEE quotient.  (8192 tokens of 8 heads, fp16: 20 us, with eight divisions a
// lane 33 us.)
template <int G>
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], uint32_t& pair) {
    uint32_t big = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) big = max(big, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    if (big > __float_as_uint(W4A16_CACHE_LIMIT)) {           // too large, infinite or NaN
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -W4A16_CACHE_LIMIT), W4A16_CACHE_LIMIT) : 0.f;
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
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
    const float inv = sc > 0.f ? __frcp_rn(sc) : 0.f;         // a scale of 0 makes every quotient 0
    constexpr float kRound = 12582912.f;                      // 1.5 2^23: adding it rounds to whole numbers, halves to even
    float r[8], far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float q = fminf(fmaxf(__fmul_rn(__fsub_rn(x[j], mn), inv), 0.f), 15.f);
        r[j] = __fsub_rn(__fadd_rn(q, kRound), kRound);
        far = fmaxf(far, fabsf(__fsub_rn(q, r[j])));
    }
    if (far > 0.4999f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[j], mn), sc)), 0.f), 15.f);
    }
    // four codes are a whole number below 2^16, exact in fp32
    const float w0 = fmaf(fmaf(fmaf(r[3], 16.f, r[2]), 16.f, r[1]), 16.f, r[0]);
    const float w1 = fmaf(fmaf(fmaf(r[7], 16.f, r[6]), 16.f, r[5]), 16.f, r[4]);
    return __byte_perm(__float_as_uint(w0 + 8388608.f), __float_as_uint(w1 + 8388608.f), 0x5410);
}

// D / 8 lanes hold one vector (a key, value or query of one token and head), 8 values a
// lane.  2^log_par such lane groups share a token: its cosines and sines are loaded once a
// lane and serve every vector that the lane takes.  The other half of a pair is fetched from
// its lane as 16-bit words.  Bound by memory with queries (8192 tokens of 64 and 8 heads, bf16:
// 64 us, 4880 GB/s), by the quantisation's instructions without.
template <int D, int G, bool BF16, bool ROT>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr int L = D / 8;
    using F = CacheFmt<D, G>;
    pdl_wait();
    const int64_t group = ((int64_t)blockIdx.x * kAppendThreads + threadIdx.x) / L;
    const int l = threadIdx.x % L, par = 1 << p.log_par;
    const int64_t token_raw = group >> p.log_par;
    const int sub = (int)(group & (par - 1));
    const bool live = token_raw < p.tokens;               // lanes of a warp stay together for the shuffles
    const int64_t token = live ? token_raw : p.tokens - 1;
    const int hk = p.c.kv_heads;

    const int64_t slot = __ldg(p.slots + token);
    const int64_t page = slot >> p.c.page_shift;
    const bool store = live && slot >= 0 && page < p.c.num_pages;
    const int row = (int)(slot & ((1 << p.c.page_shift) - 1));
    const uint4 zero = make_uint4(0, 0, 0, 0);

    auto kv_vector = [&](int vec) {
        if (!live || vec >= 2 * hk) return zero;
        const uint16_t* src = vec < hk ? p.k + token * p.k_token + vec * p.k_head : p.v + token * p.v_token + (vec - hk) * p.v_head;
        return __ldg(reinterpret_cast<const uint4*>(src) + l);
    };
    auto q_vector = [&](int vec) {
        return live && vec < p.q_heads ? __ldg(reinterpret_cast<const uint4*>(p.q + token * p.q_token + vec * p.q_head) + l) : zero;
    };
    constexpr int QB = 4;                                 // queries in flight
    uint4 kv = kv_vector(sub), q[QB];
    if constexpr (ROT) {
#pragma unroll
        for (int i = 0; i < QB; ++i) q[i] = q_vector(sub + (i << p.log_par));
    }

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
            if (!p.interleaved && l < span) {             // a c - b s here, b c + a s in the other half's lane
#pragma unroll
                for (int j = 0; j < 8; ++j) sn[j] = -sn[j];
            }
        }
    }
    // turns a vector's values (every lane of the warp comes here: the other half is another lane's)
    auto turn = [&](const uint4& raw, float (&x)[8]) {
        if (p.interleaved) {
            if (turned) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = x[2 * j], b = x[2 * j + 1];
                    x[2 * j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
                    x[2 * j + 1] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
                }
            }
        } else {
            uint4 o;
            o.x = __shfl_xor_sync(0xffffffffu, raw.x, span);
            o.y = __shfl_xor_sync(0xffffffffu, raw.y, span);
            o.z = __shfl_xor_sync(0xffffffffu, raw.z, span);
            o.w = __shfl_xor_sync(0xffffffffu, raw.w, span);
            float y[8];
            unpack8<BF16>(o, y);
            if (turned) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(y[j], sn[j]));
            }
        }
    };

    const int kv_rounds = (2 * hk + par - 1) >> p.log_par;
    for (int it = 0; it < kv_rounds; ++it) {
        const int vec = sub + (it << p.log_par);
        const bool is_v = vec >= hk;
        const uint4 raw = kv;
        if (it + 1 < kv_rounds) kv = kv_vector(vec + par);
        float x[8];
        unpack8<BF16>(raw, x);
        if constexpr (ROT) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j];
            turn(raw, y);
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = y[j];
            }
        }
        uint32_t pair;
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
    if constexpr (ROT) {
        const int q_rounds = (p.q_heads + par - 1) >> p.log_par;
        for (int it = 0; it < q_rounds; it += QB) {
            uint4 raw[QB];
#pragma unroll
            for (int i = 0; i < QB; ++i) {
                raw[i] = q[i];
                if (it + QB < q_rounds) q[i] = q_vector(sub + ((it + QB + i) << p.log_par));
            }
#pragma unroll
            for (int i = 0; i < QB; ++i) {
                if (it + i >= q_rounds) break;
                const int vec = sub + ((it + i) << p.log_par);
                float x[8];
                unpack8<BF16>(raw[i], x);
                turn(raw[i], x);
                if (live && vec < p.q_heads)
                    reinterpret_cast<uint4*>(p.q_out + (token * p.q_heads + vec) * D)[l] = pack8<BF16>(x);
            }
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

// D / 8 lanes hold one token and head, 8 keys and 8 values a lane, of kReadVecs of them: stores
// are then whole 512-byte runs of a warp.  Bound by memory: 65536 tokens of 8 heads 56.7 us, 6000
// GB/s (with one vector a lane 73.6, two 60.8, eight 60.0; with 16 neighbouring values a lane, whose
// stores fill half sectors, 72).
constexpr int kReadVecs = 4;

template <int D, int G, bool BF16>
__global__ void __launch_bounds__(kReadThreads)
cache_read_kernel(const __grid_constant__ CacheView c, const int64_t* __restrict__ slots, int64_t tokens,
                  uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    constexpr int L = D / 8, PER = kReadThreads / L;             // vectors that a CTA reads at a time
    using F = CacheFmt<D, G>;
    pdl_wait();
    const int l = threadIdx.x % L;
    const int64_t first = (int64_t)blockIdx.x * (PER * kReadVecs) + threadIdx.x / L;
    uint32_t w[kReadVecs][2], pair[kReadVecs][2];
#pragma unroll
    for (int i = 0; i < kReadVecs; ++i) {
        const uint32_t vec = (uint32_t)(first + i * PER);        // tokens * heads < 2^31
        const uint32_t token = vec / (uint32_t)c.kv_heads, head = vec % (uint32_t)c.kv_heads;
        const int64_t slot = token < tokens ? __ldg(slots + token) : -1;
        const int64_t page = slot >> c.page_shift;
        w[i][0] = w[i][1] = pair[i][0] = pair[i][1] = 0u;
        if (slot >= 0 && page < c.num_pages) {
            const uint32_t ps = 1u << c.page_shift, row = (uint32_t)slot & (ps - 1);
            const uint8_t* b = cache_block(c, page, (int)head);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                w[i][t] = *reinterpret_cast<const uint32_t*>(b + t * ps * F::CODE + row * F::CODE + l * 4);
                pair[i][t] = *reinterpret_cast<const uint32_t*>(b + 2 * ps * F::CODE + t * ps * F::PAIR + row * F::PAIR + (l * 8 / G) * 4);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kReadVecs; ++i) {
        const int64_t vec = first + i * PER;
        if (vec >= tokens * c.kv_heads) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const __half2 ph = *reinterpret_cast<const __half2*>(&pair[i][t]);
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = cached_value(w[i][t], j, __low2float(ph), __high2float(ph));
            reinterpret_cast<uint4*>((t ? v : k) + vec * D)[l] = pack8<BF16>(f);
        }
    }
}

}  // namespace w4a16
