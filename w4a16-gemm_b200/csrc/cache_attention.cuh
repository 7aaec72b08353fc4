// Attention over the 4-bit key/value cache.  Included by cache.cu only.
//
// Query i of the T of a sequence of L cached tokens sits at position p = L - T + i and sees
// the tokens t of [lo, hi): hi = min(p + 1, L) if causal, else L; lo = max(0, p + 1 - window)
// with a window, else 0.  With K_t = s_t c_t + m_t (codes c_t),
//     out = sum_t w_t V_t / sum_t w_t,   w_t = exp(scale q.K_t - max)
// and zeros where nothing is seen.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache_format.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace w4a16 {

struct AttentionParams {
    CacheView c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    int64_t q_token, q_head;     // strides in elements
    int64_t q_tokens;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    const int32_t* cu_q;
    float scale_log2;            // scale * log2(e): scores are kept in units of log 2
    int32_t table_pages, batch, max_q;
    int32_t shared;              // query heads of a key head
    int32_t window;
    bool causal, bf16;
};

// One sequence's queries and cached tokens, clamped to what the arrays hold.
struct SeqSpan {
    int64_t q0;      // first query's token
    int32_t nq;      // queries
    int32_t len;     // cached tokens
};

__device__ __forceinline__ SeqSpan seq_span(const AttentionParams& p, int b) {
    SeqSpan s;
    const int64_t most = (int64_t)p.table_pages << p.c.page_shift;
    s.len = (int32_t)min((int64_t)max(__ldg(p.seq_lens + b), 0), most);
    if (p.cu_q) {
        const int64_t a = min((int64_t)max(__ldg(p.cu_q + b), 0), p.q_tokens);
        const int64_t e = min((int64_t)max(__ldg(p.cu_q + b + 1), 0), p.q_tokens);
        s.q0 = a;
        s.nq = (int32_t)min(max(e - a, (int64_t)0), (int64_t)p.max_q);
    } else {
        s.q0 = b;
        s.nq = b < p.q_tokens ? 1 : 0;
    }
    return s;
}

// The tokens [lo, hi) that a query at position pos sees.
__device__ __forceinline__ int2 seen_range(const AttentionParams& p, int pos, int len) {
    const int hi = p.causal ? min(pos + 1, len) : len;
    const int lo = p.window ? max(0, pos + 1 - p.window) : 0;
    return make_int2(min(lo, len), hi);
}

// A page of a sequence; what the table should not hold is led back into the cache.
__device__ __forceinline__ int64_t page_of(const AttentionParams& p, int b, int index) {
    const int64_t page = __ldg(p.table + b * p.table_stride + index);
    return min(max(page, (int64_t)0), p.c.num_pages - 1);
}

// One warp a query row, the head's D values spread over its lanes, one cached token a step.
template <int D, int G>
__global__ void __launch_bounds__(256) cache_attention_kernel(const __grid_constant__ AttentionParams p) {
    using F = CacheFmt<D, G>;
    constexpr int N = D / 32;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int heads = p.shared * p.c.kv_heads;
    const int b = (int)(w / ((int64_t)p.max_q * heads));
    if (b >= p.batch) return;
    const int i = (int)(w / heads % p.max_q), head = (int)(w % heads);
    const SeqSpan s = seq_span(p, b);
    if (i >= s.nq) return;
    const int2 seen = seen_range(p, s.len - s.nq + i, s.len);
    float q[N], acc[N], top = -INFINITY, sum = 0.f;
    const uint16_t* qp = p.q + (s.q0 + i) * p.q_token + head * p.q_head + lane * N;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float a, dummy;
        unpack16(qp[j], p.bf16, a, dummy);
        q[j] = a * p.scale_log2;
        acc[j] = 0.f;
    }
    const uint32_t ps = 1u << p.c.page_shift;
    for (int t = seen.x; t < seen.y; ++t) {
        const uint8_t* blk = cache_block(p.c, page_of(p, b, t >> p.c.page_shift), head / p.shared);
        const uint32_t row = (uint32_t)t & (ps - 1);
        float val[2][N];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            const uint8_t* cp = blk + kv * ps * F::CODE + row * F::CODE + lane * N / 2;
            const uint32_t word = N == 4 ? (uint32_t)*reinterpret_cast<const uint16_t*>(cp) : (uint32_t)*cp;
            const __half2 pr = *reinterpret_cast<const __half2*>(blk + 2 * ps * F::CODE + kv * ps * F::PAIR +
                                                                 row * F::PAIR + (lane * N / G) * 4);
#pragma unroll
            for (int j = 0; j < N; ++j) val[kv][j] = cached_value(word, j, __low2float(pr), __high2float(pr));
        }
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) dot = fmaf(q[j], val[0][j], dot);
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        const float m = fmaxf(top, dot), keep = exp2f(top - m), e = exp2f(dot - m);
        top = m;
        sum = fmaf(sum, keep, e);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = fmaf(acc[j], keep, e * val[1][j]);
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    uint32_t* o = reinterpret_cast<uint32_t*>(p.out + ((s.q0 + i) * heads + head) * D + lane * N);
#pragma unroll
    for (int j = 0; j < N; j += 2) o[j / 2] = pack16(acc[j] * inv, acc[j + 1] * inv, p.bf16);
    if (p.lse && lane == 0)
        p.lse[(s.q0 + i) * heads + head] = sum > 0.f || sum != sum ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace w4a16
