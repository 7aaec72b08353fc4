// Attention over the 4-bit cache in its simplest form, for the calls with many rows.
// Included by cache.cu only.
#pragma once
#include "cache_attention.cuh"

namespace w4a16 {

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
    const int pos = s.len - s.nq + i;
    const int2 seen = make_int2(min(seen_lo(p, pos), s.len), seen_hi(p, pos, s.len));
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
    uint32_t* o = reinterpret_cast<uint32_t*>(p.out + ((int64_t)(s.q0 + i) * heads + head) * D + lane * N);
#pragma unroll
    for (int j = 0; j < N; j += 2) o[j / 2] = pack16(acc[j] * inv, acc[j + 1] * inv, p.bf16);
    if (p.lse && lane == 0)
        p.lse[(int64_t)(s.q0 + i) * heads + head] = sum > 0.f || sum != sum ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace w4a16
