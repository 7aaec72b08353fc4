// What the attention kernels over the 4-bit key/value cache share.  Included by cache.cu only.
//
// Query i of the T of a sequence of L cached tokens sits at position p = L - T + i and sees
// the tokens t of [lo, hi): hi = min(p + 1, L) if causal, else L; lo = max(0, p + 1 - window)
// with a window, else 0.  With K_t = s_t c_t + m_t (codes c_t),
//     out = sum_t w_t V_t / sum_t w_t,   w_t = exp(scale q.K_t - max)
// and zeros where nothing is seen.  The query heads that share a key head are rows of one
// problem: row r of a sequence is query r / shared, head r % shared of the key head's.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "cache_format.cuh"
#include "cache_partition.h"
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
    int32_t row_blocks;          // decode kernel: blocks of rows of the sequence with most queries
    bool causal, bf16;
    char* workspace;
};

constexpr float kLn2 = 0.6931471805599453f;

// One sequence's queries and cached tokens, clamped to what the arrays hold.
struct SeqSpan {
    int32_t q0;      // first query's token
    int32_t nq;      // queries that are answered: at most max_q
    int32_t len;     // cached tokens
    int32_t pos0;    // first query's position: by all of the sequence's queries, answered or not
};

__device__ __forceinline__ SeqSpan seq_span(const AttentionParams& p, int b) {
    SeqSpan s;
    const int64_t most = (int64_t)p.table_pages << p.c.page_shift;
    s.len = (int32_t)min((int64_t)max(__ldg(p.seq_lens + b), 0), most);
    if (p.cu_q) {
        const int64_t a = min((int64_t)max(__ldg(p.cu_q + b), 0), p.q_tokens);
        const int64_t e = min((int64_t)max(__ldg(p.cu_q + b + 1), 0), p.q_tokens);
        s.q0 = (int32_t)a;
        const int32_t all = (int32_t)max(e - a, (int64_t)0);
        s.nq = min(all, p.max_q);
        s.pos0 = s.len - all;
    } else {
        s.q0 = b;
        s.nq = b < p.q_tokens ? 1 : 0;
        s.pos0 = s.len - s.nq;
    }
    return s;
}

// Zeros, and -inf in lse, for the rows of tokens [from, to); every worker takes some of them.
template <int D>
__device__ __forceinline__ void clear_rows(const AttentionParams& p, int64_t from, int64_t to, int64_t worker, int64_t workers) {
    const int heads = p.c.kv_heads * p.shared;
    uint4* const end = reinterpret_cast<uint4*>(p.out + to * heads * D);
#pragma unroll 1
    for (uint4* o = reinterpret_cast<uint4*>(p.out + from * heads * D) + worker; o < end; o += workers) *o = make_uint4(0, 0, 0, 0);
    if (p.lse) {
        float* const lse_end = p.lse + to * heads;
#pragma unroll 1
        for (float* l = p.lse + from * heads + worker; l < lse_end; l += workers) *l = -INFINITY;
    }
}

// Rows that belong to no sequence: before the first one's queries and after the last one's, as in a call
// of fixed size that serves fewer queries.
template <int D>
__device__ __forceinline__ void clear_outside(const AttentionParams& p, int64_t worker, int64_t workers) {
    int64_t first = 0, last = p.batch;
    if (p.cu_q) {
        first = min((int64_t)max(__ldg(p.cu_q), 0), p.q_tokens);
        last = max(__ldg(p.cu_q + p.batch), 0);
    }
    if (first > 0) clear_rows<D>(p, 0, first, worker, workers);
    if (last < p.q_tokens) clear_rows<D>(p, last, p.q_tokens, worker, workers);
}

// Queries of a sequence past the max_q that are answered.
template <int D>
__device__ __forceinline__ void clear_past_max(const AttentionParams& p, const SeqSpan& s, int worker, int workers) {
    const int all = s.len - s.pos0;
    if (all > s.nq) clear_rows<D>(p, (int64_t)s.q0 + s.nq, (int64_t)s.q0 + all, worker, workers);
}

// The tokens [lo, hi) that a query at position pos sees.
__device__ __forceinline__ int seen_hi(const AttentionParams& p, int pos, int len) {
    return p.causal ? min(max(pos + 1, 0), len) : len;
}
__device__ __forceinline__ int seen_lo(const AttentionParams& p, int pos) {
    return seen_from(p.window, pos);
}

// A page of a sequence; what the table should not hold is led back into the cache.
__device__ __forceinline__ int64_t page_of(const AttentionParams& p, int b, int index) {
    const int64_t page = __ldg(p.table + b * p.table_stride + index);
    return min(max(page, (int64_t)0), p.c.num_pages - 1);
}

// Untiled bulk copy into this CTA's shared memory (16-byte aligned addresses and size).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// 2^x; tiny results flush to zero.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace w4a16
