// Device side of the quantised attention (attention.hip): what every kernel of it shares, and the row that is right for any int32 operand.
#pragma once
#include <hip/hip_runtime.h>

#include "exp_table.hpp"

namespace atlas_attn {

__device__ __constant__ const atlas::ExpTable g_exp = atlas::make_exp_table();

constexpr int SCALE = 14, ONE = 1 << SCALE;

struct Rows { int32_t* d; int64_t ts, hs; };

// Where the keys and values are: rows of a packed prompt (table == nullptr), or blocks of a paged cache
struct Args {
    Rows q, out, k, v;
    const void *ck, *cv;            // the cache: [block][kv head][place][dim]
    const int32_t *cu, *lens, *table;
    int64_t table_stride;
    uint32_t n_blocks, log_block, max_keys;
    uint32_t n_seqs, n_tokens, H, KV, G, d;
    int32_t mul, causal;
    // asked whether the graph's masked keys would weigh: their score (the graph's fill), the graph's tokens, where to tell (nullptr: not asked)
    int32_t fill;
    uint32_t graph_tokens;
    uint32_t* status;
};

struct Seq { uint32_t begin, n_new, keys, idx; };      // its first row of q, its new tokens, its keys

// the sequence's extent from the device's offsets: whatever they hold, the rows stay below n_tokens and the keys below the capacity
__device__ inline Seq seq_at(const Args& A, uint32_t s) {
    const uint32_t b = min((uint32_t)max(A.cu[s], 0), A.n_tokens), e = min((uint32_t)max(A.cu[s + 1], 0), A.n_tokens);
    Seq q{b, e > b ? e - b : 0, 0, s};
    q.keys = A.table ? min((uint32_t)max(A.lens[s], 0), A.max_keys) : q.n_new;
    return q;
}
// the keys that the i-th new token sees: [0, limit)
__device__ inline uint32_t key_limit(const Args& A, const Seq& s, uint32_t i) {
    if (!A.causal) return s.keys;
    const int64_t l = (int64_t)s.keys - s.n_new + i + 1;
    return l < 0 ? 0 : (uint32_t)l;
}
// the block that holds key j, or -1 where there is none
__device__ inline int64_t block_of(const Args& A, const Seq& s, uint32_t j) {
    const int32_t b = A.table[(int64_t)s.idx * A.table_stride + (j >> A.log_block)];
    return (uint32_t)b < A.n_blocks ? b : -1;
}
__device__ inline int64_t cache_at(const Args& A, int64_t block, uint32_t kvh, uint32_t j) {
    return (((block * A.KV + kvh) << A.log_block) + (j & ((1u << A.log_block) - 1))) * A.d;
}
__device__ inline int32_t clamp32(int64_t x) { return (int32_t)(x > 2147483647ll ? 2147483647ll : x < -2147483648ll ? -2147483648ll : x); }
__device__ inline int32_t exp_q(uint32_t z, const int32_t* hi, const int32_t* lo) {
    z = min(z, (uint32_t)atlas::ExpTable::Z_MAX);
    return (int32_t)(__umul24((uint32_t)hi[z >> atlas::ExpTable::LOG_BASE], (uint32_t)lo[z & (atlas::ExpTable::BASE - 1)]) >> SCALE);      // <= 2^28
}
// The same from tables in LDS that are shifted up by 9: the upper half of one 24-bit product is (hi lo) >> 14
template <uint32_t NT>
__device__ inline void load_exp(uint32_t* s_hi, uint32_t* s_lo) {
    for (uint32_t i = threadIdx.x; i < 512; i += NT) { s_hi[i] = (uint32_t)g_exp.hi[i] << 9; s_lo[i] = (uint32_t)g_exp.lo[i] << 9; }
}
__device__ inline uint32_t exp_lds(uint32_t z, const uint32_t* s_hi, const uint32_t* s_lo) {
    z = min(z, (uint32_t)atlas::ExpTable::Z_MAX);
    return (uint32_t)(((uint64_t)(s_hi[z >> atlas::ExpTable::LOG_BASE] & 0xffffff) * (s_lo[z & (atlas::ExpTable::BASE - 1)] & 0xffffff)) >> 32);
}
// sums of e saturate: from 2^28 + 1 on the reciprocal floor(2^28 / sum) is 0 whatever the sum
__device__ inline uint32_t add_sat(uint32_t a, uint32_t b) { const uint32_t s = a + b; return s < a ? 0xffffffffu : s; }

// Row i of a sequence, whose maximum is m: in a graph of graph_tokens tokens the keys behind it are there, with the fill as their score.  They carry no weight, as
// here, where their e is 0 and the fill is not the maximum itself; otherwise the graph's row may be another.
__device__ inline bool mask_weighs(const Args& A, const Seq& s, uint32_t i, int32_t m) {
    if ((int64_t)s.keys - s.n_new + i + 1 >= A.graph_tokens) return false;
    return A.fill > m || exp_q((uint32_t)m - (uint32_t)A.fill, g_exp.hi, g_exp.lo) > 0;
}

// ---- any operands: a workgroup takes one (token, head), 64-bit products one by one, the scores recomputed in each of the three passes.
// The softmax's floors are taken under the FINAL maximum and sum, so partial results cannot be rescaled as a float softmax's are: a pass for the
// maximum, one for the sum, one for the product.
template <class CT>
__device__ inline int32_t score_exact(const Args& A, const Seq& s, uint32_t kvh, const int32_t* q, uint32_t j, bool& there) {
    uint64_t acc = 0;
    there = true;
    if (A.table) {
        const int64_t b = block_of(A, s, j);
        there = b >= 0;
        if (!there) return 0;
        const CT* k = (const CT*)A.ck + cache_at(A, b, kvh, j);
        for (uint32_t i = 0; i < A.d; i++) acc += (uint64_t)((int64_t)q[i] * (int64_t)k[i]);
    } else {
        const int32_t* k = A.k.d + (int64_t)(s.begin + j) * A.k.ts + (int64_t)kvh * A.k.hs;
        for (uint32_t i = 0; i < A.d; i++) acc += (uint64_t)((int64_t)q[i] * (int64_t)k[i]);
    }
    const int32_t x = clamp32((int64_t)acc >> SCALE);
    return clamp32(((int64_t)x * A.mul) >> SCALE);
}

template <class CT, uint32_t NT = 256>
__device__ void row_exact(const Args& A, const Seq& s, uint32_t i, uint32_t h, int32_t* s_q, int32_t* s_p, uint64_t* s_red) {
    const uint32_t tid = threadIdx.x, kvh = h / A.G, limit = min(key_limit(A, s, i), s.keys);
    const int32_t* q = A.q.d + (int64_t)(s.begin + i) * A.q.ts + (int64_t)h * A.q.hs;
    for (uint32_t t = tid; t < A.d; t += NT) s_q[t] = q[t];
    __syncthreads();
    int64_t m = INT64_MIN;
    for (uint32_t j = tid; j < limit; j += NT) { bool there; const int32_t x = score_exact<CT>(A, s, kvh, s_q, j, there); if (there && x > m) m = x; }
    s_red[tid] = (uint64_t)m;
    __syncthreads();
    for (uint32_t w = NT / 2; w > 0; w >>= 1) { if (tid < w) s_red[tid] = (uint64_t)max((int64_t)s_red[tid], (int64_t)s_red[tid + w]); __syncthreads(); }
    m = (int64_t)s_red[0];
    __syncthreads();
    uint64_t part = 0;
    for (uint32_t j = tid; j < limit; j += NT) { bool there; const int32_t x = score_exact<CT>(A, s, kvh, s_q, j, there); if (there) part += exp_q((uint32_t)(m - x), g_exp.hi, g_exp.lo); }
    s_red[tid] = part;
    __syncthreads();
    for (uint32_t w = NT / 2; w > 0; w >>= 1) { if (tid < w) s_red[tid] += s_red[tid + w]; __syncthreads(); }
    const uint64_t sum = s_red[0];
    __syncthreads();
    const uint32_t inv = sum ? (uint32_t)((1ull << (2 * SCALE)) / sum) : 0;
    if (A.status && tid == 0 && sum && mask_weighs(A, s, i, (int32_t)m)) atomicOr(A.status, (uint32_t)ATLAS_ATTN_MASK_WEIGHS);
    uint64_t acc = 0;
    for (uint32_t j0 = 0; j0 < limit; j0 += NT) {
        const uint32_t j = j0 + tid;
        int32_t p = 0;
        if (j < limit) { bool there; const int32_t x = score_exact<CT>(A, s, kvh, s_q, j, there); if (there) p = (int32_t)(((uint32_t)exp_q((uint32_t)(m - x), g_exp.hi, g_exp.lo) * inv) >> SCALE); }
        s_p[tid] = p;
        __syncthreads();
        if (tid < A.d) {
            const uint32_t n = min(NT, limit - j0);
            for (uint32_t t = 0; t < n; t++) {
                if (!s_p[t]) continue;
                int64_t v;
                if (A.table) v = ((const CT*)A.cv)[cache_at(A, block_of(A, s, j0 + t), kvh, j0 + t) + tid];
                else v = A.v.d[(int64_t)(s.begin + j0 + t) * A.v.ts + (int64_t)kvh * A.v.hs + tid];
                acc += (uint64_t)((int64_t)s_p[t] * v);
            }
        }
        __syncthreads();
    }
    if (tid < A.d) A.out.d[(int64_t)(s.begin + i) * A.out.ts + (int64_t)h * A.out.hs + tid] = clamp32((int64_t)acc >> SCALE);
    __syncthreads();
}

// The largest s below n with base(s) <= x (base increasing, base(0) <= x), by all 64 lanes of a wave: 64 places per dependent load (one binary search
// per workgroup was 3 us of every launch).  Offsets that do not increase give some s below n.
template <class F>
__device__ inline uint32_t last_at_most(uint32_t n, uint64_t x, F base) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, at = lane * step;
        const uint32_t hit = (uint32_t)__popcll(__ballot(at < n && base(lo + at) <= x)), skip = (hit ? hit - 1 : 0) * step;
        lo += skip;
        n = min(step, n - skip);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
// the sequence that token t (uniform over the wave) belongs to, or n_seqs where it lies behind the last one
__device__ inline uint32_t find_seq(const int32_t* cu, uint32_t n_seqs, uint32_t t) {
    return (int64_t)t >= cu[n_seqs] ? n_seqs : last_at_most(n_seqs, t, [&](uint32_t s) { return (uint64_t)max(cu[s], 0); });
}

}  // namespace atlas_attn
