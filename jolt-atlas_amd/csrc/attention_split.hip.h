// The quantised attention of few query rows (decoding): bound by reading the cache once.  Up to 16 rows (the heads that share a kv head, times the new tokens) are the
// columns of v_mfma_i32_16x16x64_i8.  Keys go from memory into the fragments' own lanes (16 dims of one key: 64 contiguous bytes) and are cut into digits in
// registers, values the same with 4 dims of 16 keys per lane; nothing passes through LDS.
//
// Short contexts take one launch (k_attn_fused).  Longer ones five: k_split_plan lays the keys of all row tiles and kv heads behind each other in units of 256 and
// k_split_scores, k_split_sums and k_split_values give each of WGS workgroups the same share of that line, wherever sequences begin and end; k_split_join adds the
// shares of a row up.  Splitting costs nothing in exactness: maxima and integer sums do not depend on the order.
//
// Measured: 64 sequences of up to 8191 int32 keys, one token each, 32 heads of 128 over 8 (1.19 GB): 370 us, 3.2 TB/s (a copy: 4.8) — scores 161, sums 17, values 175, join 10, plan 5; the two
// that read the cache run at 3.7 and 3.4 TB/s, near what reading alone reaches (a torch reduction over 600 MB: 3.85; the vector unit is at work for 29 % of their cycles, the matrix
// cores for 3-6).  4 sequences of up to 65000 int16 keys, 32 heads over 4 (187 MB): 115 us — 45, 11, 40, 14, 5; one sequence of 1000 keys, 16 heads of 64 (fused, 16 workgroups): 28 us, of which 13 are fixed (a cold instruction cache, two barriers' worth of latency) and 8 go
// by 512 keys.
#pragma once
#include <algorithm>

#include "attention_tile.hip.h"

namespace atlas_attn {

struct Split {
    uint32_t *units, *rows;      // [tile]: units of 256 keys, rows, of one kv head before this tile; one entry more
    int32_t* scores;             // [row][pitch], rows in the line's order; GONE where no key counts
    int32_t* cmax;               // [part]: a share's rows follow each other at part_at()
    uint32_t* csum;              // [part]
    int64_t* part;               // [part][d]
    uint32_t *q_mag, *k_mag, *v_mag;      // [workgroup + stretch]
    uint32_t n_tiles, n_rows;
    int64_t pitch;
};
constexpr int32_t GONE = INT32_MIN;       // no score of this path reaches it: |score| < 2^30 (SPLIT_BITS)
constexpr uint32_t SPLIT_BITS = 44, UNIT = 256, WGS = 1024, TILE_ROWS = 16;

// Four elements of a row from i on, without a branch around the load: places behind the row's end get elements of the row again (they meet zeros of the
// query, or outputs that nobody stores).  FAST: head_dim is a multiple of 4, one vector load
template <bool FAST, class T>
__device__ inline void fetch4(const T* row, uint32_t i, uint32_t d, int32_t (&o)[4]) {
    if constexpr (FAST) {
        i = min(i, d - 4);
        if constexpr (sizeof(T) == 4) { const i32x4 a = *(const i32x4*)(row + i); o[0] = a[0]; o[1] = a[1]; o[2] = a[2]; o[3] = a[3]; }
        else { const i16x4 a = *(const i16x4*)(row + i); o[0] = a[0]; o[1] = a[1]; o[2] = a[2]; o[3] = a[3]; }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) o[e] = row[min(i + e, d - 1)];
    }
}

// the rows of a workgroup: 16 (token, head of the group) pairs of one sequence
struct RowTile { Seq s; uint32_t row0, n_rows, kvh; bool any; };
__device__ inline RowTile row_tile(const Args& A, uint32_t tile, uint32_t kvh) {
    RowTile t;
    t.kvh = kvh;
    auto base = [&](uint32_t s) { return (uint64_t)min((uint32_t)max(A.cu[s], 0), A.n_tokens) * A.G / TILE_ROWS + s; };
    const uint32_t si = last_at_most(A.n_seqs, tile, base);
    t.s = seq_at(A, si);
    t.n_rows = t.s.n_new * A.G;
    const uint64_t b = base(si);
    const uint64_t first = tile >= b ? (tile - b) * TILE_ROWS : ~0ull;
    t.any = first < t.n_rows;
    t.row0 = (uint32_t)first;
    return t;
}

// ---- what the split and the fused kernels share; g = lane / 16, l = lane % 16 throughout: a lane has query row l.
// FAST: head_dim is a multiple of 4 and 16 keys from a multiple of 16 on lie behind each other (prompts; blocks of 16 or more): one scalar look-up for them
template <int KS>
struct Query { v4i q0[KS], q1[KS], q2[KS]; Range range; };
template <int KS, bool FAST>
__device__ inline void load_query(const Args& A, const RowTile& R, uint32_t r, bool mine, uint32_t g, Query<KS>& Q) {
    const int32_t* q = A.q.d + (int64_t)(R.s.begin + (mine ? r / A.G : 0)) * A.q.ts + (int64_t)(R.kvh * A.G + (mine ? r % A.G : 0)) * A.q.hs;
    int32_t e[KS][4][4];
#pragma unroll
    for (int f = 0; f < KS; f++)
#pragma unroll
        for (int x = 0; x < 4; x++) fetch4<FAST>(q, f * 64 + g * 16 + x * 4, A.d, e[f][x]);
#pragma unroll
    for (int f = 0; f < KS; f++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const uint32_t i = f * 64 + g * 16 + x * 4;
#pragma unroll
            for (uint32_t y = 0; y < 4; y++) e[f][x][y] = mine && i + y < A.d ? e[f][x][y] : 0;
            int a, b, d;
            digits4(e[f][x][0], e[f][x][1], e[f][x][2], e[f][x][3], a, b, d, Q.range);
            Q.q0[f][x] = a; Q.q1[f][x] = b; Q.q2[f][x] = d;
        }
}
// the page table's entry for key j as a scalar load (j is uniform over the wave), -1 for a block that does not exist; prompts have no table: 0
__device__ inline int32_t look_up(const Args& A, const RowTile& R, uint32_t j) {
    if (!A.table) return 0;
    const auto* t = (const __attribute__((address_space(4))) int32_t*)(A.table + (int64_t)R.s.idx * A.table_stride);
    const int32_t b = t[__builtin_amdgcn_readfirstlane(j >> A.log_block)];
    return (uint32_t)b < A.n_blocks ? b : -1;
}
// where key j's row begins, its block being known; a block that does not exist: block 0, whose scores and weights do not count
template <class CT, bool VALUE>
__device__ inline const CT* key_row(const Args& A, const RowTile& R, uint32_t j, int64_t block) {
    if (A.table) return (const CT*)(VALUE ? A.cv : A.ck) + cache_at(A, max(block, (int64_t)0), R.kvh, j);
    const Rows& x = VALUE ? A.v : A.k;
    return (const CT*)x.d + (int64_t)(R.s.begin + j) * x.ts + (int64_t)R.kvh * x.hs;
}
// 16 keys from j (a multiple of 16, below k1) as they come from memory: lane l has key j + l, dims 16 g + .. of each step; in: which of them count
template <class CT, int KS, bool FAST>
struct Keys16 {
    int32_t e[KS][4][4];
    uint32_t in;
    __device__ void fetch(const Args& A, const RowTile& R, uint32_t j, int32_t block, uint32_t k1, uint32_t g, uint32_t l) {
        const uint32_t n = min(k1 - j, 16u), o = min(l, n - 1);                 // behind the end: the last key again
        const CT* row;
        if constexpr (FAST) {
            row = key_row<CT, false>(A, R, j, block) + (int64_t)o * (A.table ? (int64_t)A.d : A.k.ts);
            in = block >= 0 ? (1u << n) - 1 : 0;
        } else {
            const int64_t b = A.table ? block_of(A, R.s, j + o) : 0;
            row = key_row<CT, false>(A, R, j + o, b);
            in = (uint32_t)__ballot(b >= 0 && l < n) & 0xffff;
        }
#pragma unroll
        for (int f = 0; f < KS; f++)
#pragma unroll
            for (int y = 0; y < 4; y++) fetch4<FAST>(row, f * 64 + g * 16 + y * 4, A.d, e[f][y]);
    }
    // the scores of keys j + 4 g + i against row l, GONE where one does not count
    __device__ v4i scores(const Args& A, const Query<KS>& Q, uint32_t j, uint32_t limit, uint32_t g, Range& range) const {
        v4i a0 = {}, a1 = {}, a2 = {}, a3 = {}, a4 = {};
#pragma unroll
        for (int f = 0; f < KS; f++) {
            v4i p0, p1, p2;
#pragma unroll
            for (int y = 0; y < 4; y++) {
                int a, b, d;
                digits4(e[f][y][0], e[f][y][1], e[f][y][2], e[f][y][3], a, b, d, range);
                p0[y] = a; p1[y] = b; p2[y] = d;
            }
            a4 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, Q.q2[f], a4, 0, 0, 0);
            a3 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, Q.q1[f], a3, 0, 0, 0);
            a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, Q.q0[f], a2, 0, 0, 0);
            a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, Q.q0[f], a1, 0, 0, 0);
            a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, Q.q0[f], a0, 0, 0, 0);
            a3 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, Q.q2[f], a3, 0, 0, 0);
            a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, Q.q1[f], a2, 0, 0, 0);
            a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, Q.q1[f], a1, 0, 0, 0);
            a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, Q.q2[f], a2, 0, 0, 0);
        }
        const uint32_t see = limit > j ? min(limit - j, 16u) : 0, mask = (in & ((1u << see) - 1)) >> (4 * g);
        v4i x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int32_t v = rescale(combine<KS == 4>(a0[i], a1[i], a2[i], a3[i], a4[i]), A.mul);       // 2^14: the same score
            const int32_t keep = (int32_t)(mask << (31 - i)) >> 31;                                       // no branch
            x[i] = (v & keep) | (GONE & ~keep);
        }
        return x;
    }
};
// Every 16 keys of a wave's 64 at a time (64 of every `stride` from j0 on, below k1): the next ones are on their way while the scores of these are taken, the
// page of those behind them is being looked up.  take(j, x)
template <class CT, int KS, bool FAST, class F>
__device__ inline void each_score(const Args& A, const RowTile& R, const Query<KS>& Q, uint32_t j0, uint32_t stride, uint32_t k1, uint32_t limit, uint32_t g, uint32_t l, Range& range, F take) {
    auto next = [&](uint32_t j) { return (j & 63) == 48 ? j + 16 + stride - 64 : j + 16; };
    auto look = [&](uint32_t j) { return FAST ? look_up(A, R, min(j, k1 - 1)) : 0; };
    Keys16<CT, KS, FAST> a, b;
    uint32_t j = j0;
    if (j >= k1) return;
    int32_t page = look(j);
    a.fetch(A, R, j, page, k1, g, l);
    page = look(next(j));
#pragma unroll 1
    for (;;) {
        const uint32_t j1 = next(j);
        if (j1 < k1) b.fetch(A, R, j1, page, k1, g, l);
        page = look(next(j1));
        take(j, a.scores(A, Q, j, limit, g, range));
        if (j1 >= k1) break;
        j = next(j1);
        if (j < k1) a.fetch(A, R, j, page, k1, g, l);
        page = look(next(j));
        take(j1, b.scores(A, Q, j1, limit, g, range));
        if (j >= k1) break;
    }
}
// four weights 0 .. 2^14 as signed bytes: p = (signed byte) p + 2^8 ((p + 128) >> 8)
__device__ inline void weight_bytes(const uint32_t (&p)[4], int& lo, int& hi) {
    const uint32_t a = p[0] | (p[1] << 16), b = p[2] | (p[3] << 16);
    lo = (int)__builtin_amdgcn_perm(b, a, 0x06040200u);
    hi = (int)__builtin_amdgcn_perm(b + 0x00800080u, a + 0x00800080u, 0x07050301u);
}
// The sums with the values' digits 0, 1, 2: o[4 f + e], dims 64 (f0 + f) + 4 (4 g + i) + e of row l.  At most 128 dims at a time (VS = 2): the sums of 256 would take
// 192 registers, and where it then spills hipcc 7.2 copies a matrix instruction's result two instructions behind it, without the wait (seen in the assembly, and
// as wrong sums).
constexpr int value_steps(int ks) { return ks < 2 ? ks : 2; }
template <int VS>
struct Product { v4i o0[VS * 4] = {}, o1[VS * 4] = {}, o2[VS * 4] = {}; };
// The products of 64 weights and values at a time (64 keys of every `stride` from j0 on, below k1): byte 4 t + i of lane group g is key 16 t + 4 g + i, a lane loads
// 4 dims of each of its 16 keys.  The values of the next step are on their way from when a half's digits are taken.  weights(j, w0, w1): the weights' bytes
template <class CT, int VS, bool FAST, class F>
__device__ inline void each_product(const Args& A, const RowTile& R, int f0, uint32_t j0, uint32_t stride, uint32_t k1, uint32_t g, uint32_t l, Product<VS>& P, Range& range, F weights) {
    if (j0 >= k1) return;
    int32_t v[4][4][4];
    int32_t page[4];
    const int64_t step = A.table ? (int64_t)A.d : A.v.ts;
    const uint32_t last = (k1 - 1) & ~15u;
    auto look = [&](uint32_t j) {
        if constexpr (FAST)
#pragma unroll
            for (int t = 0; t < 4; t++) page[t] = look_up(A, R, min(j + 16 * t, last));
    };
    // behind the end, and in blocks that do not exist: any values, their weights are 0
    auto load = [&](uint32_t j, int f, int half) {
#pragma unroll
        for (int t = 2 * half; t < 2 * half + 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (FAST) {
                    const uint32_t jt = min(j + 16 * t, last);
                    fetch4<true>(key_row<CT, true>(A, R, jt, page[t]) + (int64_t)min(4 * g + i, k1 - 1 - jt) * step, (f0 + f) * 64 + l * 4, A.d, v[t][i]);
                } else {
                    const uint32_t jt = min(j + 16 * t + 4 * g + i, k1 - 1);
                    fetch4<false>(key_row<CT, true>(A, R, jt, A.table ? block_of(A, R.s, jt) : 0), (f0 + f) * 64 + l * 4, A.d, v[t][i]);
                }
            }
    };
    look(j0);
    load(j0, 0, 0);
    load(j0, 0, 1);
#pragma unroll 1
    for (uint32_t j = j0; j < k1; j += stride) {
        v4i w0, w1;
        weights(j, w0, w1);
        const bool second = __any((w1[0] | w1[1] | w1[2] | w1[3]) != 0);
#pragma unroll
        for (int f = 0; f < VS; f++) {
            v4i p[4][3];
            if (f + 1 == VS) look(min(j + stride, last));
#pragma unroll
            for (int half = 0; half < 2; half++) {
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int t = 2 * half; t < 2 * half + 2; t++) {
                        int a, b, d;
                        digits4(v[t][0][e], v[t][1][e], v[t][2][e], v[t][3][e], a, b, d, range);
                        p[e][0][t] = a; p[e][1][t] = b; p[e][2][t] = d;
                    }
                if (f + 1 < VS) load(j, f + 1, half);
                else if (j + stride < k1) load(j + stride, 0, half);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int x = f * 4 + e;
                P.o0[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[e][0], w0, P.o0[x], 0, 0, 0);
                P.o1[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[e][1], w0, P.o1[x], 0, 0, 0);
                P.o2[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[e][2], w0, P.o2[x], 0, 0, 0);
            }
            if (second) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int x = f * 4 + e;
                    P.o0[x] += __builtin_amdgcn_mfma_i32_16x16x64_i8(p[e][0], w1, v4i{}, 0, 0, 0) * 256;
                    P.o1[x] += __builtin_amdgcn_mfma_i32_16x16x64_i8(p[e][1], w1, v4i{}, 0, 0, 0) * 256;
                    P.o2[x] += __builtin_amdgcn_mfma_i32_16x16x64_i8(p[e][2], w1, v4i{}, 0, 0, 0) * 256;
                }
            }
        }
    }
}
// adds a wave's products to the workgroup's sums [row][dims]
template <int VS>
__device__ inline void add_product(const Product<VS>& P, int f0, int dims, uint32_t g, uint32_t l, unsigned long long* s_o) {
#pragma unroll
    for (int x = 0; x < VS * 4; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t y = (int64_t)P.o0[x][i] + ((int64_t)P.o1[x][i] << 8) + ((int64_t)P.o2[x][i] << 16);
            atomicAdd(&s_o[l * dims + (f0 + x / 4) * 64 + (4 * g + i) * 4 + x % 4], (unsigned long long)y);
        }
}

// ---- everything in one launch where a row's scores fit into LDS (up to FUSED_KEYS keys): 8 waves take 64 keys each in turn, the scores of 16 rows stay in LDS as scores, then
// as e, and the rows' maxima and sums are joined there.  Few launches for short contexts and prompts, one pass over the keys instead of three.
constexpr uint32_t FUSED_WAVES = 8;
inline size_t fused_keys(size_t d) { return d > 128 ? 1024 : 2048; }
inline size_t fused_pitch(size_t max_keys) { return (max_keys + 63) / 64 * 64 + 4; }
// the scores of 16 rows and behind them the products' sums; row_exact needs 8 KB
inline size_t fused_lds(size_t max_keys, size_t steps) { return std::max<size_t>(TILE_ROWS * fused_pitch(max_keys) * 4 + (steps > 2 ? TILE_ROWS * steps * 512 : 0), std::max<size_t>(8192, TILE_ROWS * steps * 512)); }

template <class CT, int KS, bool FAST>
__global__ __launch_bounds__(FUSED_WAVES * 64, 2) void k_attn_fused(Args A, uint32_t pitch) {
    constexpr int D = KS * 64;
    extern __shared__ __align__(16) int32_t s_x[];                 // [16][pitch] scores; the sums of the products afterwards
    __shared__ uint32_t s_hi[512], s_lo[512];
    __shared__ int32_t s_m[FUSED_WAVES][16];
    __shared__ uint32_t s_s[FUSED_WAVES][16], s_mag[3];
    const RowTile R = row_tile(A, blockIdx.x / A.KV, blockIdx.x % A.KV);
    if (!R.any) return;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, l = lane & 15;
    const uint32_t r = R.row0 + l, rows = min(TILE_ROWS, R.n_rows - R.row0);
    const bool mine = r < R.n_rows;
    const uint32_t limit = mine ? min(key_limit(A, R.s, r / A.G), R.s.keys) : 0;
    const uint32_t k1 = min(key_limit(A, R.s, (R.row0 + rows - 1) / A.G), R.s.keys);      // the most that a row of the tile sees
    load_exp<FUSED_WAVES * 64>(s_hi, s_lo);
    if (tid < 3) s_mag[tid] = 0;
    __syncthreads();
    Range rk;
    int32_t m = GONE;
    if (wave * 64 < k1) {
        Query<KS> Q;
        load_query<KS, FAST>(A, R, r, mine, g, Q);
        each_score<CT, KS, FAST>(A, R, Q, wave * 64, FUSED_WAVES * 64, k1, limit, g, l, rk, [&](uint32_t j, v4i x) {
            *(v4i*)(s_x + l * pitch + j + 4 * g) = x;
            m = max(max(m, max(x[0], x[1])), max(x[2], x[3]));
        });
        for (uint32_t j = (k1 + 15) & ~15u; j & 63; j += 16)                    // up to the next multiple of 64: no keys
            if (wave == j / 64 % FUSED_WAVES) *(v4i*)(s_x + l * pitch + j + 4 * g) = v4i{GONE, GONE, GONE, GONE};
        atomicOr(&s_mag[0], Q.range.word());
        atomicOr(&s_mag[1], rk.word());
    }
    m = max(m, __shfl_xor(m, 16));
    m = max(m, __shfl_xor(m, 32));
    if (g == 0) s_m[wave][l] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < FUSED_WAVES; w++) m = max(m, s_m[w][l]);
    const bool exact = ((s_mag[0] | s_mag[1]) & WIDE) || bits_of(s_mag[0]) + bits_of(s_mag[1]) + bits_of(A.d - 1) > SPLIT_BITS;
    uint32_t sum = 0;
#pragma unroll 1
    for (uint32_t j0 = wave * 64; j0 < k1; j0 += FUSED_WAVES * 64)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            v4i* at = (v4i*)(s_x + l * pitch + j0 + 16 * t + 4 * g);
            v4i x = *at;
#pragma unroll
            for (int i = 0; i < 4; i++) { x[i] = (int)exp_lds((uint32_t)m - (uint32_t)x[i], s_hi, s_lo); sum += (uint32_t)x[i]; }      // GONE lies 2^30 below: 0
            *at = x;
        }
    sum += (uint32_t)__shfl_xor((int)sum, 16);
    sum += (uint32_t)__shfl_xor((int)sum, 32);
    if (g == 0) s_s[wave][l] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < FUSED_WAVES; w++) sum += s_s[w][l];       // <= 2^25
    const uint32_t inv = m == GONE ? 0 : (1u << (2 * SCALE)) / sum;       // a row that sees no key: no weights
    if (A.status && wave == 0 && g == 0 && mine && !exact && m != GONE && mask_weighs(A, R.s, r / A.G, m)) atomicOr(A.status, (uint32_t)ATLAS_ATTN_MASK_WEIGHS);
    // up to 128 dims the sums take the scores' place; more dims are two sweeps over the weights, their sums lie behind the scores
    constexpr int VS = value_steps(KS);
    unsigned long long* s_o = (unsigned long long*)(s_x + (KS > 2 ? TILE_ROWS * pitch : 0));
    if (KS > 2) for (uint32_t i = tid; i < rows * D; i += FUSED_WAVES * 64) s_o[i] = 0;
    if (KS > 2) __syncthreads();
    Range rv;
#pragma unroll 1
    for (int f0 = 0; f0 < KS; f0 += VS) {
        Product<VS> P;
        if (!exact)
            each_product<CT, VS, FAST>(A, R, f0, wave * 64, FUSED_WAVES * 64, k1, g, l, P, rv, [&](uint32_t j, v4i& w0, v4i& w1) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const v4i e = *(const v4i*)(s_x + l * pitch + j + 16 * t + 4 * g);
                    uint32_t p[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) p[i] = __umul24((uint32_t)e[i], inv) >> SCALE;
                    int a, b;
                    weight_bytes(p, a, b);
                    w0[t] = a; w1[t] = b;
                }
            });
        if (KS <= 2) {
            __syncthreads();                                        // the weights have been read
            for (uint32_t i = tid; i < rows * D; i += FUSED_WAVES * 64) s_o[i] = 0;
            __syncthreads();
        }
        if (mine && wave * 64 < k1) add_product<VS>(P, f0, D, g, l, s_o);
    }
    atomicOr(&s_mag[2], rv.word());
    __syncthreads();
    if (exact || (s_mag[2] & WIDE)) {
        for (uint32_t x = 0; x < rows; x++)
            row_exact<CT, FUSED_WAVES * 64>(A, R.s, (R.row0 + x) / A.G, R.kvh * A.G + (R.row0 + x) % A.G, s_x, s_x + 512, (uint64_t*)(s_x + 1024));
        return;
    }
    for (uint32_t i = tid; i < rows * D; i += FUSED_WAVES * 64) {
        const uint32_t x = R.row0 + i / D, y = i % D;
        if (y < A.d) A.out.d[(int64_t)(R.s.begin + x / A.G) * A.out.ts + (int64_t)(R.kvh * A.G + x % A.G) * A.out.hs + y] = (int32_t)((int64_t)s_o[i] >> SCALE);
    }
}

// ---- longer contexts
// One workgroup: the prefix sums of the tiles' units and rows.  Offsets that do not ascend would count rows twice, more than the workspace has room for: then
// there are none.
__global__ __launch_bounds__(1024) void k_split_plan(Args A, Split S) {
    __shared__ uint32_t s_u[16], s_r[16], s_bad;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    for (uint32_t i = tid; i < A.n_seqs; i += 1024) if (A.cu[i] < 0 || A.cu[i + 1] < A.cu[i] || A.cu[i + 1] > (int64_t)A.n_tokens) s_bad = 1;
    __syncthreads();
    const bool bad = s_bad;
    uint32_t u0 = 0, r0 = 0;
    for (uint32_t i0 = 0; i0 < S.n_tiles; i0 += 1024) {
        const uint32_t i = i0 + tid;
        uint32_t u = 0, r = 0;
        if (i < S.n_tiles) {
            auto base = [&](uint32_t s) { return (uint64_t)min((uint32_t)max(A.cu[s], 0), A.n_tokens) * A.G / TILE_ROWS + s; };
            uint32_t lo = 0, hi = A.n_seqs;                        // every thread has a tile of its own: a binary search each
            while (hi - lo > 1) { const uint32_t mid = (lo + hi) / 2; if (base(mid) <= i) lo = mid; else hi = mid; }
            const Seq s = seq_at(A, lo);
            const uint64_t b = base(lo), first = i >= b ? (i - b) * TILE_ROWS : ~0ull;
            if (!bad && first < (uint64_t)s.n_new * A.G) { r = min(TILE_ROWS, s.n_new * A.G - (uint32_t)first); u = (s.keys + UNIT - 1) / UNIT; }
        }
        const uint32_t u_mine = u, r_mine = r;
#pragma unroll
        for (uint32_t o = 1; o < 64; o <<= 1) { const uint32_t a = __shfl_up(u, o), b = __shfl_up(r, o); if (lane >= o) { u += a; r += b; } }
        if (lane == 63) { s_u[wave] = u; s_r[wave] = r; }
        __syncthreads();
        uint32_t ut = 0, rt = 0;
        for (uint32_t w = 0; w < 16; w++) { if (w < wave) { u += s_u[w]; r += s_r[w]; } ut += s_u[w]; rt += s_r[w]; }
        if (i < S.n_tiles) { S.units[i] = u0 + u - u_mine; S.rows[i] = r0 + r - r_mine; }
        u0 += ut; r0 += rt;
        __syncthreads();
    }
    if (tid == 0) { S.units[S.n_tiles] = u0; S.rows[S.n_tiles] = r0; }
}
// The line's units over the workgroups: n of them have a share, the first `more` of them per + 1 units and the others per.  Half as many where a share would be
// less than 4 units: two workgroups fit a CU (4 tokens over 65000 16-bit keys: the scores 49 -> 45, the values 46 -> 40 us; 64 over up to 8191 int32 ones, which
// have more: the scores 162 -> 172, the sums 17 -> 26 us)
struct Line {
    uint32_t n, per, more;
    __device__ Line(const Args& A, const Split& S) { const uint32_t U = S.units[S.n_tiles] * A.KV; n = max(min(U, U >= 4 * WGS ? WGS : WGS / 2), 1u); per = U / n; more = U % n; }
    __device__ uint32_t begin(uint32_t w) const { return min(w, n) * per + min(w, more); }
    __device__ uint32_t owner(uint32_t u) const { const uint32_t x = more * (per + 1); return u < x ? u / (per + 1) : more + (u - x) / per; }
};
// a stretch of the line: keys [k0, k1) of a row tile under one kv head
struct Stretch {
    RowTile R;
    uint32_t tile, units, k0, k1, part, row, mag, n;      // part: of its first row in cmax, csum, part; row: of its first row in scores; mag: its place in the magnitudes; n: its rows
};
// what workgroup w has from unit u on (u < end, the end of its share)
__device__ inline Stretch stretch_at(const Args& A, const Split& S, uint32_t w, uint32_t u, uint32_t end) {
    Stretch x;
    const uint32_t t = x.tile = last_at_most(S.n_tiles, u, [&](uint32_t i) { return (uint64_t)S.units[i] * A.KV; });
    const uint32_t per = max(S.units[t + 1] - S.units[t], 1u), rel = u - S.units[t] * A.KV, kvh = min(rel / per, A.KV - 1), at = rel % per;
    x.R = row_tile(A, t, kvh);
    x.units = min(per - at, end - u);
    x.k0 = at * UNIT;
    x.k1 = min((at + x.units) * UNIT, x.R.s.keys);
    x.n = S.rows[t + 1] - S.rows[t];
    x.row = S.rows[t] * A.KV + kvh * x.n;
    x.part = w * TILE_ROWS + x.row;          // a next stretch of w lies n further, the same rows' share of w + 1 16 further: no two overlap
    x.mag = w + t * A.KV + kvh;
    return x;
}

template <class CT, int KS, bool FAST>      // KS: steps of 64 dims: 1, 2 or 4
__global__ __launch_bounds__(256, 2) void k_split_scores(Args A, Split S) {
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, l = lane & 15;
    __shared__ int32_t s_max[4][16];
    __shared__ uint32_t s_mag[2];
    const Line line(A, S);
    const uint32_t end = line.begin(blockIdx.x + 1);
#pragma unroll 1
    for (uint32_t u = line.begin(blockIdx.x); u < end;) {
        const Stretch X = stretch_at(A, S, blockIdx.x, u, end);
        const RowTile& R = X.R;
        u += X.units;
        const uint32_t r = R.row0 + l;
        const bool mine = l < X.n;
        const uint32_t limit = mine ? min(key_limit(A, R.s, r / A.G), R.s.keys) : 0;
        if (tid < 2) s_mag[tid] = 0;
        __syncthreads();
        Query<KS> Q;
        load_query<KS, FAST>(A, R, r, mine, g, Q);
        Range rk;
        int32_t m = GONE;
        int32_t* to = S.scores + (int64_t)(X.row + (mine ? l : 0)) * S.pitch + 4 * g;
        each_score<CT, KS, FAST>(A, R, Q, X.k0 + wave * 64, UNIT, X.k1, limit, g, l, rk, [&](uint32_t j, v4i x) {
            if (mine) *(v4i*)(to + j) = x;
            m = max(max(m, max(x[0], x[1])), max(x[2], x[3]));
        });
        for (uint32_t j = (X.k1 + 15) & ~15u; j & 63; j += 16)                      // up to the next multiple of 64: no keys
            if (mine && wave == j / 64 % 4) *(v4i*)(to + j) = v4i{GONE, GONE, GONE, GONE};
        m = max(m, __shfl_xor(m, 16));
        m = max(m, __shfl_xor(m, 32));
        if (g == 0) s_max[wave][l] = m;
        atomicOr(&s_mag[0], Q.range.word());
        atomicOr(&s_mag[1], rk.word());
        __syncthreads();
        if (tid < X.n) S.cmax[X.part + tid] = max(max(s_max[0][l], s_max[1][l]), max(s_max[2][l], s_max[3][l]));
        if (tid == 0) { S.q_mag[X.mag] = s_mag[0]; S.k_mag[X.mag] = s_mag[1]; }
        __syncthreads();
    }
}

// A row's value over the shares of its stretch: `with` over the places of the shares' parts
template <class F>
__device__ inline void each_share(const Args& A, const Split& S, uint32_t t, uint32_t kvh, uint32_t first, uint32_t step, F with) {
    const uint32_t per = S.units[t + 1] - S.units[t], n = S.rows[t + 1] - S.rows[t];
    if (per == 0) return;
    const Line line(A, S);
    const uint32_t p = S.units[t] * A.KV + kvh * per, w1 = line.owner(p + per - 1);
    for (uint32_t w = line.owner(p) + first; w <= w1; w += step) with(w * TILE_ROWS + S.rows[t] * A.KV + kvh * n, w + t * A.KV + kvh);
}

// a wave takes a row of the share at a time, 256 keys by 4 per lane
__global__ __launch_bounds__(256) void k_split_sums(Args A, Split S) {
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    __shared__ uint32_t s_hi[512], s_lo[512];
    load_exp<256>(s_hi, s_lo);
    __syncthreads();
    const Line line(A, S);
    const uint32_t end = line.begin(blockIdx.x + 1);
#pragma unroll 1
    for (uint32_t u = line.begin(blockIdx.x); u < end;) {
        const Stretch X = stretch_at(A, S, blockIdx.x, u, end);
        u += X.units;
        const uint32_t t = X.tile;
        for (uint32_t r = wave; r < X.n; r += 4) {
            int32_t m = GONE;
            each_share(A, S, t, X.R.kvh, lane, 64, [&](uint32_t part, uint32_t) { m = max(m, S.cmax[part + r]); });
            for (int o = 32; o; o >>= 1) m = max(m, __shfl_xor(m, o));
            uint32_t sum = 0;
            for (uint32_t j = X.k0 + lane * 4; j < X.k1; j += 256) {
                const v4i x = *(const v4i*)(S.scores + (int64_t)(X.row + r) * S.pitch + j);      // behind the last key: GONE up to the next multiple of 64
#pragma unroll
                for (int i = 0; i < 4; i++) sum = __builtin_elementwise_add_sat(sum, exp_lds((uint32_t)m - (uint32_t)x[i], s_hi, s_lo));
            }
            for (int o = 32; o; o >>= 1) sum = __builtin_elementwise_add_sat(sum, (uint32_t)__shfl_xor((int)sum, o));
            if (lane == 0) S.csum[X.part + r] = m == GONE ? 0 : sum;
        }
    }
}

template <class CT, int KS, bool FAST>
__global__ __launch_bounds__(256, 2) void k_split_values(Args A, Split S) {
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, l = lane & 15;
    constexpr int D = KS * 64, VS = value_steps(KS);
    __shared__ uint32_t s_hi[512], s_lo[512];
    __shared__ int32_t s_m[16];
    __shared__ uint32_t s_sum[16];
    __shared__ unsigned long long s_o[TILE_ROWS * D];
    __shared__ uint32_t s_mag;
    load_exp<256>(s_hi, s_lo);
    const Line line(A, S);
    const uint32_t end = line.begin(blockIdx.x + 1);
#pragma unroll 1
    for (uint32_t u = line.begin(blockIdx.x); u < end;) {
        const Stretch X = stretch_at(A, S, blockIdx.x, u, end);
        const RowTile& R = X.R;
        u += X.units;
        for (uint32_t i = tid; i < X.n * D; i += 256) s_o[i] = 0;
        if (tid == 0) s_mag = 0;
        // the rows' maxima and sums over all shares: 16 lanes of a row each
        {
            int32_t m = GONE;
            uint32_t sum = 0;
            const uint32_t r = tid >> 4;
            if (r < X.n)
                each_share(A, S, X.tile, R.kvh, tid & 15, 16, [&](uint32_t part, uint32_t) {
                    m = max(m, S.cmax[part + r]);
                    sum = __builtin_elementwise_add_sat(sum, S.csum[part + r]);
                });
            for (int o = 8; o; o >>= 1) { m = max(m, __shfl_xor(m, o)); sum = __builtin_elementwise_add_sat(sum, (uint32_t)__shfl_xor((int)sum, o)); }
            if ((tid & 15) == 0) { s_m[r] = m; s_sum[r] = sum; }
        }
        __syncthreads();
        const bool mine = l < X.n;
        const int32_t m = s_m[l];
        const uint32_t inv = mine && s_sum[l] ? (1u << (2 * SCALE)) / s_sum[l] : 0;
        const int32_t* from = S.scores + (int64_t)(X.row + (mine ? l : 0)) * S.pitch + 4 * g;      // lanes without a row: another's, inv is 0
        Range rv;
#pragma unroll 1
        for (int f0 = 0; f0 < KS; f0 += VS) {
            Product<VS> P;
            each_product<CT, VS, FAST>(A, R, f0, X.k0 + wave * 64, UNIT, X.k1, g, l, P, rv, [&](uint32_t j, v4i& w0, v4i& w1) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const v4i x = *(const v4i*)(from + j + 16 * t);
                    uint32_t p[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) p[i] = __umul24(exp_lds((uint32_t)m - (uint32_t)x[i], s_hi, s_lo), inv) >> SCALE;
                    int a, b;
                    weight_bytes(p, a, b);
                    w0[t] = a; w1[t] = b;
                }
            });
            if (mine) add_product<VS>(P, f0, D, g, l, s_o);
        }
        atomicOr(&s_mag, rv.word());
        __syncthreads();
        for (uint32_t i = tid; i < X.n * D; i += 256) {
            const uint32_t x = i / D, y = i % D;
            if (y < A.d) S.part[(int64_t)(X.part + x) * A.d + y] = (int64_t)s_o[i];
        }
        if (tid == 0) S.v_mag[X.mag] = s_mag;
        __syncthreads();
    }
}

// One workgroup per row: the shares' products added up, every dim by JOIN / DP threads; where the operands did not fit the digits, the row again in 64 bits.
// JOIN: 1024 where the rows are few (128 rows: 40 -> 14 us), 256 where they fill the chip (2048 rows: 12 us, 25 with 1024)
template <class CT, uint32_t JOIN>
__global__ __launch_bounds__(JOIN) void k_split_join(Args A, Split S, uint32_t dp) {
    const uint32_t t = blockIdx.x / A.H, h = blockIdx.x % A.H, tid = threadIdx.x, kvh = h / A.G;
    const uint32_t si = find_seq(A.cu, A.n_seqs, t);
    if (si >= A.n_seqs) return;
    const Seq s = seq_at(A, si);
    if (t < s.begin || t - s.begin >= s.n_new) return;
    const uint32_t row = (t - s.begin) * A.G + h % A.G, tile = (uint32_t)((uint64_t)s.begin * A.G / TILE_ROWS) + si + row / TILE_ROWS, r = row % TILE_ROWS;
    __shared__ uint32_t s_mag[3];
    __shared__ int32_t s_q[JOIN], s_p[JOIN];
    __shared__ uint64_t s_red[JOIN];
    __shared__ int32_t s_m;
    if (tid < 3) s_mag[tid] = 0;
    if (tid == 3) s_m = GONE;
    __syncthreads();
    const uint32_t per = S.units[tile + 1] - S.units[tile], n = S.rows[tile + 1] - S.rows[tile];
    const uint32_t y = tid & (dp - 1), parts = JOIN / dp;
    int64_t sum = 0;
    if (per) {
        const Line line(A, S);
        const uint32_t p = S.units[tile] * A.KV + kvh * per, w0 = line.owner(p), w1 = line.owner(p + per - 1), mag = tile * A.KV + kvh;
        uint32_t mq = 0, mk = 0, mv = 0;
        for (uint32_t w = w0 + tid; w <= w1; w += JOIN) { mq |= S.q_mag[w + mag]; mk |= S.k_mag[w + mag]; mv |= S.v_mag[w + mag]; }
        if (mq | mk | mv) { atomicOr(&s_mag[0], mq); atomicOr(&s_mag[1], mk); atomicOr(&s_mag[2], mv); }
        if (A.status)
            for (uint32_t w = w0 + tid; w <= w1; w += JOIN) atomicMax(&s_m, S.cmax[w * TILE_ROWS + S.rows[tile] * A.KV + kvh * n + r]);
        const int64_t* from = S.part + (int64_t)(S.rows[tile] * A.KV + kvh * n + r) * A.d + y;
        if (y < A.d)
#pragma unroll 4
            for (uint32_t w = w0 + tid / dp; w <= w1; w += parts) sum += from[(int64_t)w * TILE_ROWS * A.d];
    }
    s_red[tid] = (uint64_t)sum;
    __syncthreads();
    const uint32_t mq = s_mag[0], mk = s_mag[1], mv = s_mag[2];
    if (((mq | mk | mv) & WIDE) || bits_of(mq) + bits_of(mk) + bits_of(A.d - 1) > SPLIT_BITS) {
        row_exact<CT, JOIN>(A, s, t - s.begin, h, s_q, s_p, s_red);
        return;
    }
    if (A.status && tid == 0 && s_m != GONE && mask_weighs(A, s, t - s.begin, s_m)) atomicOr(A.status, (uint32_t)ATLAS_ATTN_MASK_WEIGHS);
    if (tid < A.d) {
        for (uint32_t p = 1; p < parts; p++) sum += (int64_t)s_red[p * dp + tid];
        A.out.d[(int64_t)t * A.out.ts + (int64_t)h * A.out.hs + tid] = (int32_t)(sum >> SCALE);
    }
}

}  // namespace atlas_attn
