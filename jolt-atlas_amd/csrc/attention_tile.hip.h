// The matrix-core path of the quantised attention for many rows of queries: keys and values cut into signed bytes once (k_attn_planes), then one workgroup per tile of
// query rows (k_attn_tile).
//
// An int32 operand in [-8421504, 8355711] is d0 + 2^8 d1 + 2^16 d2 with signed bytes d: the bytes of v + 0x808080, each less 128.  A product of two
// such operands is nine i8 products in five weights, exact in the 32-bit accumulators of v_mfma_i32_32x32x32_i8; on the vector
// unit it is a 64-bit multiply-add per element (the first kernel: 206 ms where this one takes 1.87).  The five sums recombine without 64-bit arithmetic: with hi = a2 + 2^8 a3 + 2^16 a4 and lo = a0 + 2^8 a1,
//     floor((2^16 hi + lo) / 2^14) = 4 hi + (lo >> 14),
// and hi may wrap, as long as the score itself fits 32 bits: |q| |k| d < 2^45, decided per tile from the operands' magnitudes (at 2^45, which only two
// negative powers of two reach, the score is 2^31 and clamps).  Tiles that do not qualify (and operands beyond three bytes) are computed row by row in 64 bits (row_exact).
//
// The products are taken as S^T = K Q^T, so a lane holds 16 scores of ONE query row: maximum, sum and weights stay in registers, and four weights that
// follow each other there are four bytes of the operand of O^T = V^T P^T (the keys of V's fragments are laid out in that order).  The weights
// 0 .. 2^14 are two signed bytes; of the second, most tiles have none (p < 128) and skip it.  sum_j p <= 2^14, so an output accumulator stays below
// 2^21 however many keys there are.
//
// Three passes over the scores, since the floors are taken under the final maximum and sum: maximum; e and its sum (e is held in 16 bits while the keys are few enough, HELD, or
// taken again); product.  Bound by the vector unit (recombining five sums into each score, two table look-ups) and the matrix cores together: of the cycles in which a CU has
// waves, the vector unit is at work for 51 % and the matrix cores for 42 %.  One prompt of 6000 tokens beside five of at most 31, 32 heads of 128 over 8 (295 GFLOP of
// exact products, 24 i8 products for two of them): 1.79-1.93 ms, by the card; 153-165 TFLOP/s, 1.8-2.0 POP/s in int8, where a library's int8 product of
// 8192^3 reaches 2.2-2.3.  Up to 130 new tokens for each of 12 sequences over up to 5001 keys (186 MB, 24 GFLOP): 562 us, 69 of them the digit planes (k_attn_planes, 4.6 TB/s read and
// written); the rest is the longest sequences' tiles, three passes one after the other, while the other workgroups have run out of work.
// Measured and dropped: 3 waves per SIMD (168 registers: spills, 2.6 ms), a raised wave priority around the products (none), the look-ups of 16 scores read together before
// the first product (spills, 2 % slower).
#pragma once
#include "attention_kernels.hip.h"

namespace atlas_attn {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4), aligned(2)));

constexpr uint32_t FRAGMENT = 3 * 1024;            // bytes of 32 x 32 operands: three planes
constexpr uint32_t WIDE = 0x80000000u;             // in a magnitude word: an operand beyond three signed bytes
constexpr uint32_t LOWEST = 0x40000000u;           // an operand may be -2^n, n the word's bits; all others are below 2^n

// the extremes of the operands seen
struct Range {
    int32_t hi = 0, lo = 0;
    // bits of the largest magnitude as a mask (-2^n counts n bits), WIDE where three signed bytes do not hold an operand
    __device__ uint32_t word() const { return (uint32_t)hi | (uint32_t)(lo ^ (lo >> 31)) | (hi > 8355711 || lo < -8421504 ? WIDE : 0); }
    // LOWEST where the least operand is -2^m: of the words that are joined, the one with the joint n among them says so
    __device__ uint32_t lowest() const { return lo < 0 && (lo & (0u - (uint32_t)lo)) == 0u - (uint32_t)lo ? LOWEST : 0; }
};
// four operands that follow each other along the product's inner dimension -> a dword of each digit plane.  The extremes are taken at once (the empty asm):
// left to itself the compiler keeps every operand to do it later, and spills.
__device__ inline void digits4(const int32_t v0, const int32_t v1, const int32_t v2, const int32_t v3, int& p0, int& p1, int& p2, Range& g) {
    g.hi = max(max(g.hi, max(v0, v1)), max(v2, v3));
    g.lo = min(min(g.lo, min(v0, v1)), min(v2, v3));
    asm volatile("" : "+v"(g.hi), "+v"(g.lo));
    const uint32_t u0 = v0 + 0x808080u, u1 = v1 + 0x808080u, u2 = v2 + 0x808080u, u3 = v3 + 0x808080u;
    const uint32_t t01 = __builtin_amdgcn_perm(u1, u0, 0x05010400u), t23 = __builtin_amdgcn_perm(u3, u2, 0x05010400u);
    p0 = (int)(__builtin_amdgcn_perm(t23, t01, 0x05040100u) ^ 0x80808080u);
    p1 = (int)(__builtin_amdgcn_perm(t23, t01, 0x07060302u) ^ 0x80808080u);
    p2 = (int)((__builtin_amdgcn_perm(u1, u0, 0x0c0c0602u) | __builtin_amdgcn_perm(u3, u2, 0x06020c0cu)) ^ 0x80808080u);
}
// elements [i, i + 4) of a row of d, zeros behind its end
template <class T>
__device__ inline void load4(const T* row, uint32_t i, uint32_t d, int32_t (&o)[4]) {
    if (i + 4 <= d) {
        if constexpr (sizeof(T) == 4) { const i32x4 a = *(const i32x4*)(row + i); o[0] = a[0]; o[1] = a[1]; o[2] = a[2]; o[3] = a[3]; }
        else { const i16x4 a = *(const i16x4*)(row + i); o[0] = a[0]; o[1] = a[1]; o[2] = a[2]; o[3] = a[3]; }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) o[e] = i + e < d ? (int32_t)row[i + e] : 0;
    }
}

// The same for [i, i + 16) and then zero_behind.  No branch around a load (places behind the end read elements of the row again): the loads of all
// fragments are on their way together
template <class T>
__device__ inline void fetch16(const T* row, uint32_t i, uint32_t d, int32_t (&o)[4][4]) {
    if (d % 4 == 0) {
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) {
            const T* at = row + min(i + 4 * c, d - 4);
            if constexpr (sizeof(T) == 4) { const i32x4 a = *(const i32x4*)at; o[c][0] = a[0]; o[c][1] = a[1]; o[c][2] = a[2]; o[c][3] = a[3]; }
            else { const i16x4 a = *(const i16x4*)at; o[c][0] = a[0]; o[c][1] = a[1]; o[c][2] = a[2]; o[c][3] = a[3]; }
        }
    } else {
#pragma unroll
        for (uint32_t c = 0; c < 4; c++)
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) o[c][e] = row[min(i + 4 * c + e, d - 1)];
    }
}
__device__ inline void zero_behind(uint32_t i, uint32_t d, int32_t (&o)[4][4]) {
#pragma unroll
    for (uint32_t c = 0; c < 4; c++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) o[c][e] = i + 4 * c + e < d ? o[c][e] : 0;
}

// Digit planes in the order in which the fragments are read: [kv head][tile of 32 keys][fragment of 32 dims][plane][lane][16 bytes], K's and V's each.
//   K: lane l holds key l % 32, dims 16 (l / 32) + b;   V: lane l holds dim l % 32, byte b is key 8 (b / 4) + 4 (l / 32) + b % 4 of the tile
struct Planes {
    uint8_t *k, *v;
    uint32_t *k_mag, *v_mag;       // [kv head][tile]
    uint32_t* there;               // [tile]: which of its keys exist
    uint8_t* e;                    // [workgroup][rows][held] e, 2 bytes each
    uint32_t* next;                // the counters of the tile kernel's work lists
    uint32_t tiles, per_seq;       // per_seq: tiles of a sequence (cached); 0: by its offset (prompt)
};
// Offsets cu[s] / 32 + s are far enough apart for ceil(len / 32) tiles each: no prefix sum is needed
__device__ inline uint32_t tile_base(const Args& A, const Planes& P, uint32_t s) { return P.per_seq ? s * P.per_seq : min((uint32_t)max(A.cu[s], 0), A.n_tokens) / 32 + s; }

template <class CT, int DP>
__global__ __launch_bounds__(256) void k_attn_planes(Args A, Planes P) {
    constexpr int F = DP / 32;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 8) P.next[threadIdx.x] = 0;
    const uint32_t tile = blockIdx.x, kvh = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    const uint32_t si = P.per_seq ? tile / P.per_seq : last_at_most(A.n_seqs, tile, [&](uint32_t s) { return (uint64_t)tile_base(A, P, s); });
    if (si >= A.n_seqs) return;
    const Seq s = seq_at(A, si);
    const uint32_t base = tile_base(A, P, si);
    if (tile < base || s.n_new == 0) return;
    const uint32_t j0 = (tile - base) * 32;
    if (j0 >= s.keys) return;
    __shared__ uint32_t s_mag[2];
    if (threadIdx.x < 2) s_mag[threadIdx.x] = 0;
    __syncthreads();
    // where a key's row begins: keys behind the end are the last one again, those of blocks that do not exist lie in block 0 (they do not count, their weights are 0)
    auto row = [&](uint32_t j, int64_t block, bool value) -> const CT* {
        if (A.table) return (const CT*)(value ? A.cv : A.ck) + cache_at(A, max(block, (int64_t)0), kvh, j);
        const Rows& r = value ? A.v : A.k;
        return (const CT*)r.d + (int64_t)(s.begin + j) * r.ts + (int64_t)kvh * r.hs;
    };
    const int64_t at = ((int64_t)kvh * P.tiles + tile) * (F * FRAGMENT);
    Range rk, rv;
    const uint32_t jk = min(j0 + l32, s.keys - 1);
    const int64_t mine = A.table ? block_of(A, s, jk) : 0;
    const CT* kr = row(jk, mine, false);
    if (wave == 0 && kvh == 0) { const uint64_t b = __ballot(mine >= 0 && j0 + l32 < s.keys); if (lane == 0) P.there[tile] = (uint32_t)b; }
    // Two fragments or fewer: K's and V's on waves of their own.  More: a wave has both, their loads on their way together (128 dims: 90 -> 71 us for 185 MB read)
    constexpr bool BOTH = F > 2;
    const bool ks = BOTH || wave < F, vs = BOTH || (wave >= F && wave < 2 * F);
    // a lane's 16 keys among the values: four times 4 that follow each other
    const CT* vr[4][4];
    if (vs)
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const uint32_t j = min(j0 + 8 * c + 4 * half + x, s.keys - 1);
            if (x > 0 && j0 + 8 * c + 4 * half + x < s.keys && (!A.table || A.log_block >= 2)) vr[c][x] = vr[c][0] + (int64_t)x * (A.table ? (int64_t)A.d : A.v.ts);
            else vr[c][x] = row(j, A.table ? block_of(A, s, j) : 0, true);
        }
#pragma unroll 1
    for (int f = BOTH ? wave : wave % F; f < F; f += 4) {
        int32_t e[4][4], v[4][4];
        if (ks) fetch16(kr, f * 32 + half * 16, A.d, e);
        if (vs)
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int x = 0; x < 4; x++) v[c][x] = (int32_t)vr[c][x][min(f * 32 + l32, A.d - 1)];
        v4i p0, p1, p2;
        if (ks) {
            zero_behind(f * 32 + half * 16, A.d, e);
#pragma unroll
            for (int c = 0; c < 4; c++) { int a, b, g; digits4(e[c][0], e[c][1], e[c][2], e[c][3], a, b, g, rk); p0[c] = a; p1[c] = b; p2[c] = g; }
            v4i* to = (v4i*)(P.k + at + f * (int)FRAGMENT) + lane;
            to[0] = p0; to[64] = p1; to[128] = p2;
        }
        if (vs) {
#pragma unroll
            for (int c = 0; c < 4; c++) { int a, b, g; digits4(v[c][0], v[c][1], v[c][2], v[c][3], a, b, g, rv); p0[c] = a; p1[c] = b; p2[c] = g; }
            v4i* to = (v4i*)(P.v + at + f * (int)FRAGMENT) + lane;
            to[0] = p0; to[64] = p1; to[128] = p2;
        }
    }
    atomicOr(&s_mag[0], rk.word() | rk.lowest());
    atomicOr(&s_mag[1], rv.word());
    __syncthreads();
    if (threadIdx.x == 0) { P.k_mag[(size_t)kvh * P.tiles + tile] = s_mag[0]; P.v_mag[(size_t)kvh * P.tiles + tile] = s_mag[1]; }
}

__device__ inline uint32_t bits_of(uint32_t mag) { mag &= ~LOWEST; return mag ? 32 - __builtin_clz(mag) : 0; }

// 16 bytes per lane from global memory to LDS without a register on the way; lds: the wave's first byte
__device__ inline void copy_to_lds(const uint8_t* src, uint8_t* lds, uint32_t bytes, uint32_t wave, uint32_t lane) {
    for (uint32_t o = wave * 1024; o < bytes; o += 4096)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + o + lane * 16), (__attribute__((address_space(3))) void*)(lds + o), 16, 0, 0);
}
// until at most N of the wave's loads and stores are outstanding; the other counters untouched
template <int N>
__device__ inline void wait_loads() { static_assert(N < 16); __builtin_amdgcn_s_waitcnt(0x0f70 | N); }

// the Mul node's rescale: floor(s c / 2^14) with 1 <= c <= 2^14, s = 2^14 a + b:  a c + floor(b c / 2^14), in 24-bit multiplications
__device__ inline int32_t rescale(int32_t s, int32_t c) {
    const int32_t a = s >> SCALE, b = s & (ONE - 1);
    return __mul24(a, c) + (int32_t)(__umul24((uint32_t)b, (uint32_t)c) >> SCALE);
}

// floor((a0 + 2^8 a1 + 2^16 a2 + 2^24 a3 + 2^32 a4) / 2^14), which fits 32 bits; LONG: more than 128 dims, where 2^8 a1 may not, so that the low part is
// shifted down first (the floors nest)
template <bool LONG>
__device__ inline int32_t combine(int32_t a0, int32_t a1, int32_t a2, int32_t a3, int32_t a4) {
    uint32_t hi = (uint32_t)a2 + ((uint32_t)a3 << 8) + ((uint32_t)a4 << 16);
    asm("" : "+v"(hi));                       // or the shift by 2 is distributed over the three: an instruction more
    const int32_t lo = LONG ? ((a0 >> 8) + a1) >> 6 : (a0 + (int32_t)((uint32_t)a1 << 8)) >> SCALE;
    return (int32_t)((hi << 2) + (uint32_t)lo);
}

// m - rescale(s), the subtraction inside the multiply-add
__device__ inline uint32_t below(int32_t m, int32_t s, int32_t c) {
    return (uint32_t)(__mul24(s >> SCALE, -c) + m) - (__umul24((uint32_t)s & (ONE - 1), (uint32_t)c) >> SCALE);
}

// SPLIT waves share 32 query rows: each scores its own keys and carries 1 / SPLIT of the output's dims
template <int DP, int SPLIT>
struct TileShape {
    static constexpr int F = DP / 32;                         // fragments of 32 dims
    static constexpr int GROUPS = 4 / SPLIT, ROWS = 32 * GROUPS;
    static constexpr int SUBS = SPLIT < 2 ? 2 : SPLIT;        // key sub-tiles of 32 per step
    static constexpr int KEYS = 32 * SUBS, MY_SUBS = SUBS / SPLIT;
    static constexpr int OF = F / SPLIT;                      // output fragments of a wave
    static constexpr uint32_t TILE = F * FRAGMENT, STEP = TILE * SUBS;
    static constexpr int BUFS = DP == 256 ? 1 : 3;            // two steps are on their way while one is worked on; of 256 dims 160 KB of LDS hold one step
    static constexpr int COPIES = STEP / 4096;                // that a wave has issued for a step, at least
    static constexpr uint32_t LUT = 4096, LDS = LUT + STEP * BUFS + 1024;
    static constexpr int WAVES = LDS > 80 * 1024 ? 1 : 2;     // per SIMD
};
// Many tiles: two workgroups per CU, as many rows to a fragment of keys as the registers carry.  FEW tiles: half the rows and twice the waves to a row, so that a tile is
// done in half the time.  A prompt of 2000 with 16 heads of 64 (266 tiles): 206 -> 149 us; with 15 heads of 80 (125 tiles for 512 tokens, 474 for 2000, one workgroup per CU
// then): 64 -> 54 us, but 183 -> 233 us.
constexpr int tile_split(int dp, bool few) { return dp == 32 ? 1 : dp == 64 ? (few ? 2 : 1) : dp == 128 ? (few ? 4 : 2) : 4; }
// The workgroups that fit the chip at once take tiles from a counter.  Each has room for the e of HELD keys of its rows; where a tile has more keys, the scores of the
// others are taken a third time.
constexpr uint32_t TILE_WGS = 512, HELD = 16384;

template <class CT, int DP, int SPLIT, bool LONG>      // LONG: tiles may have more than HELD keys; the product's sums then live through another pass over scores
__global__ __launch_bounds__(256, (TileShape<DP, SPLIT>::WAVES)) void k_attn_tile(Args A, Planes P, uint32_t n_work, uint32_t held) {
    using T = TileShape<DP, SPLIT>;
    constexpr int F = T::F, SUBS = T::SUBS;
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t* s_hi = (uint32_t*)lds;
    uint32_t* s_lo = s_hi + 512;
    uint8_t* s_a = lds + T::LUT;
    uint32_t* s_red = (uint32_t*)(s_a + T::STEP * T::BUFS);        // 256 words
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const uint32_t group = wave / SPLIT, part = wave % SPLIT;
    load_exp<256>(s_hi, s_lo);
    // e of this wave's rows: [tile of 32 keys][lane][16], 2 bytes each, in the order in which a lane has its scores
    const uint32_t held_steps = held / T::KEYS;
    // Work lists by kv head: workgroups go to the 8 XCDs in turn, and those of one XCD begin with the same heads, so that its L2 holds their planes.  A list that
    // has run out is followed by the next one.
    const uint32_t lists = A.KV % 8 == 0 ? 8 : A.KV % 4 == 0 ? 4 : A.KV % 2 == 0 ? 2 : 1;
    uint32_t list = blockIdx.x % lists, tried = 0;
    v4i* const e_rows = (v4i*)(P.e + ((size_t)blockIdx.x * T::GROUPS + group) * held * 64) + lane * 2;
#pragma unroll 1
    for (;;) {
        __syncthreads();
        if (tid == 0) s_red[3] = atomicAdd(P.next + list, 1u);
        if (tid < 3) s_red[tid] = 0;
        if (tid == 4) s_red[4] = 0;
        __syncthreads();
        const uint32_t work = __builtin_amdgcn_readfirstlane(s_red[3]);
        if (work >= n_work / lists) {
            if (++tried == lists) return;
            list = (list + 1) % lists;
            continue;
        }
        const uint32_t heads = A.KV / lists, kvh = list + lists * (work % heads), qt = n_work / A.KV - 1 - work / heads;      // late tiles (many keys under the causal mask) first
        auto q_base = [&](uint32_t s) { return (uint64_t)min((uint32_t)max(A.cu[s], 0), A.n_tokens) * A.G / T::ROWS + s; };
        const uint32_t si = last_at_most(A.n_seqs, qt, q_base);
        const Seq s = seq_at(A, si);
        const uint64_t first = (uint64_t)(qt - q_base(si)) * T::ROWS;
        const uint32_t n_rows = s.n_new * A.G;
        if (qt < q_base(si) || first >= n_rows) continue;
        const uint32_t row0 = (uint32_t)first, rows = min((uint32_t)T::ROWS, n_rows - row0);
        const uint32_t base = tile_base(A, P, si);
        // my row; lanes behind the last one repeat it
        const bool mine = row0 + group * 32 + l32 < n_rows;
        const uint32_t rr = min(row0 + group * 32 + l32, n_rows - 1), tok = rr / A.G, head = kvh * A.G + rr % A.G;
        const uint32_t limit = min(key_limit(A, s, tok), s.keys);
        const uint32_t most = min(key_limit(A, s, (row0 + rows - 1) / A.G), s.keys), n_steps = (most + T::KEYS - 1) / T::KEYS;

        v4i q0[F], q1[F], q2[F];
        bool holes;                                   // some of the sequence's keys lie in blocks that do not exist
        {
            uint32_t mq = 0, mk = 0, mv = 0;
            Range rq;
            const int32_t* q = A.q.d + (int64_t)(s.begin + tok) * A.q.ts + (int64_t)head * A.q.hs;
#pragma unroll
            for (int f = 0; f < F; f++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    int32_t e[4];
                    load4(q, f * 32 + half * 16 + c * 4, A.d, e);
                    int a, b, g;
                    digits4(e[0], e[1], e[2], e[3], a, b, g, rq);
                    q0[f][c] = a; q1[f][c] = b; q2[f][c] = g;
                }
            const uint32_t tiles = (most + 31) / 32;
            uint32_t hole = 0;
            for (uint32_t i = tid; i < tiles; i += 256) {
                mk |= P.k_mag[(size_t)kvh * P.tiles + base + i]; mv |= P.v_mag[(size_t)kvh * P.tiles + base + i];
                const uint32_t n = s.keys - i * 32;
                hole |= ~P.there[base + i] & (n < 32 ? (1u << n) - 1 : ~0u);
            }
            if (hole) s_red[4] = 1;
            atomicOr(&s_red[0], rq.word() | rq.lowest());
            if (mk) atomicOr(&s_red[1], mk);
            if (mv) atomicOr(&s_red[2], mv);
            __syncthreads();
            mq = s_red[0]; mk = s_red[1]; mv = s_red[2];
            holes = s_red[4];
            __syncthreads();
            const uint32_t most_bits = mq & mk & LOWEST ? 44 : 45;         // |q| |k| d may BE 2^45 where both have their lowest
            if (((mq | mk | mv) & WIDE) || bits_of(mq) + bits_of(mk) + bits_of(A.d - 1) > most_bits) {
                int32_t* x_q = (int32_t*)s_a;                          // 1 KB, 1 KB, 2 KB of the tile buffer
                for (uint32_t x = 0; x < rows; x++) row_exact<CT>(A, s, (row0 + x) / A.G, kvh * A.G + (row0 + x) % A.G, x_q, x_q + 256, (uint64_t*)(x_q + 512));
                continue;
            }
        }
        const uint8_t* gk = P.k + ((int64_t)kvh * P.tiles + base) * T::TILE;
        const uint8_t* gv = P.v + ((int64_t)kvh * P.tiles + base) * T::TILE;
        // Steps [from, to) of a plane array through the LDS buffers: begin() sends the first on their way, arrive() waits for one, lets all waves be done with the
        // one before it, and sends the next into that one's place
        auto begin = [&](const uint8_t* src, uint32_t from, uint32_t to) {
            if (T::BUFS == 3 && from < to) copy_to_lds(src + (int64_t)from * T::STEP, s_a, T::STEP, wave, lane);
            if (T::BUFS == 3 && from + 1 < to) copy_to_lds(src + (int64_t)(from + 1) * T::STEP, s_a + T::STEP, T::STEP, wave, lane);
        };
        auto arrive = [&](const uint8_t* src, uint32_t from, uint32_t step, uint32_t to) -> const uint8_t* {
            if constexpr (T::BUFS == 1) {
                __syncthreads();
                copy_to_lds(src + (int64_t)step * T::STEP, s_a, T::STEP, wave, lane);
                wait_loads<0>();
                __syncthreads();
                return s_a;
            } else {
                const uint32_t at = (step - from) % 3;
                if (step + 1 < to) wait_loads<T::COPIES>(); else wait_loads<0>();       // the next step's copies may still be out
                __syncthreads();
                if (step + 2 < to) copy_to_lds(src + (int64_t)(step + 2) * T::STEP, s_a + (at == 0 ? 2 : at - 1) * T::STEP, T::STEP, wave, lane);
                return s_a + at * T::STEP;
            }
        };
        // the scores of sub-tile `sub` of the step in `buf` before the Mul node, in one sweep over the fragments with five accumulators
        auto scores = [&](const uint8_t* buf, int sub, v16i& x) {
            // All fragments are read first: left to itself the compiler reads each into the same registers right before its products, and LDS' latency
            // stands between every four of them
            v4i k[F][3];
            const v4i* kf = (const v4i*)(buf + sub * T::TILE) + lane;
#pragma unroll
            for (int f = 0; f < F; f++)
#pragma unroll
                for (int p = 0; p < 3; p++) k[f][p] = kf[f * 192 + p * 64];
            __builtin_amdgcn_sched_barrier(0);
            v16i a0 = {}, a1 = {}, a2 = {}, a3 = {}, a4 = {};
#pragma unroll
            for (int f = 0; f < F; f++) {
                a4 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][2], q2[f], a4, 0, 0, 0);
                a3 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][2], q1[f], a3, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][2], q0[f], a2, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][1], q0[f], a1, 0, 0, 0);
                a0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][0], q0[f], a0, 0, 0, 0);
                a3 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][1], q2[f], a3, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][1], q1[f], a2, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][0], q1[f], a1, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[f][0], q2[f], a2, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = combine<DP == 256>(a0[i], a1[i], a2[i], a3[i], a4[i]);
        };
        // which of a lane's 16 keys of a sub-tile count, as bits 8 c + i of 4 half + ..; ~0 where all of the wave's do
        auto seen = [&](uint32_t step, int sub) -> uint32_t {
            const uint32_t j0 = step * T::KEYS + sub * 32;
            uint32_t in = limit >= j0 + 32 ? ~0u : limit > j0 ? (1u << (limit - j0)) - 1 : 0;
            if (holes) in &= j0 < s.keys ? P.there[base + j0 / 32] : 0;
            return __all(in == ~0u) ? ~0u : in >> (4 * half);
        };
        int32_t m = INT32_MIN;
        uint32_t sum = 0;
        // steps [from, to): their maximum (MAX), or their e, summed and held
        enum { MAX, SUM, HOLD };
        auto pass = [&](uint32_t from, uint32_t to, int what) {
            begin(gk, from, to);
#pragma unroll 1
            for (uint32_t step = from; step < to; step++) {
                const uint8_t* buf = arrive(gk, from, step, to);
#pragma unroll 1
                for (int y = 0; y < T::MY_SUBS; y++) {
                    const int sub = part * T::MY_SUBS + y;
                    const uint32_t in = seen(step, sub);
                    const bool any = __any(in != 0);
                    v16i x;
                    if (any) scores(buf, sub, x);
                    if (what == MAX) {
                        if (!any) continue;
                        if (in != ~0u)
#pragma unroll
                            for (int i = 0; i < 16; i++) { const int32_t keep = (int32_t)(in << (31 - (8 * (i / 4) + i % 4))) >> 31; x[i] = (x[i] & keep) | (INT32_MIN & ~keep); }
#pragma unroll
                        for (int i = 0; i < 16; i++) m = max(m, x[i]);
                    } else {
                        uint32_t e[16] = {};
                        if (any) {
#pragma unroll
                            for (int i = 0; i < 16; i++) e[i] = exp_lds(below(m, x[i], A.mul), s_hi, s_lo);
                            if (in != ~0u)
#pragma unroll
                                for (int i = 0; i < 16; i++) e[i] &= (uint32_t)((int32_t)(in << (31 - (8 * (i / 4) + i % 4))) >> 31);
                        }
                        if (what == SUM) {
                            uint32_t t = 0;
#pragma unroll
                            for (int i = 0; i < 16; i++) t += e[i];                       // <= 2^18
                            sum = __builtin_elementwise_add_sat(sum, t);
                        }
                        if (!LONG || step - from < held_steps) {
                            v4i w[2];
#pragma unroll
                            for (int i = 0; i < 8; i++) w[i / 4][i % 4] = (int)(e[2 * i] | (e[2 * i + 1] << 16));
                            v4i* to_e = e_rows + (size_t)((step - from) * SUBS + sub) * 128;
                            to_e[0] = w[0]; to_e[1] = w[1];
                        }
                    }
                }
            }
            __threadfence_block();
            __syncthreads();
        };
#pragma unroll 1
        for (int what = MAX; what <= SUM; what++) {
            pass(0, n_steps, what);
            // the other half-wave has the rest of the row's keys, and so have the waves that share the rows
            // (the Mul node's rescale does not change the order: it is left to the maximum)
            if (what == MAX) m = max(m, __shfl_xor(m, 32)); else sum = __builtin_elementwise_add_sat(sum, (uint32_t)__shfl_xor((int)sum, 32));
            if (SPLIT > 1) {
                if (half == 0) s_red[wave * 32 + l32] = what == MAX ? (uint32_t)m : sum;
                __syncthreads();
                for (int p = 0; p < SPLIT; p++) {
                    const uint32_t o = s_red[(group * SPLIT + p) * 32 + l32];
                    if (p != (int)part) { if (what == MAX) m = max(m, (int32_t)o); else sum = __builtin_elementwise_add_sat(sum, o); }
                }
                __syncthreads();
            }
            if (what == MAX) m = rescale(m, A.mul);
        }
        const uint32_t inv = sum ? (1u << (2 * SCALE)) / sum : 0;
        if (A.status && part == 0 && half == 0 && mine && sum && mask_weighs(A, s, tok, m)) atomicOr(A.status, (uint32_t)ATLAS_ATTN_MASK_WEIGHS);

        // ---- the weights from the e that are held, and their product with the values.  o[.][f]: the sums with the values' digit 0, 1, 2
        v16i o0[T::OF] = {}, o1[T::OF] = {}, o2[T::OF] = {};
        auto product = [&](uint32_t from, uint32_t to) {
            if (from >= to) return;
            v4i w[SUBS][2];
            auto load_e = [&](uint32_t step) {
#pragma unroll
                for (int sub = 0; sub < SUBS; sub++) { const v4i* x = e_rows + (size_t)((step - from) * SUBS + sub) * 128; w[sub][0] = x[0]; w[sub][1] = x[1]; }
            };
            begin(gv, from, to);
            load_e(from);
#pragma unroll 1
            for (uint32_t step = from; step < to; step++) {
                // p = (signed byte) p + 2^8 ((p + 128) >> 8)
                v4i b0[SUBS], b1[SUBS];
#pragma unroll
                for (int sub = 0; sub < SUBS; sub++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t a = (uint32_t)w[sub][c / 2][2 * (c % 2)], b = (uint32_t)w[sub][c / 2][2 * (c % 2) + 1];
                        a = (__umul24(a & 0xffff, inv) >> SCALE) | ((__umul24(a >> 16, inv) >> SCALE) << 16);
                        b = (__umul24(b & 0xffff, inv) >> SCALE) | ((__umul24(b >> 16, inv) >> SCALE) << 16);
                        b0[sub][c] = (int)__builtin_amdgcn_perm(b, a, 0x06040200u);
                        b1[sub][c] = (int)__builtin_amdgcn_perm(b + 0x00800080u, a + 0x00800080u, 0x07050301u);
                    }
                const uint8_t* buf = arrive(gv, from, step, to);
                v4i v[SUBS][T::OF][3];
#pragma unroll
                for (int sub = 0; sub < SUBS; sub++)
#pragma unroll
                    for (int f = 0; f < T::OF; f++)
#pragma unroll
                        for (int p = 0; p < 3; p++) v[sub][f][p] = ((const v4i*)(buf + sub * T::TILE + (part * T::OF + f) * (int)FRAGMENT) + lane)[p * 64];
                if (step + 1 < to) load_e(step + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int sub = 0; sub < SUBS; sub++) {
                    const bool second = __any((b1[sub][0] | b1[sub][1] | b1[sub][2] | b1[sub][3]) != 0);
#pragma unroll
                    for (int f = 0; f < T::OF; f++) {
                        o0[f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(v[sub][f][0], b0[sub], o0[f], 0, 0, 0);
                        o1[f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(v[sub][f][1], b0[sub], o1[f], 0, 0, 0);
                        o2[f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(v[sub][f][2], b0[sub], o2[f], 0, 0, 0);
                    }
                    if (second) {
#pragma unroll
                        for (int f = 0; f < T::OF; f++) {
                            o0[f] += __builtin_amdgcn_mfma_i32_32x32x32_i8(v[sub][f][0], b1[sub], v16i{}, 0, 0, 0) * 256;
                            o1[f] += __builtin_amdgcn_mfma_i32_32x32x32_i8(v[sub][f][1], b1[sub], v16i{}, 0, 0, 0) * 256;
                            o2[f] += __builtin_amdgcn_mfma_i32_32x32x32_i8(v[sub][f][2], b1[sub], v16i{}, 0, 0, 0) * 256;
                        }
                    }
                }
            }
            __syncthreads();
        };
        product(0, LONG ? min(n_steps, held_steps) : n_steps);
        if constexpr (LONG)
#pragma unroll 1
            for (uint32_t from = held_steps; from < n_steps; from += held_steps) {
                pass(from, min(n_steps, from + held_steps), HOLD);
                product(from, min(n_steps, from + held_steps));
            }
        // floor((o0 + 2^8 o1 + 2^16 o2) / 2^14): a lane holds dims 8 c + 4 half .. + 3 of its row
        if (mine) {
            int32_t* out = A.out.d + (int64_t)(s.begin + tok) * A.out.ts + (int64_t)head * A.out.hs;
#pragma unroll
            for (int f = 0; f < T::OF; f++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t i = (part * T::OF + f) * 32 + 8 * c + 4 * half;
                    i32x4 y;
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = (int32_t)(((int64_t)o0[f][4 * c + e] + ((int64_t)o1[f][4 * c + e] << 8) + ((int64_t)o2[f][4 * c + e] << 16)) >> SCALE);
                    if (i + 4 <= A.d) *(i32x4*)(out + i) = y;
                    else for (uint32_t e = 0; e < 4; e++) if (i + e < A.d) out[i + e] = y[e];
                }
        }
    }
}

}  // namespace atlas_attn
