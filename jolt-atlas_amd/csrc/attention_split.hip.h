// The quantised attention of few query rows over long caches (decoding): bound by reading the cache once.  The keys of a sequence are split over workgroups in chunks,
// and four launches join them: k_split_scores (reads the keys, keeps the scores and each chunk's maximum), k_split_sums, k_split_values (reads the values), k_split_join.
// Splitting costs nothing in exactness: maxima and integer sums do not depend on the order.
//
// Up to 16 rows (the heads that share a kv head, times the new tokens) are the columns of v_mfma_i32_16x16x64_i8.  Keys go from memory into the fragments' own lanes
// (16 dims of one key: 64 contiguous bytes) and are cut into digits in registers, values the same with 4 dims of 16 keys per lane; nothing
// passes through LDS.  About 4.3 vector operations per element against 32 that the memory's rate leaves room for.
#pragma once
#include "attention_tile.hip.h"

namespace atlas_attn {

struct Split {
    int32_t* scores;             // [row][pitch]; row = token * heads + head; GONE where no key counts
    int32_t* cmax;               // [chunk][row]
    uint32_t* csum;              // [segment][row]
    int32_t* rmax;               // [row]
    uint32_t *q_mag, *k_mag, *v_mag;      // [row tile * kv heads + kv head], the latter two by chunk in front
    int64_t* part;               // [chunk][row][d]
    uint32_t chunk, n_chunks, n_tiles, n_rows;
    int64_t pitch;
};
constexpr int32_t GONE = INT32_MIN;       // no score of this path reaches it: |score| < 2^30 (SPLIT_BITS)
constexpr uint32_t SPLIT_BITS = 44, SEGMENT = 4096, TILE_ROWS = 16;

// Four elements of a row from i on, without a branch around the load: places behind the row's end get elements of the row again (they meet zeros of the
// query, or outputs that nobody stores).  QUAD: head_dim is a multiple of 4, one vector load
template <bool QUAD, class T>
__device__ inline void fetch4(const T* row, uint32_t i, uint32_t d, int32_t (&o)[4]) {
    if constexpr (QUAD) {
        i = min(i, d - 4);
        if constexpr (sizeof(T) == 4) { const i32x4 a = *(const i32x4*)(row + i); o[0] = a[0]; o[1] = a[1]; o[2] = a[2]; o[3] = a[3]; }
        else { const i16x4 a = *(const i16x4*)(row + i); o[0] = a[0]; o[1] = a[1]; o[2] = a[2]; o[3] = a[3]; }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) o[e] = row[min(i + e, d - 1)];
    }
}

// the rows of a workgroup: 16 (token, head of the group) pairs of one sequence
struct RowTile { Seq s; uint32_t row0, n_rows, tile, kvh; bool any; };
__device__ inline RowTile row_tile(const Args& A, uint32_t x) {
    RowTile t;
    t.kvh = x % A.KV; t.tile = x / A.KV;
    auto base = [&](uint32_t s) { return (uint64_t)min((uint32_t)max(A.cu[s], 0), A.n_tokens) * A.G / TILE_ROWS + s; };
    const uint32_t si = last_at_most(A.n_seqs, t.tile, base);
    t.s = seq_at(A, si);
    t.n_rows = t.s.n_new * A.G;
    const uint64_t b = base(si);
    const uint64_t first = t.tile >= b ? (t.tile - b) * TILE_ROWS : ~0ull;
    t.any = first < t.n_rows;
    t.row0 = (uint32_t)first;
    return t;
}
__device__ inline uint32_t row_id(const Args& A, const RowTile& t, uint32_t r) { return (t.s.begin + r / A.G) * A.H + t.kvh * A.G + r % A.G; }

template <class CT, int KS, bool QUAD>      // KS: steps of 64 dims
__global__ __launch_bounds__(256, KS > 2 ? 1 : 2) void k_split_scores(Args A, Split S) {
    const RowTile R = row_tile(A, blockIdx.x);
    const uint32_t c = blockIdx.y, k0 = c * S.chunk;
    if (!R.any || k0 >= R.s.keys) return;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, l = lane & 15;
    const uint32_t r = R.row0 + l;
    const bool mine = r < R.n_rows;
    const uint32_t id = mine ? row_id(A, R, r) : 0, limit = mine ? min(key_limit(A, R.s, r / A.G), R.s.keys) : 0;
    __shared__ int32_t s_max[4][16];
    __shared__ uint32_t s_mag[2];
    if (tid < 2) s_mag[tid] = 0;
    __syncthreads();
    v4i q0[KS], q1[KS], q2[KS];
    Range rq, rk;
    {
        const int32_t* q = A.q.d + (int64_t)(R.s.begin + (mine ? r / A.G : 0)) * A.q.ts + (int64_t)(R.kvh * A.G + (mine ? r % A.G : 0)) * A.q.hs;
#pragma unroll
        for (int f = 0; f < KS; f++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                int32_t e[4];
                const uint32_t i = f * 64 + g * 16 + x * 4;
                fetch4<QUAD>(q, i, A.d, e);
#pragma unroll
                for (uint32_t y = 0; y < 4; y++) e[y] = mine && i + y < A.d ? e[y] : 0;
                int a, b, d;
                digits4(e[0], e[1], e[2], e[3], a, b, d, rq);
                q0[f][x] = a; q1[f][x] = b; q2[f][x] = d;
            }
    }
    int32_t m = GONE;
    const uint32_t k1 = min(k0 + S.chunk, R.s.keys);
#pragma unroll 1
    for (uint32_t j0 = k0 + wave * 64; j0 < k1; j0 += 256) {
        const CT* row[4];
        uint32_t there[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint32_t j = min(j0 + 16 * t + l, k1 - 1);              // behind the end: the last key again, its score does not count
            const int64_t b = block_of(A, R.s, j);
            row[t] = (const CT*)A.ck + cache_at(A, max(b, (int64_t)0), R.kvh, j);
            there[t] = (uint32_t)__ballot(b >= 0 && j0 + 16 * t + l < k1) & 0xffff;
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (t == 2) __builtin_amdgcn_sched_barrier(0);               // two sub-tiles' loads in flight; all four would spill
            v4i a0 = {}, a1 = {}, a2 = {}, a3 = {}, a4 = {};
#pragma unroll
            for (int f = 0; f < KS; f++) {
                v4i p0, p1, p2;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    int32_t e[4];
                    fetch4<QUAD>(row[t], f * 64 + g * 16 + x * 4, A.d, e);
                    int a, b, d;
                    digits4(e[0], e[1], e[2], e[3], a, b, d, rk);
                    p0[x] = a; p1[x] = b; p2[x] = d;
                }
                a4 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, q2[f], a4, 0, 0, 0);
                a3 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, q1[f], a3, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, q0[f], a2, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, q0[f], a1, 0, 0, 0);
                a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, q0[f], a0, 0, 0, 0);
                a3 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, q2[f], a3, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, q1[f], a2, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, q1[f], a1, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, q2[f], a2, 0, 0, 0);
            }
            v4i x;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int32_t v = A.mul != ONE ? rescale(combine<KS == 4>(a0[i], a1[i], a2[i], a3[i], a4[i]), A.mul) : combine<KS == 4>(a0[i], a1[i], a2[i], a3[i], a4[i]);
                const uint32_t at = 4 * g + i;
                x[i] = ((there[t] >> at) & 1) && j0 + 16 * t + at < limit ? v : GONE;
                m = max(m, x[i]);
            }
            if (mine) *(v4i*)(S.scores + (int64_t)id * S.pitch + j0 + 16 * t + 4 * g) = x;
        }
    }
    m = max(m, __shfl_xor(m, 16));
    m = max(m, __shfl_xor(m, 32));
    if (g == 0) s_max[wave][l] = m;
    atomicOr(&s_mag[0], rq.word());
    atomicOr(&s_mag[1], rk.word());
    __syncthreads();
    if (tid < 16 && mine) S.cmax[(int64_t)c * S.n_rows + id] = max(max(s_max[0][l], s_max[1][l]), max(s_max[2][l], s_max[3][l]));
    if (tid == 0) { S.k_mag[(int64_t)c * gridDim.x + blockIdx.x] = s_mag[1]; if (c == 0) S.q_mag[blockIdx.x] = s_mag[0]; }
}

// one workgroup per row and segment of 4096 keys
__global__ __launch_bounds__(256) void k_split_sums(Args A, Split S) {
    const uint32_t id = blockIdx.x, t = id / A.H, seg = blockIdx.y, tid = threadIdx.x;
    const uint32_t si = find_seq(A.cu, A.n_seqs, t);
    if (si >= A.n_seqs) return;
    const Seq s = seq_at(A, si);
    if (t < s.begin || t - s.begin >= s.n_new || seg * SEGMENT >= s.keys) return;
    __shared__ int32_t s_hi[512], s_lo[512], s_m[4];
    __shared__ uint32_t s_s[4];
    for (uint32_t i = tid; i < 512; i += 256) { s_hi[i] = g_exp.hi[i]; s_lo[i] = g_exp.lo[i]; }
    const uint32_t chunks = (s.keys + S.chunk - 1) / S.chunk;
    int32_t m = GONE;
    for (uint32_t c = tid; c < chunks; c += 256) m = max(m, S.cmax[(int64_t)c * S.n_rows + id]);
    for (int o = 32; o; o >>= 1) m = max(m, __shfl_xor(m, o));
    if ((tid & 63) == 0) s_m[tid >> 6] = m;
    __syncthreads();
    m = max(max(s_m[0], s_m[1]), max(s_m[2], s_m[3]));
    const uint32_t end = min((seg + 1) * SEGMENT, s.keys);
    uint32_t sum = 0;
    for (uint32_t j = seg * SEGMENT + tid * 4; j < end; j += 1024) {
        const v4i x = *(const v4i*)(S.scores + (int64_t)id * S.pitch + j);      // behind the last key: GONE up to the next multiple of 64
#pragma unroll
        for (int i = 0; i < 4; i++) sum += x[i] == GONE ? 0u : (uint32_t)exp_q((uint32_t)m - (uint32_t)x[i], s_hi, s_lo);      // 16 e <= 2^18 per thread
    }
    for (int o = 32; o; o >>= 1) sum += (uint32_t)__shfl_xor((int)sum, o);
    if ((tid & 63) == 0) s_s[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) { S.csum[(int64_t)seg * S.n_rows + id] = s_s[0] + s_s[1] + s_s[2] + s_s[3]; if (seg == 0) S.rmax[id] = m; }      // <= 2^26
}

template <class CT, int KS, bool QUAD>
__global__ __launch_bounds__(256, KS > 2 ? 1 : 2) void k_split_values(Args A, Split S) {
    const RowTile R = row_tile(A, blockIdx.x);
    const uint32_t c = blockIdx.y, k0 = c * S.chunk;
    if (!R.any || k0 >= R.s.keys) return;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, l = lane & 15;
    constexpr int D = KS * 64;
    __shared__ int32_t s_hi[512], s_lo[512];
    __shared__ unsigned long long s_o[TILE_ROWS * D];
    __shared__ uint32_t s_mag;
    for (uint32_t i = tid; i < 512; i += 256) { s_hi[i] = g_exp.hi[i]; s_lo[i] = g_exp.lo[i]; }
    for (uint32_t i = tid; i < TILE_ROWS * D; i += 256) s_o[i] = 0;
    if (tid == 0) s_mag = 0;
    const uint32_t r = R.row0 + l;
    const bool mine = r < R.n_rows;
    const uint32_t id = mine ? row_id(A, R, r) : 0;
    int32_t m = 0;
    uint32_t inv = 0;
    if (mine) {
        m = S.rmax[id];
        uint32_t sum = 0;
        for (uint32_t x = 0; x * SEGMENT < R.s.keys; x++) sum = __builtin_elementwise_add_sat(sum, S.csum[(int64_t)x * S.n_rows + id]);
        inv = sum ? (1u << (2 * SCALE)) / sum : 0;
    }
    __syncthreads();
    v4i o0[KS * 4] = {}, o1[KS * 4] = {}, o2[KS * 4] = {};
    Range rv;
    const uint32_t k1 = min(k0 + S.chunk, R.s.keys);
#pragma unroll 1
    for (uint32_t j0 = k0 + wave * 64; j0 < k1; j0 += 256) {
        v4i w0 = {}, w1 = {};
        if (mine) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const v4i x = *(const v4i*)(S.scores + (int64_t)id * S.pitch + j0 + 16 * t + 4 * g);
                uint32_t p[4];
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] = x[i] == GONE ? 0 : __umul24((uint32_t)exp_q((uint32_t)m - (uint32_t)x[i], s_hi, s_lo), inv) >> SCALE;
                const uint32_t a = p[0] | (p[1] << 16), b = p[2] | (p[3] << 16);
                w0[t] = (int)__builtin_amdgcn_perm(b, a, 0x06040200u);
                w1[t] = (int)__builtin_amdgcn_perm(b + 0x00800080u, a + 0x00800080u, 0x07050301u);
            }
        }
        const bool second = __any((w1[0] | w1[1] | w1[2] | w1[3]) != 0);
        // the rows of this lane's 16 keys: 16 t + 4 g + i
        const CT* vr[4][4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t j = min(j0 + 16 * t + 4 * g + i, k1 - 1);      // behind the end, and in blocks that do not exist: any values, their weights are 0
                if (i > 0 && A.log_block >= 2 && j0 + 16 * t + 4 * g + i < k1) vr[t][i] = vr[t][0] + (int64_t)i * A.d;
                else vr[t][i] = (const CT*)A.cv + cache_at(A, max(block_of(A, R.s, j), (int64_t)0), R.kvh, j);
            }
#pragma unroll
        for (int f = 0; f < KS; f++) {
            if (f) __builtin_amdgcn_sched_barrier(0);
            int32_t v[4][4][4];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) fetch4<QUAD>(vr[t][i], f * 64 + l * 4, A.d, v[t][i]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v4i p0, p1, p2;
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    int a, b, d;
                    digits4(v[t][0][e], v[t][1][e], v[t][2][e], v[t][3][e], a, b, d, rv);
                    p0[t] = a; p1[t] = b; p2[t] = d;
                }
                const int x = f * 4 + e;
                o0[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, w0, o0[x], 0, 0, 0);
                o1[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, w0, o1[x], 0, 0, 0);
                o2[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, w0, o2[x], 0, 0, 0);
                if (second) {
                    o0[x] += __builtin_amdgcn_mfma_i32_16x16x64_i8(p0, w1, v4i{}, 0, 0, 0) * 256;
                    o1[x] += __builtin_amdgcn_mfma_i32_16x16x64_i8(p1, w1, v4i{}, 0, 0, 0) * 256;
                    o2[x] += __builtin_amdgcn_mfma_i32_16x16x64_i8(p2, w1, v4i{}, 0, 0, 0) * 256;
                }
            }
        }
    }
    atomicOr(&s_mag, rv.word());
    if (mine) {
#pragma unroll
        for (int x = 0; x < KS * 4; x++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t y = (int64_t)o0[x][i] + ((int64_t)o1[x][i] << 8) + ((int64_t)o2[x][i] << 16);
                atomicAdd(&s_o[l * D + (x / 4) * 64 + (4 * g + i) * 4 + x % 4], (unsigned long long)y);
            }
    }
    __syncthreads();
    const uint32_t rows = min(TILE_ROWS, R.n_rows - R.row0);
    for (uint32_t i = tid; i < rows * D; i += 256) {
        const uint32_t x = i / D, y = i % D;
        if (y < A.d) S.part[((int64_t)c * S.n_rows + row_id(A, R, R.row0 + x)) * A.d + y] = (int64_t)s_o[i];
    }
    if (tid == 0) S.v_mag[(int64_t)c * gridDim.x + blockIdx.x] = s_mag;
}

// the chunks' products added up; where the operands did not fit the digits, the rows again in 64 bits
template <class CT>
__global__ __launch_bounds__(256) void k_split_join(Args A, Split S) {
    const RowTile R = row_tile(A, blockIdx.x);
    if (!R.any) return;
    const uint32_t tid = threadIdx.x, chunks = (R.s.keys + S.chunk - 1) / S.chunk, rows = min(TILE_ROWS, R.n_rows - R.row0);
    __shared__ uint32_t s_mag[3];
    __shared__ int32_t s_q[256], s_p[256];
    __shared__ uint64_t s_red[256];
    if (tid < 3) s_mag[tid] = 0;
    __syncthreads();
    for (uint32_t c = tid; c < chunks; c += 256) {
        atomicOr(&s_mag[1], S.k_mag[(int64_t)c * gridDim.x + blockIdx.x]);
        atomicOr(&s_mag[2], S.v_mag[(int64_t)c * gridDim.x + blockIdx.x]);
        if (c == 0) atomicOr(&s_mag[0], S.q_mag[blockIdx.x]);
    }
    __syncthreads();
    const uint32_t mq = s_mag[0], mk = s_mag[1], mv = s_mag[2];
    if (((mq | mk | mv) & WIDE) || bits_of(mq) + bits_of(mk) + bits_of(A.d - 1) > SPLIT_BITS) {
        for (uint32_t x = 0; x < rows; x++) row_exact<CT>(A, R.s, (R.row0 + x) / A.G, R.kvh * A.G + (R.row0 + x) % A.G, s_q, s_p, s_red);
        return;
    }
    for (uint32_t i = tid; i < rows * A.d; i += 256) {
        const uint32_t x = R.row0 + i / A.d, y = i % A.d, id = row_id(A, R, x);
        int64_t sum = 0;
        for (uint32_t c = 0; c < chunks; c++) sum += S.part[((int64_t)c * S.n_rows + id) * A.d + y];
        A.out.d[(int64_t)(R.s.begin + x / A.G) * A.out.ts + (int64_t)(R.kvh * A.G + x % A.G) * A.out.hs + y] = (int32_t)(sum >> SCALE);
    }
}

}  // namespace atlas_attn
