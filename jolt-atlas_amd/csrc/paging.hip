// The paged cache of generation (include/atlas_hip.h: atlas_kv_plan, atlas_kv_write): block tables and slot maps from request lengths, on the device, and
// the write of new keys and values into their slots.
#include "runtime.hpp"

#include "attention_launch.hpp"

using atlas_attn::log2_of;
using atlas_rt::fail;

namespace {

typedef int32_t int4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int16_t short4u __attribute__((ext_vector_type(4), aligned(2)));

// ---- the write: 4 elements of one row's head per thread, 16 bytes in and 16 (or 8) out.  Bound by memory: 16001 tokens of 8 heads of
// 128 into a 16-bit cache (131 MB in, 66 out) 39 us, 5.0 TB/s, where a copy of 4 GB reaches 4.8; 64 tokens 8 us, which is the time to enqueue it.
struct WriteArgs {
    const int32_t *k, *v;
    int64_t k_ts, k_hs, v_ts, v_hs;
    const int64_t* slots;
    void *ck, *cv;
    uint32_t* status;
    uint32_t n_tokens, KV, d, log_block;
    int64_t n_slots;
};
template <class CT>
__global__ __launch_bounds__(256) void k_kv_write(WriteArgs W) {
    const uint32_t quads = (W.d + 3) / 4, per_row = W.KV * quads;
    const uint64_t n = (uint64_t)W.n_tokens * per_row;
    uint32_t told = 0;
    for (uint64_t x = (uint64_t)blockIdx.x * 256 + threadIdx.x; x < n; x += (uint64_t)gridDim.x * 256) {
        const uint32_t t = (uint32_t)(x / per_row), r = (uint32_t)(x % per_row), h = r / quads, i = (r % quads) * 4;
        const int64_t slot = W.slots[t];
        if (slot < 0) continue;
        if (slot >= W.n_slots) { told |= ATLAS_KV_BAD_SLOT; continue; }
        const int64_t at = ((((slot >> W.log_block) * W.KV + h) << W.log_block) + (slot & ((1ll << W.log_block) - 1))) * W.d + i;
        const uint32_t m = min(4u, W.d - i);
#pragma unroll
        for (int which = 0; which < 2; which++) {
            const int32_t* src = which ? W.v + t * W.v_ts + h * W.v_hs + i : W.k + t * W.k_ts + h * W.k_hs + i;
            CT* dst = (CT*)(which ? W.cv : W.ck) + at;
            if (m == 4) {
                const int4u a = *(const int4u*)src;
                if constexpr (sizeof(CT) == 4) { *(int4u*)dst = a; }
                else {
                    short4u o;
#pragma unroll
                    for (int e = 0; e < 4; e++) { const int32_t c = max(-32768, min(32767, a[e])); if (c != a[e]) told |= ATLAS_KV_NARROW; o[e] = (int16_t)c; }
                    *(short4u*)dst = o;
                }
            } else {
                for (uint32_t e = 0; e < m; e++) {
                    const int32_t a = src[e], c = sizeof(CT) == 4 ? a : max(-32768, min(32767, a));
                    if (c != a) told |= ATLAS_KV_NARROW;
                    dst[e] = (CT)c;
                }
            }
        }
    }
    if (told && W.status) atomicOr(W.status, told);
}

// ---- the plan.  need_i = ceil((c_i + n_i) / B) - ceil(c_i / B) blocks; P_i their exclusive prefix sum over the requests, R the blocks given back: block t of request i is
// stack[n_free + R - 1 - P_i - t].  Bound by latency: 64 single tokens 11 us (10 of them the kernel), 4000 requests 27 + 6 us, which is the one workgroup that
// adds them up, 1024 at a time (2.5 MB are touched: 0.5 us).
struct PlanArgs {
    const int32_t *have, *fresh;
    int32_t *table, *free_, *n_free_out, *cu, *lens, *positions;
    const int32_t* n_free;
    int64_t* slots;
    uint32_t* status;
    uint32_t* ws;                    // [0] status, [1] the stack's top; [4 + i] = P_i
    int64_t table_stride;
    uint32_t n, max_tokens, log_block, n_blocks, max_blocks;
};
struct Request { uint32_t tokens, need, back, bad; };
__device__ inline Request request_at(const PlanArgs& P, uint32_t i) {
    Request r{0, 0, 0, 0};
    const int64_t c = P.have[i], f = P.fresh[i], B = (int64_t)1 << P.log_block, cols = P.max_blocks;
    if (c < 0 || f < -1) { r.bad = ATLAS_KV_BAD_LENGTH; return r; }
    const int64_t hb = (c + B - 1) >> P.log_block, tb = (c + (f > 0 ? f : 0) + B - 1) >> P.log_block;
    if (tb > cols || c + f > 0x7fffffff) { r.bad = ATLAS_KV_NO_COLUMNS; return r; }
    if (f < 0) r.back = (uint32_t)hb;
    else { r.tokens = (uint32_t)f; r.need = (uint32_t)(tb - hb); }
    return r;
}
// inclusive scan of three 64-bit counters over the workgroup of 1024
struct Three { uint64_t a, b, c; };
__device__ inline Three scan3(Three v, Three* s_w, Three& total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint64_t a = __shfl_up(v.a, o), b = __shfl_up(v.b, o), c = __shfl_up(v.c, o);
        if (lane >= o) { v.a += a; v.b += b; v.c += c; }
    }
    if (lane == 63) s_w[wave] = v;
    __syncthreads();
    Three base{0, 0, 0};
    total = Three{0, 0, 0};
    for (uint32_t w = 0; w < 16; w++) { const Three t = s_w[w]; if (w < wave) { base.a += t.a; base.b += t.b; base.c += t.c; } total.a += t.a; total.b += t.b; total.c += t.c; }
    __syncthreads();
    v.a += base.a; v.b += base.b; v.c += base.c;
    return v;
}
// one workgroup: the sums of the step, whether it fits, the offsets, and the blocks that come back
__device__ void plan_scan(const PlanArgs& P) {
    __shared__ Three s_w[16];
    __shared__ uint32_t s_bad;
    const uint32_t tid = threadIdx.x;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    Three sum{0, 0, 0};
    uint32_t bad = 0;
    for (uint32_t i = tid; i < P.n; i += 1024) { const Request r = request_at(P, i); sum.a += r.tokens; sum.b += r.need; sum.c += r.back; bad |= r.bad; }
    if (bad) atomicOr(&s_bad, bad);
    Three total;
    scan3(sum, s_w, total);
    const int64_t n_free = *P.n_free;
    __syncthreads();
    bad = s_bad;
    if (n_free < 0 || n_free + (int64_t)total.c > P.n_blocks) bad |= ATLAS_KV_BAD_LENGTH;
    else if ((int64_t)total.b > n_free + (int64_t)total.c) bad |= ATLAS_KV_NO_BLOCKS;
    if (total.a > P.max_tokens) bad |= ATLAS_KV_NO_TOKENS;
    const int64_t top = n_free + (int64_t)total.c;
    __syncthreads();
    if (tid == 0) { P.ws[0] = bad; P.ws[1] = (uint32_t)top; *P.status = bad; *P.n_free_out = (int32_t)(bad ? n_free : top - (int64_t)total.b); P.cu[0] = 0; }
    Three before{0, 0, 0};
    for (uint32_t i0 = 0; i0 < P.n; i0 += 1024) {
        const uint32_t i = i0 + tid;
        Request r{0, 0, 0, 0};
        if (i < P.n && !bad) r = request_at(P, i);
        Three all;
        const Three inc = scan3(Three{r.tokens, r.need, r.back}, s_w, all);
        if (i < P.n) {
            const int32_t c = P.have[i];
            P.cu[i + 1] = bad ? 0 : (int32_t)(before.a + inc.a);
            P.lens[i] = bad ? c : P.fresh[i] < 0 ? 0 : c + (int32_t)r.tokens;
            P.ws[4 + i] = (uint32_t)(before.b + inc.b - r.need);
        }
        // the blocks of ended requests: their waves copy them, 64 entries at a time (one thread per request took 85 us where 120 of 4000 requests ended)
        for (uint64_t todo = __ballot(r.back != 0); todo; todo &= todo - 1) {
            const int from = __builtin_ctzll(todo);
            const uint32_t who = i0 + (tid & ~63u) + from, n = __shfl(r.back, from);
            const int64_t to = n_free + (int64_t)__shfl((unsigned long long)(before.c + inc.c - r.back), from);
            for (uint32_t b = tid & 63; b < n; b += 64) P.free_[to + b] = P.table[(int64_t)who * P.table_stride + b];
        }
        before.a += all.a; before.b += all.b; before.c += all.c;
    }
}
// the new tokens: token t of the step belongs to request i with cu[i] <= t < cu[i + 1]; the token that opens a block enters it into the table
__device__ void plan_tokens(const PlanArgs& P, uint32_t first, uint32_t step) {
    const uint32_t bad = P.ws[0];
    const int64_t top = P.ws[1];
    const uint32_t total = bad ? 0 : (uint32_t)P.cu[P.n], mask = (1u << P.log_block) - 1;
    for (uint32_t t = first; t < P.max_tokens; t += step) {
        if (t >= total) { P.slots[t] = -1; if (P.positions) P.positions[t] = 0; continue; }
        uint32_t lo = 0, hi = P.n;
        while (hi - lo > 1) { const uint32_t mid = (lo + hi) / 2; if (t >= (uint32_t)P.cu[mid]) lo = mid; else hi = mid; }
        const uint32_t have = (uint32_t)P.have[lo], pos = have + (t - (uint32_t)P.cu[lo]), col = pos >> P.log_block, old = (have + mask) >> P.log_block;
        int32_t* entry = P.table + (int64_t)lo * P.table_stride + col;
        int32_t block;
        if (col < old) block = *entry;
        else {
            block = P.free_[top - 1 - (int64_t)P.ws[4 + lo] - (col - old)];
            if ((pos & mask) == 0) *entry = block;
        }
        P.slots[t] = (int64_t)block * (1ll << P.log_block) + (pos & mask);
        if (P.positions) P.positions[t] = (int32_t)pos;
    }
}
// Up to here one workgroup does both parts, beyond it the tokens have a launch of their own: 1024 tokens of 64 requests 9.8 us in one launch and 11.3 in two, of 1024 requests 11.9
// and 13.1; 4096 of 64 requests 14.3 and 11.4, 4000 of 4000 requests 33 and 27.
constexpr uint32_t PLAN_ONE = 2048;
__global__ __launch_bounds__(1024) void k_plan_one(PlanArgs P) {
    plan_scan(P);
    __threadfence_block();
    __syncthreads();
    plan_tokens(P, threadIdx.x, 1024);
}
__global__ __launch_bounds__(1024) void k_plan_scan(PlanArgs P) { plan_scan(P); }
__global__ __launch_bounds__(256) void k_plan_tokens(PlanArgs P) { plan_tokens(P, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256); }

bool block_ok(size_t b) { return b >= 1 && b <= 4096 && (b & (b - 1)) == 0; }

}  // namespace

extern "C" {

int atlas_kv_write(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* k, const atlas_attn_rows_t* v, const int64_t* d_slots, size_t n_tokens,
                   const atlas_kv_cache_t* cache, uint32_t* d_status, void* stream) {
    const char* why = atlas_attn::bad_shape(shape);
    if (!why) why = atlas_attn::bad_sizes(0, n_tokens);
    if (!why) why = atlas_attn::bad_rows(k, n_tokens, shape->n_kv_heads, shape->head_dim);
    if (!why) why = atlas_attn::bad_rows(v, n_tokens, shape->n_kv_heads, shape->head_dim);
    if (!why) why = atlas_attn::bad_cache(cache);
    if (!why && ((n_tokens && !d_slots) || (uintptr_t)d_slots % 8)) why = "kv_write: slots are null or not 8-byte aligned";
    if (!why && (uintptr_t)d_status % 4) why = "kv_write: status must be 4-byte aligned";
    if (why) return fail(ATLAS_EINVAL, why);
    if (!n_tokens) return ATLAS_OK;
    atlas_attn::Launch L;
    if (int rc = L.begin(stream)) return rc;
    if (int rc = L.on_device({k->d, v->d, d_slots, cache->d_k, cache->d_v, d_status})) return rc;
    WriteArgs W{k->d, v->d, (int64_t)k->token_stride, (int64_t)k->head_stride, (int64_t)v->token_stride, (int64_t)v->head_stride, d_slots, cache->d_k, cache->d_v, d_status,
                (uint32_t)n_tokens, (uint32_t)shape->n_kv_heads, (uint32_t)shape->head_dim, log2_of(cache->block_size), (int64_t)(cache->n_blocks * cache->block_size)};
    const uint64_t n = (uint64_t)n_tokens * W.KV * ((W.d + 3) / 4);
    const unsigned grid = (unsigned)std::min<uint64_t>((n + 255) / 256, 256 * 16);
    if (cache->bits == 16) k_kv_write<int16_t><<<grid, 256, 0, L.stream>>>(W);
    else k_kv_write<int32_t><<<grid, 256, 0, L.stream>>>(W);
    return L.end();
}

size_t atlas_kv_plan_workspace(size_t n_seqs, size_t max_tokens) {
    return atlas_attn::bad_sizes(n_seqs, max_tokens) ? 0 : 16 + 4 * n_seqs;
}

int atlas_kv_plan(size_t block_size, size_t n_blocks, const int32_t* d_cached_lens, const int32_t* d_new_lens, size_t n_seqs, int32_t* d_block_table, size_t max_blocks,
                  size_t table_stride, int32_t* d_free_blocks, const int32_t* d_n_free, int32_t* d_n_free_out, int32_t* d_cu_new, int32_t* d_kv_lens, int64_t* d_slots,
                  int32_t* d_positions, size_t max_tokens, uint32_t* d_status, void* d_workspace, size_t workspace_bytes, void* stream) {
    const char* why = atlas_attn::bad_sizes(n_seqs, max_tokens);
    if (!why && !block_ok(block_size)) why = "kv_plan: block_size must be a power of two, at most 4096";
    if (!why && (n_blocks < 1 || n_blocks > 0x7fffffff)) why = "kv_plan: n_blocks must be 1 .. 2^31 - 1";
    if (!why && (max_blocks > 0x7fffffff / block_size || table_stride < max_blocks || table_stride > 0x7fffffff)) why = "kv_plan: table_stride must be at least max_blocks, the keys of a row below 2^31";
    if (!why && ((n_seqs && (!d_cached_lens || !d_new_lens || (max_blocks && !d_block_table) || !d_kv_lens)) || !d_free_blocks || !d_n_free || !d_n_free_out || !d_cu_new || (max_tokens && !d_slots) || !d_status)) why = "kv_plan: null argument";
    if (!why && n_seqs && (d_kv_lens == d_cached_lens || d_kv_lens == d_new_lens)) why = "kv_plan: kv_lens may not be cached_lens or new_lens";
    if (!why && (uintptr_t)d_slots % 8) why = "kv_plan: slots must be 8-byte aligned";
    if (!why && (uintptr_t)d_status % 4) why = "kv_plan: status must be 4-byte aligned";
    if (!why && atlas_attn::unaligned({d_cached_lens, d_new_lens, d_block_table, d_free_blocks, d_n_free, d_n_free_out, d_cu_new, d_kv_lens, d_positions})) why = "kv_plan: int32 arrays must be 4-byte aligned";
    if (!why && (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < atlas_kv_plan_workspace(n_seqs, max_tokens))) why = "kv_plan: workspace is null, unaligned or too small";
    if (why) return fail(ATLAS_EINVAL, why);
    atlas_attn::Launch L;
    if (int rc = L.begin(stream)) return rc;
    if (int rc = L.on_device({d_cached_lens, d_new_lens, d_block_table, d_free_blocks, d_n_free, d_n_free_out, d_cu_new, d_kv_lens, d_slots, d_positions, d_status, d_workspace})) return rc;
    PlanArgs P{d_cached_lens, d_new_lens, d_block_table, d_free_blocks, d_n_free_out, d_cu_new, d_kv_lens, d_positions, d_n_free, d_slots, d_status, (uint32_t*)d_workspace,
               (int64_t)table_stride, (uint32_t)n_seqs, (uint32_t)max_tokens, log2_of(block_size), (uint32_t)n_blocks, (uint32_t)max_blocks};
    if (max_tokens <= PLAN_ONE) k_plan_one<<<1, 1024, 0, L.stream>>>(P);
    else {
        k_plan_scan<<<1, 1024, 0, L.stream>>>(P);
        k_plan_tokens<<<(unsigned)std::min<size_t>((max_tokens + 255) / 256, 2048), 256, 0, L.stream>>>(P);
    }
    return L.end();
}

}  // extern "C"
