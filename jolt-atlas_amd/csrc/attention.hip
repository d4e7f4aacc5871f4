// Quantised attention for generation (include/atlas_hip.h: atlas_attn_*, atlas_kv_write): the attention of a model graph in the graph executor's integers, over packed
// prompts and over a paged cache.  Mathematics at the kernels (attention_kernels.hip.h).
#include "runtime.hpp"

#include "attention_kernels.hip.h"
#include "attention_launch.hpp"
#include "attention_split.hip.h"
#include "attention_tile.hip.h"

namespace {

using namespace atlas_attn;

Rows rows_of(const atlas_attn_rows_t* r) { return Rows{r->d, (int64_t)r->token_stride, (int64_t)r->head_stride}; }
Args args_of(const atlas_attn_shape_t* s, const atlas_attn_rows_t* q, const int32_t* cu, size_t n_seqs, size_t n_tokens, const atlas_attn_rows_t* out,
             const atlas_attn_mask_t* mask) {
    Args A{};
    A.q = rows_of(q); A.out = rows_of(out);
    A.cu = cu; A.n_seqs = (uint32_t)n_seqs; A.n_tokens = (uint32_t)n_tokens;
    A.H = (uint32_t)s->n_heads; A.KV = (uint32_t)s->n_kv_heads; A.G = A.H / A.KV; A.d = (uint32_t)s->head_dim;
    A.mul = s->score_mul; A.causal = s->causal;
    if (mask) { A.fill = mask->fill; A.graph_tokens = mask->n_tokens; A.status = mask->d_status; }
    return A;
}

// head sizes are padded to the fragments of the tile kernel
int padded_dim(size_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }
// f(padded dims, waves to a row)
template <class F>
auto with_shape(int dp, bool few, F f) {
    auto go = [&](auto d) {
        constexpr int DP = decltype(d)::value;
        if (few) return f(d, std::integral_constant<int, tile_split(DP, true)>{});
        return f(d, std::integral_constant<int, tile_split(DP, false)>{});
    };
    switch (dp) {
        case 32: return go(std::integral_constant<int, 32>{});
        case 64: return go(std::integral_constant<int, 64>{});
        case 128: return go(std::integral_constant<int, 128>{});
        default: return go(std::integral_constant<int, 256>{});
    }
}

// the digit planes and the held e of the tile kernel in a workspace; cached_keys = 0: packed prompts
struct PlanesLayout {
    bool few;
    size_t max_keys, tiles, per_seq, held, work, wgs, v_at, mag_at, there_at, next_at, e_at, bytes;
    PlanesLayout(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t cached_keys) {
        const size_t slack = 4;                                        // a step reads up to 4 tiles: its last ones may lie behind a sequence's end
        const int dp = padded_dim(s->head_dim);
        const size_t G = s->n_heads / s->n_kv_heads, usual = with_shape(dp, false, [](auto d, auto w) { return TileShape<decltype(d)::value, decltype(w)::value>::ROWS; });
        few = (n_tokens * G / usual + n_seqs) * s->n_kv_heads < (dp <= 64 ? 512 : 192);
        const size_t rows = with_shape(dp, few, [](auto d, auto w) { return TileShape<decltype(d)::value, decltype(w)::value>::ROWS; });
        per_seq = (cached_keys + 31) / 32;
        max_keys = cached_keys ? cached_keys : n_tokens;
        tiles = (cached_keys ? n_seqs * per_seq : n_tokens / 32 + n_seqs) + slack;
        held = std::min<size_t>((max_keys + 127) / 128 * 128, HELD);
        work = (n_tokens * G / rows + n_seqs) * s->n_kv_heads;
        wgs = std::min<size_t>(work, TILE_WGS);
        const size_t one = tiles * s->n_kv_heads * (size_t)(dp / 32) * FRAGMENT;
        v_at = one;
        mag_at = 2 * one;
        there_at = mag_at + 8 * tiles * s->n_kv_heads;
        next_at = there_at + 4 * tiles;
        e_at = (next_at + 32 + 15) / 16 * 16;
        bytes = e_at + wgs * rows * held * 2;
    }
    Planes at(void* ws, const atlas_attn_shape_t* s) const {
        uint8_t* w = (uint8_t*)ws;
        return Planes{w, w + v_at, (uint32_t*)(w + mag_at), (uint32_t*)(w + mag_at) + tiles * s->n_kv_heads, (uint32_t*)(w + there_at), w + e_at, (uint32_t*)(w + next_at), (uint32_t)tiles, (uint32_t)per_seq};
    }
};
template <class CT>
int launch_tiles(const Args& A, const PlanesLayout& L, const Planes& P, hipStream_t stream) {
    return with_shape(padded_dim(A.d), L.few, [&](auto dim, auto split) -> int {
        constexpr int DP = decltype(dim)::value, SPLIT = decltype(split)::value;
        using T = TileShape<DP, SPLIT>;
        k_attn_planes<CT, DP><<<dim3((unsigned)L.tiles, A.KV), 256, 0, stream>>>(A, P);
        auto* k = L.max_keys > HELD ? &k_attn_tile<CT, DP, SPLIT, true> : &k_attn_tile<CT, DP, SPLIT, false>;
        if (T::LDS > 65536) HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS));
        k<<<(unsigned)L.wgs, 256, T::LDS, stream>>>(A, P, (uint32_t)L.work, (uint32_t)L.held);
        return ATLAS_OK;
    });
}
// On average more than 96 query rows to a sequence and kv head: tiles; below, 16 rows at a time that read the cache themselves.  One MI355X, int32, 64 sequences of 2000
// keys: 32 heads of 128 over 8, 16 new tokens (64 rows) 820 us in tiles and 833 us in 16 rows, 32 new tokens 961 and 1599 us; 16 heads of 64, 32 new
// tokens (32 rows) 1346 and 581 us.  The host knows no sequence's own rows: where a few have many and many have few, all go one way (a chunk of 2000 tokens beside 63 single
// tokens over up to 8191 keys, 32 heads of 128 over 8: 1774 us in one call, 256 + 647 in two).
bool many_rows(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens) { return n_tokens * (s->n_heads / s->n_kv_heads) > 96 * n_seqs; }
// Few rows: the workspace of the split path
struct SplitLayout {
    Split S{};
    size_t bytes;
    SplitLayout(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t max_keys, void* ws) {
        const size_t G = s->n_heads / s->n_kv_heads, tiles = n_tokens * G / TILE_ROWS + n_seqs, rows = n_tokens * s->n_heads, parts = WGS * TILE_ROWS + rows, mags = WGS + tiles * s->n_kv_heads;
        const size_t pitch = (max_keys + 63) / 64 * 64;
        size_t at = 0;
        auto take = [&](size_t n) { const size_t was = at; at += (n + 15) / 16 * 16; return (uint8_t*)ws + was; };
        S.n_tiles = (uint32_t)tiles; S.n_rows = (uint32_t)rows; S.pitch = (int64_t)pitch;
        S.scores = (int32_t*)take(rows * pitch * 4);
        S.part = (int64_t*)take(parts * s->head_dim * 8);
        S.cmax = (int32_t*)take(parts * 4);
        S.csum = (uint32_t*)take(parts * 4);
        S.q_mag = (uint32_t*)take(mags * 4);
        S.k_mag = (uint32_t*)take(mags * 4);
        S.v_mag = (uint32_t*)take(mags * 4);
        S.units = (uint32_t*)take((tiles + 1) * 4);
        S.rows = (uint32_t*)take((tiles + 1) * 4);
        bytes = at + 16;
    }
};
// f(steps of 64 dims, FAST)
template <class CT, class F>
void with_steps(const Args& A, F f) {
    auto dims = [&](auto fast) {
        switch ((A.d + 63) / 64) {
            case 1: f(std::integral_constant<int, 1>{}, fast); break;
            case 2: f(std::integral_constant<int, 2>{}, fast); break;
            default: f(std::integral_constant<int, 4>{}, fast);
        }
    };
    if (A.d % 4 == 0 && (!A.table || A.log_block >= 4)) dims(std::true_type{}); else dims(std::false_type{});
}
template <class CT>
int launch_split(const Args& A, const SplitLayout& L, hipStream_t stream) {
    k_split_plan<<<1, 1024, 0, stream>>>(A, L.S);
    with_steps<CT>(A, [&](auto ks, auto fast) {
        k_split_scores<CT, decltype(ks)::value, decltype(fast)::value><<<WGS, 256, 0, stream>>>(A, L.S);
        k_split_sums<<<WGS, 256, 0, stream>>>(A, L.S);
        k_split_values<CT, decltype(ks)::value, decltype(fast)::value><<<WGS, 256, 0, stream>>>(A, L.S);
    });
    if (L.S.n_rows < 512) k_split_join<CT, 1024><<<L.S.n_rows, 1024, 0, stream>>>(A, L.S, (uint32_t)padded_dim(A.d));
    else k_split_join<CT, 256><<<L.S.n_rows, 256, 0, stream>>>(A, L.S, (uint32_t)padded_dim(A.d));
    return ATLAS_OK;
}

// One launch while LDS holds the scores.  Few rows: up to 1024 keys, beyond that where there are workgroups enough for the chip (16 heads of 64, one token over
// 1000 / 2000 keys: 28 / 42 us in one launch of 16 workgroups, 32 / 33 us in the split path's five; 16 such tokens over 2000 keys: 56 and 80 us; the rule does not
// go by the heads: one token of 32 heads of 128 over 8 and 1000 keys takes 43 us in its 8 workgroups, 39 in five launches).  Many rows: while
// the 16-row workgroups fit the chip about once (16 heads of 64, a prompt of 512: 39 us and 55 us in tiles, of 1024: 92 and 85 us).
bool fused(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t max_keys, bool many) {
    const size_t wgs = (n_tokens * (s->n_heads / s->n_kv_heads) / TILE_ROWS + n_seqs) * s->n_kv_heads;
    if (max_keys > fused_keys(s->head_dim)) return false;
    return many ? wgs <= 640 : max_keys <= 1024 || wgs >= 256;
}
enum class Path { FUSED, TILES, SPLIT };
Path path_of(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t max_keys, bool many) {
    if (!n_seqs || !n_tokens) return Path::FUSED;                  // nothing is launched, nothing is needed
    return fused(s, n_seqs, n_tokens, max_keys, many) ? Path::FUSED : many ? Path::TILES : Path::SPLIT;
}
// What a path's launches and 32-bit counters hold: a launch has fewer than 2^32 threads
const char* too_many(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t max_keys, bool cached, Path path) {
    const size_t row_tiles = n_tokens * (s->n_heads / s->n_kv_heads) / TILE_ROWS + n_seqs, launch = 0xffffffff;
    bool over;
    if (path == Path::FUSED) over = row_tiles * s->n_kv_heads > launch / (FUSED_WAVES * 64);
    else if (path == Path::TILES) {
        const PlanesLayout L(s, n_seqs, n_tokens, cached ? std::max<size_t>(max_keys, 1) : 0);
        over = L.work > 0x7fffffff || L.tiles > launch / 256;
    } else {
        const size_t units = (max_keys + UNIT - 1) / UNIT;
        over = n_tokens * s->n_heads > launch / 256 || row_tiles * s->n_kv_heads > 0x40000000 || row_tiles * s->n_kv_heads * units > 0x7fffffff;
    }
    return over ? "attention: too many sequences, rows or keys for one call" : nullptr;
}
// What a call over a cache needs
size_t cached_bytes(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t max_keys, Path path) {
    if (path == Path::FUSED) return 16;
    return path == Path::TILES ? PlanesLayout(s, n_seqs, n_tokens, std::max<size_t>(max_keys, 1)).bytes : SplitLayout(s, n_seqs, n_tokens, max_keys, nullptr).bytes;
}
// The most that one of at most so many sequences, tokens and keys needs: a smaller one may take another path, and the one launch needs nothing.  Each layout grows with its
// arguments, so the largest call that can take the path stands for all: the split path has up to 96 rows to a sequence, tiles the fewest sequences.
size_t most_bytes(const atlas_attn_shape_t* s, size_t n_seqs, size_t n_tokens, size_t max_keys) {
    const size_t G = s->n_heads / s->n_kv_heads, tokens = std::min(n_tokens, 96 * n_seqs / G), seqs = n_tokens ? std::min(n_seqs, (n_tokens * G - 1) / 96) : 0;
    size_t most = 16;
    if (tokens && !fused(s, 1, 1, max_keys, false)) most = std::max(most, cached_bytes(s, n_seqs, tokens, max_keys, Path::SPLIT));
    if (seqs && !fused(s, seqs, n_tokens, max_keys, true)) most = std::max(most, cached_bytes(s, seqs, n_tokens, max_keys, Path::TILES));
    return most;
}
template <class CT>
int launch_fused(const Args& A, size_t max_keys, hipStream_t stream) {
    const uint64_t wgs = ((uint64_t)A.n_tokens * A.G / TILE_ROWS + A.n_seqs) * A.KV;
    int rc = ATLAS_OK;
    with_steps<CT>(A, [&](auto ks, auto fast) {
        constexpr int KS = decltype(ks)::value;
        auto* k = &k_attn_fused<CT, KS, decltype(fast)::value>;
        const size_t lds = fused_lds(max_keys, KS);
        if (lds > 65536 - 6144 && hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) { rc = fail(ATLAS_ENODEV, "attention: LDS"); return; }
        k<<<(unsigned)wgs, FUSED_WAVES * 64, lds, stream>>>(A, (uint32_t)fused_pitch(max_keys));
    });
    return rc;
}

int attn_prompt(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* q, const atlas_attn_rows_t* k, const atlas_attn_rows_t* v,
                const int32_t* d_cu_seqlens, size_t n_seqs, size_t n_tokens, const atlas_attn_rows_t* out,
                const atlas_attn_mask_t* mask, void* d_workspace, size_t workspace_bytes, void* stream) {
    const char* why = bad_shape(shape);
    if (!why) why = bad_sizes(n_seqs, n_tokens);
    if (!why) why = bad_count(shape, n_tokens);
    if (!why) why = bad_rows(q, n_tokens, shape->n_heads, shape->head_dim);
    if (!why) why = bad_rows(k, n_tokens, shape->n_kv_heads, shape->head_dim);
    if (!why) why = bad_rows(v, n_tokens, shape->n_kv_heads, shape->head_dim);
    if (!why) why = bad_rows(out, n_tokens, shape->n_heads, shape->head_dim);
    if (!why) why = bad_out(out, n_tokens, shape->n_heads, shape->head_dim);
    if (!why && n_tokens && (out->d == q->d || out->d == k->d || out->d == v->d)) why = "attn_prompt: out may not be q, k or v";
    if (!why && n_seqs && n_tokens && !d_cu_seqlens) why = "attn_prompt: cu_seqlens is null";
    if (!why && unaligned({d_cu_seqlens})) why = "attn_prompt: cu_seqlens must be 4-byte aligned";
    const Path path = why ? Path::FUSED : path_of(shape, n_seqs, n_tokens, n_tokens, true);
    if (!why) why = too_many(shape, n_seqs, n_tokens, n_tokens, false, path);
    if (!why && (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < atlas_attn_prompt_workspace(shape, n_seqs, n_tokens))) why = "attn_prompt: workspace is null, unaligned or too small";
    if (!why && mask) why = bad_mask(shape, mask);
    if (why) return fail(ATLAS_EINVAL, why);
    if (!n_seqs || !n_tokens) return ATLAS_OK;
    Launch L;
    if (int rc = L.begin(stream)) return rc;
    if (int rc = L.on_device({q->d, k->d, v->d, d_cu_seqlens, out->d, d_workspace, mask ? mask->d_status : nullptr})) return rc;
    Args A = args_of(shape, q, d_cu_seqlens, n_seqs, n_tokens, out, mask);
    A.k = rows_of(k); A.v = rows_of(v);
    if (path == Path::FUSED) {
        if (int rc = launch_fused<int32_t>(A, n_tokens, L.stream)) return rc;
        return L.end();
    }
    const PlanesLayout P(shape, n_seqs, n_tokens, 0);
    if (int rc = launch_tiles<int32_t>(A, P, P.at(d_workspace, shape), L.stream)) return rc;
    return L.end();
}

int attn_cached(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* q, const int32_t* d_cu_new, const int32_t* d_kv_lens, size_t n_seqs, size_t n_tokens,
                const atlas_kv_cache_t* cache, const int32_t* d_block_table, size_t max_blocks, size_t table_stride, const atlas_attn_rows_t* out,
                const atlas_attn_mask_t* mask, void* d_workspace, size_t workspace_bytes, void* stream) {
    const char* why = bad_shape(shape);
    if (!why) why = bad_sizes(n_seqs, n_tokens);
    if (!why) why = bad_count(shape, n_tokens);
    if (!why) why = bad_rows(q, n_tokens, shape->n_heads, shape->head_dim);
    if (!why) why = bad_rows(out, n_tokens, shape->n_heads, shape->head_dim);
    if (!why) why = bad_out(out, n_tokens, shape->n_heads, shape->head_dim);
    if (!why) why = bad_cache(cache);
    if (!why && n_tokens && out->d == q->d) why = "attn_cached: out may not be q";
    if (!why && n_seqs && n_tokens && (!d_cu_new || !d_kv_lens || (max_blocks && !d_block_table))) why = "attn_cached: cu_new, kv_lens or block_table is null";
    if (!why && unaligned({d_cu_new, d_kv_lens, d_block_table})) why = "attn_cached: cu_new, kv_lens and block_table must be 4-byte aligned";
    if (!why && (max_blocks > 0x7fffffff / cache->block_size || table_stride < max_blocks || table_stride > 0x7fffffff)) why = "attn_cached: table_stride must be at least max_blocks, the keys of a row below 2^31";
    const Path path = why ? Path::FUSED : path_of(shape, n_seqs, n_tokens, max_blocks * cache->block_size, many_rows(shape, n_seqs, n_tokens));
    if (!why) why = too_many(shape, n_seqs, n_tokens, max_blocks * cache->block_size, true, path);
    if (!why && (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < cached_bytes(shape, n_seqs, n_tokens, max_blocks * cache->block_size, path))) why = "attn_cached: workspace is null, unaligned or too small";
    if (!why && mask) why = bad_mask(shape, mask);
    if (why) return fail(ATLAS_EINVAL, why);
    if (!n_seqs || !n_tokens) return ATLAS_OK;
    Launch L;
    if (int rc = L.begin(stream)) return rc;
    if (int rc = L.on_device({q->d, d_cu_new, d_kv_lens, cache->d_k, cache->d_v, d_block_table, out->d, d_workspace, mask ? mask->d_status : nullptr})) return rc;
    Args A = args_of(shape, q, d_cu_new, n_seqs, n_tokens, out, mask);
    // a table without columns (nothing is cached, its array may be empty) is never looked at
    A.ck = cache->d_k; A.cv = cache->d_v; A.lens = d_kv_lens; A.table = max_blocks ? d_block_table : d_kv_lens; A.table_stride = (int64_t)table_stride;
    A.n_blocks = (uint32_t)cache->n_blocks; A.log_block = log2_of(cache->block_size); A.max_keys = (uint32_t)(max_blocks * cache->block_size);
    if (path == Path::FUSED) {
        if (int rc = cache->bits == 16 ? launch_fused<int16_t>(A, A.max_keys, L.stream) : launch_fused<int32_t>(A, A.max_keys, L.stream)) return rc;
        return L.end();
    }
    if (path == Path::TILES) {
        const PlanesLayout P(shape, n_seqs, n_tokens, std::max<size_t>(A.max_keys, 1));
        if (int rc = cache->bits == 16 ? launch_tiles<int16_t>(A, P, P.at(d_workspace, shape), L.stream) : launch_tiles<int32_t>(A, P, P.at(d_workspace, shape), L.stream)) return rc;
        return L.end();
    }
    const SplitLayout P(shape, n_seqs, n_tokens, A.max_keys, d_workspace);
    if (int rc = cache->bits == 16 ? launch_split<int16_t>(A, P, L.stream) : launch_split<int32_t>(A, P, L.stream)) return rc;
    return L.end();
}

}  // namespace

extern "C" {

size_t atlas_attn_prompt_workspace(const atlas_attn_shape_t* shape, size_t n_seqs, size_t n_tokens) {
    if (bad_shape(shape) || bad_sizes(n_seqs, n_tokens) || bad_count(shape, n_tokens)) return 0;
    const Path path = path_of(shape, n_seqs, n_tokens, n_tokens, true);
    if (too_many(shape, n_seqs, n_tokens, n_tokens, false, path)) return 0;
    return path == Path::FUSED ? 16 : PlanesLayout(shape, n_seqs, n_tokens, 0).bytes;
}

int atlas_attn_prompt(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* q, const atlas_attn_rows_t* k, const atlas_attn_rows_t* v,
                      const int32_t* d_cu_seqlens, size_t n_seqs, size_t n_tokens, const atlas_attn_rows_t* out, void* d_workspace, size_t workspace_bytes,
                      void* stream) {
    return attn_prompt(shape, q, k, v, d_cu_seqlens, n_seqs, n_tokens, out, nullptr, d_workspace, workspace_bytes, stream);
}
int atlas_attn_prompt_masked(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* q, const atlas_attn_rows_t* k, const atlas_attn_rows_t* v,
                             const int32_t* d_cu_seqlens, size_t n_seqs, size_t n_tokens, const atlas_attn_rows_t* out, const atlas_attn_mask_t* mask, void* d_workspace, size_t workspace_bytes,
                             void* stream) {
    if (!mask) return fail(ATLAS_EINVAL, "attn_prompt: mask is null");
    return attn_prompt(shape, q, k, v, d_cu_seqlens, n_seqs, n_tokens, out, mask, d_workspace, workspace_bytes, stream);
}

size_t atlas_attn_cached_workspace(const atlas_attn_shape_t* shape, size_t n_seqs, size_t n_tokens, const atlas_kv_cache_t* cache, size_t max_blocks) {
    if (bad_shape(shape) || bad_sizes(n_seqs, n_tokens) || bad_count(shape, n_tokens) || bad_cache(cache) || max_blocks > 0x7fffffff / cache->block_size) return 0;
    const size_t max_keys = max_blocks * cache->block_size;
    const Path path = path_of(shape, n_seqs, n_tokens, max_keys, many_rows(shape, n_seqs, n_tokens));
    if (too_many(shape, n_seqs, n_tokens, max_keys, true, path)) return 0;
    return most_bytes(shape, n_seqs, n_tokens, max_keys);
}

int atlas_attn_cached(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* q, const int32_t* d_cu_new, const int32_t* d_kv_lens, size_t n_seqs, size_t n_tokens,
                      const atlas_kv_cache_t* cache, const int32_t* d_block_table, size_t max_blocks, size_t table_stride, const atlas_attn_rows_t* out,
                      void* d_workspace, size_t workspace_bytes, void* stream) {
    return attn_cached(shape, q, d_cu_new, d_kv_lens, n_seqs, n_tokens, cache, d_block_table, max_blocks, table_stride, out, nullptr, d_workspace, workspace_bytes, stream);
}
int atlas_attn_cached_masked(const atlas_attn_shape_t* shape, const atlas_attn_rows_t* q, const int32_t* d_cu_new, const int32_t* d_kv_lens, size_t n_seqs, size_t n_tokens,
                             const atlas_kv_cache_t* cache, const int32_t* d_block_table, size_t max_blocks, size_t table_stride, const atlas_attn_rows_t* out,
                             const atlas_attn_mask_t* mask, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (!mask) return fail(ATLAS_EINVAL, "attn_cached: mask is null");
    return attn_cached(shape, q, d_cu_new, d_kv_lens, n_seqs, n_tokens, cache, d_block_table, max_blocks, table_stride, out, mask, d_workspace, workspace_bytes, stream);
}

}  // extern "C"
