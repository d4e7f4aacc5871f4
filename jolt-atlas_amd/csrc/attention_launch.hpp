// Argument checks and the launch scope that the entry points of the quantised attention share (attention.hip, paging.hip).
#pragma once
#include <algorithm>
#include <initializer_list>

#include "runtime.hpp"

namespace atlas_attn {
using atlas_rt::fail;
using atlas_rt::rt;

constexpr size_t MAX_HEADS = 1024, MAX_DIM = 256, MAX_BLOCK = 4096, MAX_TOKENS = (size_t)1 << 30, MAX_SEQS = (size_t)1 << 24;

inline const char* bad_shape(const atlas_attn_shape_t* s) {
    if (!s) return "attention: shape is null";
    if (s->n_heads < 1 || s->n_heads > MAX_HEADS || s->n_kv_heads < 1 || s->n_kv_heads > s->n_heads || s->n_heads % s->n_kv_heads) return "attention: n_kv_heads must divide n_heads (1 .. 1024)";
    if (s->head_dim < 1 || s->head_dim > MAX_DIM) return "attention: head_dim must be 1 .. 256";
    if (s->score_mul < 1 || s->score_mul > (1 << 14)) return "attention: score_mul must be 1 .. 2^14";
    if (s->causal != 0 && s->causal != 1) return "attention: causal must be 0 or 1";
    return nullptr;
}
// strides cannot make two heads of a row overlap, and offsets stay in 63 bits
inline const char* bad_rows(const atlas_attn_rows_t* r, size_t n_tokens, size_t heads, size_t dim) {
    if (!r || (!r->d && n_tokens)) return "attention: rows are null";
    if ((uintptr_t)r->d % 4) return "attention: rows must be 4-byte aligned";
    if (r->token_stride > ((size_t)1 << 32) || r->head_stride > ((size_t)1 << 32)) return "attention: strides must be at most 2^32";
    if ((heads > 1 && r->head_stride < dim) || (n_tokens > 1 && r->token_stride < dim)) return "attention: strides must be at least head_dim";
    return nullptr;
}
// rows that are written: no two of them may share an element
inline const char* bad_out(const atlas_attn_rows_t* r, size_t n_tokens, size_t heads, size_t dim) {
    const size_t inner = (heads - 1) * r->head_stride + dim, outer = n_tokens ? (n_tokens - 1) * r->token_stride + dim : 0;
    if (n_tokens > 1 && heads > 1 && r->token_stride < inner && r->head_stride < outer) return "attention: rows of out overlap";
    return nullptr;
}
inline const char* bad_cache(const atlas_kv_cache_t* c) {
    if (!c || !c->d_k || !c->d_v) return "attention: cache is null";
    if (c->bits != 16 && c->bits != 32) return "attention: a cache has 16 or 32 bits";
    if ((uintptr_t)c->d_k % (c->bits / 8) || (uintptr_t)c->d_v % (c->bits / 8)) return "attention: cache alignment";
    if (c->block_size < 1 || c->block_size > MAX_BLOCK || (c->block_size & (c->block_size - 1))) return "attention: block_size must be a power of two, at most 4096";
    if (c->n_blocks < 1 || c->n_blocks > 0x7fffffff) return "attention: n_blocks must be 1 .. 2^31 - 1";
    return nullptr;
}
inline bool unaligned(std::initializer_list<const void*> ps) {          // int32 arrays
    for (const void* p : ps) if ((uintptr_t)p % 4) return true;
    return false;
}
inline const char* bad_mask(const atlas_attn_shape_t* s, const atlas_attn_mask_t* m) {
    if (!m || !m->d_status || unaligned({m->d_status})) return "attention: mask or its status is null or not 4-byte aligned";
    if (m->n_tokens < 1 || m->n_tokens > 0x7fffffff) return "attention: a mask's n_tokens must be 1 .. 2^31 - 1";
    if (!s->causal) return "attention: a graph's mask is causal";
    return nullptr;
}
inline uint32_t log2_of(size_t v) { uint32_t l = 0; while (((size_t)1 << l) < v) l++; return l; }

// Enqueues on the caller's stream, or on the library's: that one under its lock (another thread's pipeline may have it on a lane).  The calling thread's
// current device is the runtime's for the length of the call (the caller may have moved on to another since atlas_init).
struct Launch {
    std::unique_lock<atlas_rt::Mutex> lk;
    hipStream_t stream = nullptr;
    int back = -1;
    int begin(void* user) {
        NEED_INIT();
        int dev = -1;
        HIP_TRY(hipGetDevice(&dev));
        if (dev != rt().device) { HIP_TRY(hipSetDevice(rt().device)); back = dev; }
        if (!user) { lk = std::unique_lock<atlas_rt::Mutex>(rt().mu); stream = rt().stream; }
        else stream = user == ATLAS_STREAM_DEFAULT ? nullptr : (hipStream_t)user;
        (void)hipGetLastError();          // of an earlier call of the caller's: end() is to tell of these launches
        return ATLAS_OK;
    }
    // every pointer must be memory of the runtime's device (managed and pinned host memory that the device maps is refused too: the kernels are
    // written for HBM).  A pointer that HIP does not know would fault the GPU; the look-up costs a fraction of a microsecond.
    int on_device(std::initializer_list<const void*> ps) {
        for (const void* p : ps) {
            if (!p) continue;
            hipPointerAttribute_t at{};
            const hipError_t e = hipPointerGetAttributes(&at, p);
            if (e != hipSuccess) { (void)hipGetLastError(); return fail(ATLAS_EINVAL, "attention: a pointer is not device memory"); }
            if (at.type != hipMemoryTypeDevice || at.device != rt().device) return fail(ATLAS_EINVAL, "attention: a pointer is not memory of the runtime's device");
        }
        return ATLAS_OK;
    }
    int end() { HIP_TRY(hipGetLastError()); return ATLAS_OK; }
    ~Launch() { if (back >= 0) (void)hipSetDevice(back); }
};
inline const char* bad_sizes(size_t n_seqs, size_t n_tokens) {
    return n_seqs > MAX_SEQS ? "attention: more than 2^24 sequences" : n_tokens > MAX_TOKENS ? "attention: more than 2^30 tokens" : nullptr;
}
// the query rows of a sequence under one kv head are counted in 32 bits, and so are the up to 255 places of a tile behind its last one
inline const char* bad_count(const atlas_attn_shape_t* s, size_t n_tokens) {
    return n_tokens * (s->n_heads / s->n_kv_heads) > 0xffffff00 ? "attention: more than 2^32 - 256 query rows to a kv head" : nullptr;
}

}  // namespace atlas_attn
