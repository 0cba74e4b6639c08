// paged.hpp -- the paged K/V cache (ane_decode.h) as its kernels see it:
// host checks, and the lookups that keep a broken table inside the pool.
#pragma once

#include "../../include/ane_decode.h"
#include "common.hpp"

namespace ane {

constexpr uint32_t kMaxTokens = 1u << 23;     // rows of a packed batch
constexpr uint32_t kMaxRequests = 1u << 16;   // sequences or pages named in one call

inline uint64_t page_cap(const ane_paged_cache* c) { return (uint64_t)c->max_pages * c->page_size; }
inline uint64_t page_elems(const ane_paged_cache* c) { return (uint64_t)c->n_kv_heads * c->page_size * c->head_dim; }

// ANE_OK, or what is wrong with the cache's description (nothing on the device is read).
inline int cache_status(const ane_paged_cache* c) {
    if (!c) return ANE_ERR_BAD_POINTER;
    if (c->n_layers == 0 || c->n_kv_heads == 0 || c->n_heads == 0 || c->n_heads % c->n_kv_heads != 0 ||
        c->n_heads / c->n_kv_heads > 128 || c->n_kv_heads > 4096 || (c->head_dim != 64 && c->head_dim != 128) ||
        c->page_size == 0 || c->page_size % 16 != 0 || c->page_size > (1u << 20) || c->n_pages == 0 ||
        c->n_pages >= (1u << 31) || c->n_seqs == 0 || c->n_seqs >= (1u << 31) || c->max_pages == 0 ||
        page_cap(c) > (1ull << 30))
        return ANE_ERR_INVALID_ARG;
    if (!c->k_pages || !c->v_pages || !c->page_table || !c->kv_len) return ANE_ERR_BAD_POINTER;
    if ((((uintptr_t)c->k_pages) | ((uintptr_t)c->v_pages)) & 15) return ANE_ERR_INVALID_ARG;
    if ((((uintptr_t)c->page_table) | ((uintptr_t)c->kv_len) | ((uintptr_t)c->page_refs)) & 3) return ANE_ERR_INVALID_ARG;
    return ANE_OK;
}

// Largest s in [0, n) with key(s) <= x, by one whole wave (key ascending,
// key(0) <= x): 64 probes a step, so one load up to 64 entries and two up to
// 4096.  Any other key still ends, with some s in [0, n).
template <class Key>
__device__ __forceinline__ uint32_t wave_search(uint32_t n, uint64_t x, Key key) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, len = n;
    while (len > 1) {
        const uint32_t step = (len + 63) / 64, i = lane * step;
        const bool le = i < len && key(lo + i) <= x;
        const uint64_t m = __ballot(le);
        const uint32_t c = m ? 63 - (uint32_t)__builtin_clzll(m) : 0;
        lo += c * step;
        len = min(step, len - c * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace ane
