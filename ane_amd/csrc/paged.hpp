// paged.hpp -- the paged K/V cache (ane_decode.h) as its kernels see it: host
// checks, the lookups that keep a broken table inside the pool, activations
// eight at a time.
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

// Eight activations from element i on, 16-byte aligned.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
template <class T>
__device__ __forceinline__ void load8(const void* p, uint64_t i, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const h8 a = *reinterpret_cast<const h8*>(static_cast<const _Float16*>(p) + i);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)a[e];
    }
}
template <class T>
__device__ __forceinline__ void store8(void* p, uint64_t i, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        float* o = static_cast<float*>(p) + i;
        *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(o + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        h8 a;
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] = (_Float16)x[e];
        *reinterpret_cast<h8*>(static_cast<_Float16*>(p) + i) = a;
    }
}

}  // namespace ane
