// paged_attention.hip -- attention over the paged K/V cache: causal prompts and
// batches of single tokens.
#include <math.h>

#include "paged.hpp"

namespace ane {
namespace {

struct AttnArgs {
    const void* q;
    void* out;
    const uint16_t *kp, *vp;  // this layer's pages
    const uint32_t *table, *kv_len, *seqs, *q_start;
    uint64_t q_stride, out_stride;
    uint32_t n, n_tokens, n_heads, n_kv, ps, n_pages, max_pages, n_seqs;
    float scale;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One wave per (token, head): the lane holds hd/64 of the dimensions, keys one
// after the other with the running maximum and sum.
template <class T, int HD>
__global__ void __launch_bounds__(64) k_attn_simple(AttnArgs a) {
    constexpr int E = HD / 64;
    const uint32_t t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, g = h / (a.n_heads / a.n_kv);
    uint32_t s = t, first = t, last = t + 1;
    if (a.q_start) {
        s = wave_search(a.n, t, [&](uint32_t i) { return (uint64_t)a.q_start[i]; });
        first = a.q_start[s];
        last = a.q_start[s + 1];
        if (t < first || t >= last) return;
    }
    const uint32_t id = a.seqs ? a.seqs[s] : s;
    int64_t seen = 0;
    if (id < a.n_seqs)
        seen = min((int64_t)a.kv_len[id], (int64_t)a.max_pages * a.ps) - (int64_t)(last - 1 - t);
    float q[E], o[E] = {};
    for (int e = 0; e < E; e++)
        q[e] = (float)static_cast<const T*>(a.q)[t * a.q_stride + h * HD + lane * E + e] * a.scale;
    float m = -INFINITY, l = 0.0f;
    for (int64_t j = 0; j < seen; j++) {
        const uint32_t page = a.table[(uint64_t)id * a.max_pages + j / a.ps];
        float k[E] = {}, v[E] = {};
        if (page < a.n_pages) {
            const uint64_t at = (((uint64_t)page * a.n_kv + g) * a.ps + j % a.ps) * HD + lane * E;
            for (int e = 0; e < E; e++) k[e] = half_bits_to_float(a.kp[at + e]), v[e] = half_bits_to_float(a.vp[at + e]);
        }
        float d = 0.0f;
        for (int e = 0; e < E; e++) d += q[e] * k[e];
        d = wave_sum(d);
        const float mn = fmaxf(m, d), w = expf(m - mn), p = expf(d - mn);
        l = l * w + p;
        for (int e = 0; e < E; e++) o[e] = o[e] * w + p * v[e];
        m = mn;
    }
    for (int e = 0; e < E; e++)
        static_cast<T*>(a.out)[t * a.out_stride + h * HD + lane * E + e] = (T)(seen > 0 ? o[e] / l : 0.0f);
}

int attention_status(const ane_paged_cache* c, uint32_t layer, uint32_t n, uint32_t n_tokens, int type, const void* q,
                     uint64_t q_stride, float scale, const void* out, uint64_t out_stride) {
    const int st = cache_status(c);
    if (st) return st;
    const uint32_t size = type == ANE_TYPE_F32 ? 4 : 2;
    const uint64_t width = (uint64_t)c->n_heads * c->head_dim;
    if (layer >= c->n_layers || n_tokens > kMaxTokens || n > kMaxTokens ||
        (type != ANE_TYPE_F32 && type != ANE_TYPE_F16) || !(scale > 0.0f) || !isfinite(scale))
        return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    if (!q || !out) return ANE_ERR_BAD_POINTER;
    if ((((uintptr_t)q) | ((uintptr_t)out)) & 15 || (q_stride * size) & 15 || (out_stride * size) & 15 ||
        q_stride < width || out_stride < width)
        return ANE_ERR_INVALID_ARG;
    return ANE_OK;
}

int simple_launch(const ane_paged_cache* c, uint32_t layer, const uint32_t* seqs, uint32_t n, const uint32_t* q_start,
                  uint32_t n_tokens, int type, const void* q, uint64_t q_stride, float scale, void* out,
                  uint64_t out_stride, void* stream) {
    AttnArgs a;
    const uint64_t lo = page_elems(c) * c->n_pages * layer;
    a.q = q, a.out = out, a.kp = c->k_pages + lo, a.vp = c->v_pages + lo;
    a.table = c->page_table, a.kv_len = c->kv_len, a.seqs = seqs, a.q_start = q_start;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.n = n, a.n_tokens = n_tokens, a.n_heads = c->n_heads, a.n_kv = c->n_kv_heads, a.ps = c->page_size;
    a.n_pages = c->n_pages, a.max_pages = c->max_pages, a.n_seqs = c->n_seqs, a.scale = scale;
    auto* f = type == ANE_TYPE_F32 ? (c->head_dim == 64 ? k_attn_simple<float, 64> : k_attn_simple<float, 128>)
                                   : (c->head_dim == 64 ? k_attn_simple<_Float16, 64> : k_attn_simple<_Float16, 128>);
    hipLaunchKernelGGL(f, dim3(n_tokens, c->n_heads), dim3(64), 0, (hipStream_t)stream, a);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

}  // namespace
}  // namespace ane

using namespace ane;

extern "C" size_t ane_hip_attention_prompt_workspace_size(const ane_paged_cache* cache, uint32_t n, uint32_t n_tokens,
                                                          uint32_t max_len) {
    return 0;
}

extern "C" int ane_hip_attention_prompt(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                        const uint32_t* q_start, uint32_t n_tokens, uint32_t max_len, int type,
                                        const void* q, uint64_t q_stride, float scale, void* out, uint64_t out_stride,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    const int st = attention_status(cache, layer, n, n_tokens, type, q, q_stride, scale, out, out_stride);
    if (st) return st;
    if (!q_start && n_tokens != n) return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    return simple_launch(cache, layer, seqs, n, q_start, n_tokens, type, q, q_stride, scale, out, out_stride, stream);
}

extern "C" size_t ane_hip_attention_shared_workspace_size(const ane_paged_cache* cache, uint32_t n, uint32_t n_groups,
                                                          uint32_t max_prefix, uint32_t max_len) {
    return 0;
}

extern "C" int ane_hip_attention_shared(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                        uint32_t n_groups, const uint32_t* group_start, const uint32_t* prefix_len,
                                        uint32_t max_prefix, uint32_t max_len, int type, const void* q,
                                        uint64_t q_stride, float scale, void* out, uint64_t out_stride, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const int st = attention_status(cache, layer, n, n, type, q, q_stride, scale, out, out_stride);
    if (st || n == 0) return st;
    if (n_groups > n) return ANE_ERR_INVALID_ARG;
    if (n_groups && (!group_start || !prefix_len)) return ANE_ERR_BAD_POINTER;
    return simple_launch(cache, layer, seqs, n, nullptr, n, type, q, q_stride, scale, out, out_stride, stream);
}
