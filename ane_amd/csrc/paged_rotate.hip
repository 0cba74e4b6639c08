// paged_rotate.hip -- RMSNorm of each q and k head, the position rotation, and
// the append of k and v to the paged cache, in one pass over q, k and v.
//
//   y = x, or (x / sqrt(mean(x^2) + eps)) * w over the head's values
//   pair i of the leading rot_dim values: (a, b) -> (a c - b s, a s + b c),
//   c, s = factor * (cos, sin)(position * freqs[i])
// pairs being neighbours (2i, 2i + 1) or halves (i, i + rot_dim / 2).
//
// The angle is formed and reduced in fp64 and its cosine and sine are rounded
// once, and no table of positions is read.  The fp64 product position * freq is off by at
// most 2^-53 of the angle: nothing beside fp32's rounding up to 2^25 radians, as much
// as one such rounding (6e-8) at 2^29.
#include <algorithm>

#include "paged.hpp"

namespace ane {
namespace {

struct RotateArgs {
    const void *q, *k, *v;
    void* q_out;
    const double* freqs;
    const float *q_norm, *k_norm;
    uint16_t *kp, *vp;  // this layer's pages
    const uint32_t *table, *kv_len, *seqs, *q_start;
    uint64_t q_stride, kv_stride, q_out_stride;
    double factor;
    float eps;
    uint32_t n, rot, n_heads, n_kv, ps, n_pages, max_pages, n_seqs;
};

// factor * (cos, sin)(a) by the series of both after the nearest multiple of
// pi/2 (pi/2 in two parts: exact products in the fma) is taken off: |r| <= pi/4,
// where the first terms left out are below 1e-16.
__device__ __forceinline__ float2 turn_of(double a, double factor) {
    const double n = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.57079632679489661923, a);
    r = __builtin_fma(-n, 6.123233995736766036e-17, r);
    const double z = r * r;
    double s = -1.0 / 1307674368000.0;
    s = __builtin_fma(s, z, 1.0 / 6227020800.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    s = __builtin_fma(s * z, r, r);
    double c = 1.0 / 20922789888000.0;
    c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const int m = (int)(n - 4.0 * __builtin_floor(n * 0.25));  // n mod 4
    const double co = m & 1 ? s : c, si = m & 1 ? c : s;
    return make_float2((float)((m == 1 || m == 2 ? -co : co) * factor), (float)((m & 2 ? -si : si) * factor));
}

// One workgroup per token; a thread takes 8 values of one head at a time, always
// the same 8 of the HD: its norm weights, cosines and sines stay in registers.
// The values of the first kAhead heads are loaded before the token's sequence is
// looked up, so that the chain start -> length -> angles runs while they arrive.
// Each wave works the token's angles out for itself (a lane a pair) and spreads
// them through LDS: no wait for another wave.  HALF: halves, else neighbours.
constexpr uint32_t kAhead = 3;
template <class TI, class TQ, int HD, bool HALF>
__global__ void __launch_bounds__(256) k_paged_rotate(RotateArgs a) {
    constexpr uint32_t per = HD / 8;
    __shared__ float2 turns[4][64];
    const uint32_t t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, d = tid % per * 8, width = blockDim.x;
    const uint32_t qu = a.q ? a.n_heads * per : 0, ku = a.n_kv * per, units = qu + 2 * ku;
    auto load = [&](uint32_t u, float(&x)[8]) {
        if (u < qu) load8<TI>(a.q, t * a.q_stride + u * 8, x);
        else if (u < qu + ku) load8<TI>(a.k, t * a.kv_stride + (u - qu) * 8, x);
        else if (u < units) load8<TI>(a.v, t * a.kv_stride + (u - qu - ku) * 8, x);
        else
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = 0.0f;
    };
    float x[kAhead][8];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; i++) load(tid + i * width, x[i]);
    float qw[8], kw[8];
    if (a.q_norm)
#pragma unroll
        for (int e = 0; e < 8; e++) qw[e] = a.q_norm[d + e];
    if (a.k_norm)
#pragma unroll
        for (int e = 0; e < 8; e++) kw[e] = a.k_norm[d + e];
    const double freq = lane < a.rot / 2 ? a.freqs[lane] : 0.0;

    // the token's sequence, position and page
    uint32_t s = t, first = t, last = t + 1;
    if (a.q_start) {
        s = wave_search(a.n, t, [&](uint32_t i) { return (uint64_t)a.q_start[i]; });
        first = a.q_start[s];
        last = a.q_start[s + 1];
        if (t < first || t >= last) return;  // before the first sequence or behind the last
    }
    const uint32_t id = a.seqs ? a.seqs[s] : s;
    int64_t pos = -1;
    uint32_t page = ANE_NO_PAGE, row = 0;
    if (id < a.n_seqs) {
        // (the length as attention counts it, or a row would see another token's keys)
        pos = (int64_t)min((uint64_t)a.kv_len[id], (uint64_t)a.max_pages * a.ps) - (int64_t)(last - t);
        if (pos >= 0) {
            page = a.table[(uint64_t)id * a.max_pages + (uint32_t)pos / a.ps];
            row = (uint32_t)pos % a.ps;
        }
    }
    float co[8], si[8];  // of value d + e's pair
    if (a.rot) {
        float2* mine = turns[tid >> 6];
        mine[lane] = turn_of((double)pos * freq, a.factor);
        __builtin_amdgcn_wave_barrier();
        wait_lgkmcnt0();
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) {
            const float2 c = mine[(HALF ? (d + e) % max(a.rot / 2, 1u) : (d + e) / 2) & 63];
            co[e] = c.x, si[e] = c.y;
        }
    }
    // halves: the other value of a pair is rot / 16 lanes up or down
    const bool upper = HALF && d >= a.rot / 2;
    const uint32_t other = upper ? lane - a.rot / 16 : lane + a.rot / 16;

    auto put = [&](uint32_t u, float(&v)[8]) {
        const bool isq = u < qu, isv = u >= qu + ku;
        const float* w = isq ? a.q_norm : a.k_norm;
        if (w && !isv) {  // (whole heads: all lanes of one agree)
            // (squares in fp64, and the head brought near 1 by 2^k, 4^k <= mean + eps:
            // any head of fp32 values has its norm)
            double ss = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) ss = __builtin_fma((double)v[e], (double)v[e], ss);
            ss += dpp_f64<kDppQuadXor1>(ss);
            ss += dpp_f64<kDppQuadXor2>(ss);
            ss += dpp_f64<kDppHalfMirror>(ss);
            if (HD == 128) ss += dpp_f64<kDppRowMirror>(ss);
            const double m = ss * (1.0 / HD) + (double)a.eps;
            const int k = ((int)((uint32_t)__double2hiint(m) >> 20) - 1023) >> 1;
            const float inv = 1.0f / sqrtf((float)__builtin_ldexp(m, -2 * k));
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __builtin_ldexpf(v[e], -k) * inv * (isq ? qw[e] : kw[e]);
        }
        if (a.rot) {
            float y[8];
            if constexpr (HALF) {
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = __shfl(v[e], other, 64);
            }
            if (!isv && d < a.rot) {
                if constexpr (HALF) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[e] = upper ? __fadd_rn(__fmul_rn(y[e], si[e]), __fmul_rn(v[e], co[e]))
                                     : __fsub_rn(__fmul_rn(v[e], co[e]), __fmul_rn(y[e], si[e]));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float p = v[e], r = v[e + 1];
                        v[e] = __fsub_rn(__fmul_rn(p, co[e]), __fmul_rn(r, si[e]));
                        v[e + 1] = __fadd_rn(__fmul_rn(p, si[e]), __fmul_rn(r, co[e]));
                    }
                }
            }
        }
        if (u >= units) return;
        if (isq) {
            if (pos < 0)
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = 0.0f;
            store8<TQ>(a.q_out, t * a.q_out_stride + u * 8, v);
        } else if (page < a.n_pages) {
            const uint32_t g = (u - qu - (isv ? ku : 0)) / per;
            store8<_Float16>(isv ? a.vp : a.kp, (((uint64_t)page * a.n_kv + g) * a.ps + row) * HD + d, v);
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; i++) put(tid + i * width, x[i]);
    for (uint32_t i = kAhead; i * width < units; i++) {  // (all lanes: they exchange values)
        load(tid + i * width, x[0]);
        put(tid + i * width, x[0]);
    }
}

template <class TI, class TQ>
void launch(const RotateArgs& a, uint32_t hd, bool half, uint32_t n_tokens, hipStream_t s) {
    const auto f = hd == 128 ? (half ? k_paged_rotate<TI, TQ, 128, true> : k_paged_rotate<TI, TQ, 128, false>)
                             : (half ? k_paged_rotate<TI, TQ, 64, true> : k_paged_rotate<TI, TQ, 64, false>);
    const uint32_t units = ((a.q ? a.n_heads : 0) + 2 * a.n_kv) * hd / 8;
    hipLaunchKernelGGL(f, dim3(n_tokens), dim3(64 * std::min((units + 64 * kAhead - 1) / (64 * kAhead), 4u)), 0, s, a);
}

}  // namespace
}  // namespace ane

using namespace ane;

extern "C" int ane_hip_paged_norm_rope_append(const ane_paged_cache* cache, uint32_t layer, const uint32_t* seqs, uint32_t n,
                                              const uint32_t* q_start, uint32_t n_tokens, int in_type, const void* q,
                                              uint64_t q_stride, const void* k, const void* v, uint64_t kv_stride,
                                              const ane_rope* rope, const float* q_norm, const float* k_norm, float eps,
                                              int q_out_type, void* q_out, uint64_t q_out_stride, void* stream) {
    const int st = cache_status(cache);
    if (st) return st;
    const uint32_t rot = rope ? rope->rot_dim : 0;
    if (layer >= cache->n_layers || n_tokens > kMaxTokens || (in_type != ANE_TYPE_F32 && in_type != ANE_TYPE_F16) ||
        (q_out_type != ANE_TYPE_F32 && q_out_type != ANE_TYPE_F16) || (!q_start && n_tokens != n) || rot % 16 ||
        rot > cache->head_dim || (rot && !(rope->factor > 0.0 && rope->factor < 1e30)) || !(eps >= 0.0f) || !(eps < 1e30f))
        return ANE_ERR_INVALID_ARG;
    if (n == 0 || n_tokens == 0) return ANE_OK;
    if (!k || !v || (!q != !q_out) || (rot && !rope->freqs)) return ANE_ERR_BAD_POINTER;
    const uint32_t isz = in_type == ANE_TYPE_F32 ? 4 : 2, osz = q_out_type == ANE_TYPE_F32 ? 4 : 2;
    const uint64_t qw = (uint64_t)cache->n_heads * cache->head_dim;
    if ((((uintptr_t)q) | ((uintptr_t)k) | ((uintptr_t)v) | ((uintptr_t)q_out)) & 15 ||
        (((uintptr_t)q_norm) | ((uintptr_t)k_norm) | ((uintptr_t)q_start) | ((uintptr_t)seqs)) & 3 ||
        (rot && ((uintptr_t)rope->freqs) & 7) || (kv_stride * isz) & 15 ||
        kv_stride < (uint64_t)cache->n_kv_heads * cache->head_dim ||
        (q && ((q_stride * isz) & 15 || (q_out_stride * osz) & 15 || q_stride < qw || q_out_stride < qw)))
        return ANE_ERR_INVALID_ARG;
    RotateArgs a;
    const uint64_t lo = page_elems(cache) * cache->n_pages * layer;
    a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.rot = rot, a.freqs = rot ? rope->freqs : nullptr, a.factor = rot ? rope->factor : 1.0;
    a.kp = cache->k_pages + lo, a.vp = cache->v_pages + lo;
    a.table = cache->page_table, a.kv_len = cache->kv_len, a.seqs = seqs, a.q_start = q_start;
    a.q_stride = q_stride, a.kv_stride = kv_stride, a.q_out_stride = q_out_stride;
    a.n = n, a.n_heads = cache->n_heads, a.n_kv = cache->n_kv_heads, a.ps = cache->page_size, a.n_pages = cache->n_pages;
    a.max_pages = cache->max_pages, a.n_seqs = cache->n_seqs;
    const bool half = rot && rope->halves;
    hipStream_t s = (hipStream_t)stream;
    if (in_type == ANE_TYPE_F32)
        q_out_type == ANE_TYPE_F32 ? launch<float, float>(a, cache->head_dim, half, n_tokens, s)
                                   : launch<float, _Float16>(a, cache->head_dim, half, n_tokens, s);
    else
        q_out_type == ANE_TYPE_F32 ? launch<_Float16, float>(a, cache->head_dim, half, n_tokens, s)
                                   : launch<_Float16, _Float16>(a, cache->head_dim, half, n_tokens, s);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}
