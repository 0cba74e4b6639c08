// linear_i8.hip -- the int8 linear layer of a batch: tokens quantized with a
// scale each, the product with an int8 weight matrix, and the scales of token
// and output channel applied as it is written.
//
//   y = x, or fl(fl(x * inv) * norm_w) with inv as ane_hip_rms_norm's
//   q[t][k] = rint(y * fl(fl(1 / max|y_t|) * 127)),  qs[t] = max|y_t| / 127
//   out[t][n] = fl(fl((float)sum_k q[t][k] w[n][k] * qs[t]) * ws[n]) + bias[n] + residual[t][n]
//
// The sum is an exact int32 (K below 2^17), so no split of K and no order of
// its terms changes a result.
#include "../../include/ane_decode.h"
#include "gemm_i8.hpp"
#include <algorithm>

namespace ane {
namespace {

// Eight values from p on, whatever their alignment (dword loads that the
// memory system takes at any address).
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
    T v[8];
};
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)e.v[i];
}

struct QuantArgs {
    const void* x;
    uint64_t x_stride, q_stride;
    const float* norm_w;
    int8_t* q;
    float* scales;
    uint32_t T, K;
    float eps;
    uint32_t* zero;  // kScaledCounts words to clear, or null
};

// Values k .. k + 7 of a row of K, zeros past its end.
template <class T>
__device__ __forceinline__ void load_part(const T* x, uint32_t k, uint32_t K, float (&y)[8]) {
    if (k + 8 <= K) {
        load8<T>(x + k, y);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) y[e] = k + e < K ? (float)x[k + e] : 0.0f;
    }
}
__device__ __forceinline__ void apply_norm(float (&y)[8], float inv, const float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = __fmul_rn(__fmul_rn(y[e], inv), w[e]);
}

// The sum of squares of the 32-block that lanes 4 i .. 4 i + 3 hold, in the order of
// common.hpp's canonical sum (in all four lanes).
__device__ __forceinline__ double block_sumsq(const float (&y)[8]) {
    double v = sumsq4_f64(make_float4(y[0], y[1], y[2], y[3])) + sumsq4_f64(make_float4(y[4], y[5], y[6], y[7]));
    v += dpp_f64<kDppQuadXor1>(v);
    v += dpp_f64<kDppQuadXor2>(v);
    return v;
}
// canon_total_f64, its tree by lane permutes where a row of 16 lanes will do: the
// same pairs are added (a mirrored lane holds what lane ^ 4 or ^ 8 holds).
__device__ __forceinline__ double blocks_total(const double* s, uint32_t nb) {
    const uint32_t lane = threadIdx.x & 63;
    double c = 0.0;
    for (uint32_t b = lane; b < nb; b += 64) c += s[b];
    c += dpp_f64<kDppQuadXor1>(c);
    c += dpp_f64<kDppQuadXor2>(c);
    c += dpp_f64<kDppHalfMirror>(c);
    c += dpp_f64<kDppRowMirror>(c);
    c += __shfl_xor(c, 16, 64);
    c += __shfl_xor(c, 32, 64);
    return c;
}
__device__ __forceinline__ uint32_t largest(uint32_t top, const float (&y)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, abs_key(y[e]));
    return top;
}

// How a token is quantized, from its largest magnitude (as a key: NaN above all).
struct TokenScale {
    float up, per, scale;
    bool plain;
    __device__ __forceinline__ TokenScale(uint32_t top) {
        // (a maximum below 2^-96 is brought up first: its reciprocal would not be finite; the
        // scale is divided as it is, or a denormal one would be rounded twice)
        up = top < 0x0f800000u ? 0x1p96f : 1.0f;
        const float m = __uint_as_float(top) * up;
        per = top == 0 ? 127.0f : __fmul_rn(1.0f / m, 127.0f);
        scale = top == 0 ? 1.0f : __uint_as_float(top) / 127.0f;
        // (every |y per| is below 127.5 then: 1 / m is off by 2^-24 of itself, above 2^126, where
        // it is denormal, by 2^-22, the two products by 2^-24 each)
        plain = up == 1.0f && fast_quant_ok(m, per);
    }
    __device__ __forceinline__ uint2 pack(const float (&y)[8]) const {
        if (plain) return make_uint2(pack4_fast(y[0], y[1], y[2], y[3], per), pack4_fast(y[4], y[5], y[6], y[7], per));
        return make_uint2(pack4(y[0] * up, y[1] * up, y[2] * up, y[3] * up, per),
                          pack4(y[4] * up, y[5] * up, y[6] * up, y[7] * up, per));
    }
};

constexpr uint32_t kMaxK = (1u << 17) - 1;      // |sum| <= K 2^14 < 2^31

// NW waves a token; thread i takes the values 8 i .. 8 i + 7 of every run of
// 512 NW, of which R stay in registers between the passes (sum of squares,
// maximum, output); a token of more runs (R = 0) is read again in each.
template <class T, int NW, int R>
__global__ void __launch_bounds__(NW > 4 ? 64 * NW : 256) k_quantize_tokens(QuantArgs a) {
    constexpr uint32_t kPer = NW > 4 ? 1 : 4 / NW, kRun = 512 * NW;
    constexpr uint32_t kBlocks = R ? R * kRun / 32 : (kMaxK + 31) / 32;  // of a token
    __shared__ double blocks[kPer][kBlocks];
    __shared__ uint32_t tops[NW];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t t = blockIdx.x * kPer + wave / NW, i0 = (wave % NW * 64 + lane) * 8;
    if (a.zero && blockIdx.x == 0 && threadIdx.x < kScaledCounts) a.zero[threadIdx.x] = 0;
    if (NW == 1 && t >= a.T) return;  // (whole waves, and nothing below waits for another one)
    const T* x = static_cast<const T*>(a.x) + (uint64_t)t * a.x_stride;
    const uint32_t runs = R ? R : (a.K + kRun - 1) / kRun;
    float v[R ? R : 1][8];
    // run r again (R = 0) or from its registers, normalised where asked
    auto part = [&](uint32_t r) -> float(&)[8] {
        if constexpr (R) return v[r];
        load_part<T>(x, r * kRun + i0, a.K, v[0]);
        return v[0];
    };
    auto normed = [&](uint32_t r, float inv) {
        float w[8];
        load_part<float>(a.norm_w, r * kRun + i0, a.K, w);
        apply_norm(v[R ? r : 0], inv, w);
    };
    auto each = [&](auto f) {
        if constexpr (R) {
#pragma unroll
            for (uint32_t r = 0; r < (uint32_t)R; r++) f(r);
        } else {
            for (uint32_t r = 0; r < runs; r++) f(r);
        }
    };
    if constexpr (R) each([&](uint32_t r) { load_part<T>(x, r * kRun + i0, a.K, v[r]); });

    float inv = 1.0f;
    if (a.norm_w) {
        double* const s = blocks[wave / NW];
        each([&](uint32_t r) {
            const double b = block_sumsq(part(r));
            const uint32_t at = (r * kRun + i0) / 32;
            if ((lane & 3) == 0 && at < kBlocks) s[at] = b;  // (past the token's end: zeros)
        });
        if constexpr (NW > 1) __syncthreads();
        else wait_lgkmcnt0();
        inv = rms_inv(blocks_total(s, (a.K + 31) / 32), a.K, a.eps);
    }
    uint32_t top = 0;
    each([&](uint32_t r) {
        float(&y)[8] = part(r);
        if (a.norm_w) normed(r, inv);
        top = largest(top, y);
    });
    top = wave_max_u32(top);
    if constexpr (NW > 1) {
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        top = wave_max_u32(lane < NW ? tops[lane] : 0);
    }
    const TokenScale ts(top);
    if (wave % NW == 0 && lane == 0) a.scales[t] = ts.scale;
    const uint32_t Kp = (a.K + 15) & ~15u;  // zeros up to here
    each([&](uint32_t r) {
        const uint32_t k = r * kRun + i0;
        if (k >= Kp) return;
        float(&y)[8] = part(r);
        if (!R && a.norm_w) normed(r, inv);
        *reinterpret_cast<uint2*>(a.q + (uint64_t)t * a.q_stride + k) = ts.pack(y);
    });
}

constexpr uint32_t kMaxRows = 65535u * 128;     // of x and of w: workgroups of 128 in a launch's y

// One wave a token from 1024 tokens on (4096 x 4096 fp16 behind a norm 19.9 -> 13.2
// us, 3.8 TB/s; without one 10.4, 4.8), sixteen up to 256 (32 x 14336 fp32 4.8 -> 3.4),
// four between.
constexpr uint32_t kManyTokens = 1024, kFewTokens = 256, kMaxFour = 16384;  // (values that four waves hold)
// Longer tokens take 1024 threads each, and a launch holds fewer than 2^32.
bool quantize_fits(uint32_t T, uint32_t K) { return K <= kMaxFour || launch_fits(T, 1024); }
template <class T>
void launch_quantize(const QuantArgs& a, hipStream_t s) {
    auto go = [&](auto* f, uint32_t nw) {
        hipLaunchKernelGGL(f, dim3(nw == 1 ? (a.T + 3) / 4 : a.T), dim3(nw > 4 ? 64 * nw : 256), 0, s, a);
    };
    if (a.K <= 512) return go(k_quantize_tokens<T, 1, 1>, 1);
    if (a.T >= kManyTokens && a.K <= 2048) return go(k_quantize_tokens<T, 1, 4>, 1);
    if (a.T >= kManyTokens && a.K <= 4096) return go(k_quantize_tokens<T, 1, 8>, 1);
    if (a.T <= kFewTokens || a.K > kMaxFour) {
        if (a.K <= 2048) return go(k_quantize_tokens<T, 4, 1>, 4);
        if (a.K <= 8192) return go(k_quantize_tokens<T, 16, 1>, 16);
        if (a.K <= kMaxFour) return go(k_quantize_tokens<T, 16, 2>, 16);
        return go(k_quantize_tokens<T, 16, 0>, 16);
    }
    switch ((a.K + 2047) / 2048) {
        case 1: return go(k_quantize_tokens<T, 4, 1>, 4);
        case 2: return go(k_quantize_tokens<T, 4, 2>, 4);
        case 3: return go(k_quantize_tokens<T, 4, 3>, 4);
        case 4: return go(k_quantize_tokens<T, 4, 4>, 4);
        case 5: return go(k_quantize_tokens<T, 4, 5>, 4);
        case 6: return go(k_quantize_tokens<T, 4, 6>, 4);
        case 7: return go(k_quantize_tokens<T, 4, 7>, 4);
        default: return go(k_quantize_tokens<T, 4, 8>, 4);
    }
}

__device__ __forceinline__ int wave_sum_i32(int v) {
    v += (int)dpp_u32<kDppQuadXor1>((uint32_t)v);
    v += (int)dpp_u32<kDppQuadXor2>((uint32_t)v);
    v += (int)dpp_u32<kDppHalfMirror>((uint32_t)v);
    v += (int)dpp_u32<kDppRowMirror>((uint32_t)v);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
           __builtin_amdgcn_readlane(v, 48);
}

// One token, quantized where it is multiplied: every workgroup quantizes the whole
// token for itself (R runs of 4096 values) into LDS, and each of its eight waves sums
// up rows of the weights, 1 KB of one a step (16 values a lane, four-way dot products),
// D steps on their way at a time, the first of them while the token is quantized.  One
// launch, and rows read front to back: 28672 x 4096 19.8 us, 5.9 TB/s, where the matrix
// cores' layout (64 bytes of each of 16 rows a load) takes 27; 6144 x 4096 behind a
// norm 7.9, the quantizer's launch and the few-row kernel's 11.6.  Eight or twelve
// steps at a time, or four waves, gain nothing.
template <class T, int R, int D>
__global__ void __launch_bounds__(512) k_linear_one(QuantArgs a, GemmParams p, uint32_t rows) {
    constexpr uint32_t kRun = 4096;
    __shared__ __attribute__((aligned(16))) uint8_t q[R * kRun];
    __shared__ double blocks[R * kRun / 32];
    __shared__ uint32_t tops[8];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const T* x = static_cast<const T*>(a.x);
    float v[R][8], w[R][8];
#pragma unroll
    for (uint32_t r = 0; r < (uint32_t)R; r++) load_part<T>(x, r * kRun + tid * 8, a.K, v[r]);
    if (a.norm_w)
#pragma unroll
        for (uint32_t r = 0; r < (uint32_t)R; r++) load_part<float>(a.norm_w, r * kRun + tid * 8, a.K, w[r]);
    __builtin_amdgcn_sched_barrier(0);  // loads return in order: the token's before the weights

    // this wave's rows n0 .. n0 + m - 1, its steps in order: chunk c of row n
    const uint32_t n0 = min((blockIdx.x * 8 + wave) * rows, p.Nout), m = min(rows, p.Nout - n0);
    const uint32_t chunks = (p.Kp + 1023) / 1024, steps = m * chunks;
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.B, (uint32_t)(p.colsB * p.ldb));
    uint32_t lc = 0, lo = n0 * (uint32_t)p.ldb;  // of the next load: chunk, row's offset
    auto load = [&] {
        const uint32_t k = lc * 1024 + lane * 16;
        const v4i b = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rb, k < p.Kp ? lo + k : 0x80000000u, 0, kCpolNt));
        if (++lc == chunks) lc = 0, lo += (uint32_t)p.ldb;
        return b;
    };
    v4i b[D];
#pragma unroll
    for (uint32_t d = 0; d < (uint32_t)D; d++)
        if (d < steps) b[d] = load();
    __builtin_amdgcn_sched_barrier(0);

    if (a.norm_w) {
#pragma unroll
        for (uint32_t r = 0; r < (uint32_t)R; r++) {
            const double s = block_sumsq(v[r]);
            if ((lane & 3) == 0) blocks[(r * kRun + tid * 8) / 32] = s;
        }
        wait_lgkmcnt0();
        lds_barrier();
        const float inv = rms_inv(blocks_total(blocks, (a.K + 31) / 32), a.K, a.eps);
#pragma unroll
        for (uint32_t r = 0; r < (uint32_t)R; r++) apply_norm(v[r], inv, w[r]);
    }
    uint32_t top = 0;
#pragma unroll
    for (uint32_t r = 0; r < (uint32_t)R; r++) top = largest(top, v[r]);
    top = wave_max_u32(top);
    if (lane == 0) tops[wave] = top;
    wait_lgkmcnt0();
    lds_barrier();
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, tops[i]);
    const TokenScale ts(top);
#pragma unroll
    for (uint32_t r = 0; r < (uint32_t)R; r++) *reinterpret_cast<uint2*>(q + r * kRun + tid * 8) = ts.pack(v[r]);
    wait_lgkmcnt0();
    lds_barrier();

    int acc = 0, mine = 0;  // lane i: row n0 + i's sum
    uint32_t c = 0, row = 0;
    for (uint32_t j = 0; j < steps; j += D) {
#pragma unroll
        for (uint32_t d = 0; d < (uint32_t)D; d++) {
            if (j + d >= steps) break;
            const v4i y = *reinterpret_cast<const v4i*>(q + c * 1024 + lane * 16);
#pragma unroll
            for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_sdot4(y[e], b[d][e], acc, false);
            if (j + D + d < steps) b[d] = load();
            if (++c == chunks) {
                acc = wave_sum_i32(acc);
                if (lane == row) mine = acc;
                acc = 0, c = 0, row++;
            }
        }
    }
    if (lane < m) {
        const uint32_t n = n0 + lane;
        sc_put(p, 0, n, sc_out(mine, ts.scale, p.cs[n], p.bias ? p.bias[n] : 0.0f));
    }
}

// The same for TT tokens that are quantized already: they are copied to LDS whole, a
// step of the weights meets 1 KB of each.  4 x 28672 x 4096 20 us, 5.9 TB/s (64-tiles
// 26), 4 x 4096 x 14336 12 (14).
template <int TT, int D>
__global__ void __launch_bounds__(512) k_linear_dot(GemmParams p, uint32_t rows) {
    extern __shared__ __attribute__((aligned(16))) uint8_t qs[];  // [TT][chunks][1024]
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t chunks = (p.Kp + 1023) / 1024;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.A, (uint32_t)(p.rowsA * p.lda));
    // (rows past the last token, and values past the last, are zeros)
    for (uint32_t i = wave; i < TT * chunks; i += 8) {
        const uint32_t t = i / chunks, k = (i - t * chunks) * 1024 + lane * 16;
        copy16_to_lds(ra, qs + i * 1024, t < p.Mout && k < p.Kp ? t * (uint32_t)p.lda + k : 0x80000000u);
    }
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t n0 = min((blockIdx.x * 8 + wave) * rows, p.Nout), m = min(rows, p.Nout - n0);
    const uint32_t steps = m * chunks;
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(p.B, (uint32_t)(p.colsB * p.ldb));
    uint32_t lc = 0, lo = n0 * (uint32_t)p.ldb;  // of the next load: chunk, row's offset
    auto load = [&] {
        const uint32_t k = lc * 1024 + lane * 16;
        const v4i b = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rb, k < p.Kp ? lo + k : 0x80000000u, 0, kCpolNt));
        if (++lc == chunks) lc = 0, lo += (uint32_t)p.ldb;
        return b;
    };
    v4i b[D];
#pragma unroll
    for (uint32_t d = 0; d < (uint32_t)D; d++) b[d] = d < steps ? load() : v4i{0, 0, 0, 0};
    __builtin_amdgcn_sched_barrier(0);
    if (steps >= (uint32_t)D) wait_vmcnt<D>();  // the tokens' copies
    else wait_vmcnt<0>();
    lds_barrier();

    int acc[TT], mine = 0;  // lane i: token i % TT's sum over row n0 + i / TT
#pragma unroll
    for (int t = 0; t < TT; t++) acc[t] = 0;
    uint32_t c = 0, row = 0;
    for (uint32_t j = 0; j < steps; j += D) {
#pragma unroll
        for (uint32_t d = 0; d < (uint32_t)D; d++) {
            if (j + d >= steps) break;
            v4i y[TT];
#pragma unroll
            for (int t = 0; t < TT; t++) y[t] = *reinterpret_cast<const v4i*>(qs + (t * chunks + c) * 1024 + lane * 16);
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[t] = __builtin_amdgcn_sdot4(y[t][e], b[d][e], acc[t], false);
            if (j + D + d < steps) b[d] = load();
            if (++c == chunks) {
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    const int sum = wave_sum_i32(acc[t]);
                    if (lane == row * TT + t) mine = sum;
                    acc[t] = 0;
                }
                c = 0, row++;
            }
        }
    }
    const uint32_t n = n0 + lane / TT, t = lane % TT;
    if (lane < m * TT && t < p.Mout) sc_put(p, t, n, sc_out(mine, p.rs[t], p.cs[n], p.bias ? p.bias[n] : 0.0f));
}

// Its runs of 4096 values, or 0 where it does not apply: tokens that registers hold,
// weights within 32-bit offsets (0x80000000 marks an empty load).
uint32_t linear_one_runs(const GemmParams& p, uint32_t K) {
    if (p.Mout != 1 || p.colsB * p.ldb >= (1ull << 31)) return 0;
    return K <= 4096 ? 1 : K <= 8192 ? 2 : K <= 16384 ? 4 : 0;
}
template <class T>
void launch_one(const QuantArgs& a, const GemmParams& p, uint32_t runs, hipStream_t s) {
    // two workgroups a CU (one: 28672 x 4096 22, 20 so), of at most 64 rows a wave
    const uint32_t rows = std::min(64u, (p.Nout + 4095) / 4096);
    const auto f = runs == 1 ? k_linear_one<T, 1, 4> : runs == 2 ? k_linear_one<T, 2, 4> : k_linear_one<T, 4, 4>;
    hipLaunchKernelGGL(f, dim3((p.Nout + 8 * rows - 1) / (8 * rows)), dim3(512), 0, s, a, p, rows);
}

template <int TT>
int launch_dot(const GemmParams& p, hipStream_t s) {
    const uint32_t rows = std::min(64u / TT, (p.Nout + 4095) / 4096), lds = TT * (uint32_t)((p.Kp + 1023) / 1024) * 1024;
    hipLaunchKernelGGL((k_linear_dot<TT, 4>), dim3((p.Nout + 8 * rows - 1) / (8 * rows)), dim3(512), lds, s, p, rows);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

int quantize(int type, const QuantArgs& a, hipStream_t s) {
    type == ANE_TYPE_F32 ? launch_quantize<float>(a, s) : launch_quantize<_Float16>(a, s);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

uint64_t item_size(int type) { return type == ANE_TYPE_F32 ? 4 : 2; }
bool known_type(int type) { return type == ANE_TYPE_F32 || type == ANE_TYPE_F16; }
bool off(const void* p, uint64_t n) { return ((uintptr_t)p) % n != 0; }

int tokens_status(uint32_t T, uint32_t K, int type, const void* x, uint64_t x_stride, const float* norm_w, float eps) {
    if (T > kMaxRows || K == 0 || K > kMaxK || !quantize_fits(T, K) || !known_type(type) || !(eps >= 0.0f) || !(eps < 1e30f))
        return ANE_ERR_INVALID_ARG;
    if (T == 0) return ANE_OK;
    if (!x) return ANE_ERR_BAD_POINTER;
    if (off(x, item_size(type)) || off(norm_w, 4) || (T > 1 && x_stride < K)) return ANE_ERR_INVALID_ARG;
    return ANE_OK;
}
int product_status(uint32_t T, uint32_t N, uint32_t K, const int8_t* w, uint64_t w_stride, const float* w_scales,
                   const float* bias, const void* residual, uint64_t residual_stride, int out_type, const void* out,
                   uint64_t out_stride) {
    if (T > kMaxRows || N > kMaxRows || (uint64_t)T * N >= (1ull << 38) || K == 0 || K > kMaxK || !known_type(out_type)) return ANE_ERR_INVALID_ARG;
    if (T == 0 || N == 0) return ANE_OK;
    if (!w || !w_scales || !out) return ANE_ERR_BAD_POINTER;
    const uint64_t size = item_size(out_type);
    if (off(w, 16) || w_stride % 16 || w_stride < K || w_stride >= (1ull << 31) || off(w_scales, 4) || off(bias, 4) ||
        off(residual, size) || off(out, size) || (T > 1 && (out_stride < N || (residual && residual_stride < N))))
        return ANE_ERR_INVALID_ARG;
    return ANE_OK;
}

uint64_t row_bytes(uint32_t K) { return ceil_to(K, 128); }  // of q in a workspace
uint64_t q_bytes(uint32_t T, uint32_t K) { return ceil_to(T * row_bytes(K), 256); }

// Of a linear_i8 call: q, its scales, and where K is split the counts and sums of the parts.
struct LinearSpace {
    ScaledPlan plan;
    uint64_t scales, counts, planes, bytes;
};
uint64_t plane_bytes(uint64_t rows, uint32_t N) { return rows * ceil_to(N, 4) * 4; }  // of sums, over all parts
LinearSpace linear_space(uint32_t T, uint32_t N, uint32_t K) {
    LinearSpace l;
    l.plan = scaled_plan(T, N, K, true);
    l.scales = q_bytes(T, K);
    l.counts = l.scales + ceil_to((uint64_t)T * 4, 256);
    l.planes = l.counts + (l.plan.split > 1 ? kScaledCounts * 4 : 0);
    l.bytes = l.planes + (l.plan.split > 1 ? plane_bytes((uint64_t)l.plan.split * T, N) : 0);
    return l;
}

GemmParams product(uint32_t T, uint32_t N, uint32_t K, const int8_t* q, uint64_t q_stride, const float* q_scales, const int8_t* w,
                   uint64_t w_stride, const float* w_scales, const float* bias, const void* residual, uint64_t residual_stride,
                   int out_type, void* out, uint64_t out_stride) {
    GemmParams p{};
    p.A = q, p.lda = q_stride, p.rowsA = T, p.Mout = T;
    p.B = w, p.ldb = w_stride, p.colsB = N, p.Nout = N;
    p.Kp = (uint32_t)ceil_to(K, 16);
    p.rs = q_scales, p.cs = w_scales, p.bias = bias;
    p.res = residual, p.ldr = residual ? residual_stride : out_stride;
    p.half = out_type == ANE_TYPE_F16;
    p.C = static_cast<float*>(out), p.ldc = out_stride;
    return p;
}

}  // namespace

bool gemm_dot_eligible(const GemmParams& p) {
    const uint32_t tt = p.Mout <= 1 ? 1 : p.Mout <= 2 ? 2 : p.Mout <= 4 ? 4 : 8;
    return p.Mout <= 8 && tt * ceil_to(p.Kp, 1024) <= 64 * 1024 && p.colsB * p.ldb < (1ull << 31) && p.rowsA * p.lda < (1ull << 31);
}

int launch_gemm_dot(const GemmParams& p, hipStream_t s) {
    return p.Mout <= 1 ? launch_dot<1>(p, s) : p.Mout <= 2 ? launch_dot<2>(p, s) : p.Mout <= 4 ? launch_dot<4>(p, s) : launch_dot<8>(p, s);
}

}  // namespace ane

using namespace ane;

extern "C" int ane_hip_quantize_tokens(uint32_t T, uint32_t K, int type, const void* x, uint64_t x_stride,
                                       const float* norm_w, float eps, int8_t* q, uint64_t q_stride, float* scales,
                                       void* stream) {
    const int st = tokens_status(T, K, type, x, x_stride, norm_w, eps);
    if (st || T == 0) return st;
    if (!q || !scales) return ANE_ERR_BAD_POINTER;
    if (off(q, 16) || q_stride % 16 || q_stride < K || off(scales, 4)) return ANE_ERR_INVALID_ARG;
    return quantize(type, QuantArgs{x, x_stride, q_stride, norm_w, q, scales, T, K, eps, nullptr}, (hipStream_t)stream);
}

extern "C" int ane_hip_dense_i8_scaled(uint32_t T, uint32_t N, uint32_t K, const int8_t* q, uint64_t q_stride,
                                       const float* q_scales, const int8_t* w, uint64_t w_stride, const float* w_scales,
                                       const float* bias, const void* residual, uint64_t residual_stride, int out_type,
                                       void* out, uint64_t out_stride, void* stream) {
    const int st = product_status(T, N, K, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out, out_stride);
    if (st || T == 0 || N == 0) return st;
    if (!q || !q_scales) return ANE_ERR_BAD_POINTER;
    if (off(q, 16) || q_stride % 16 || q_stride < K || q_stride >= (1ull << 31) || off(q_scales, 4)) return ANE_ERR_INVALID_ARG;
    return launch_gemm_scaled(product(T, N, K, q, q_stride, q_scales, w, w_stride, w_scales, bias, residual, residual_stride,
                                      out_type, out, out_stride),
                              scaled_plan(T, N, K, false), (hipStream_t)stream);
}

extern "C" size_t ane_hip_linear_i8_workspace_size(uint32_t T, uint32_t N, uint32_t K) {
    if (T == 0 || T > kMaxRows || N == 0 || N > kMaxRows || K == 0 || K > kMaxK) return 0;
    const LinearSpace l = linear_space(T, N, K);
    const uint64_t rows = scaled_split_rows(T, N, K);  // (a call of fewer tokens may split K where this one does not)
    return std::max(l.bytes, rows ? l.counts + kScaledCounts * 4 + plane_bytes(rows, N) : 0);
}

extern "C" int ane_hip_linear_i8(uint32_t T, uint32_t N, uint32_t K, int type, const void* x, uint64_t x_stride,
                                 const float* norm_w, float eps, const int8_t* w, uint64_t w_stride, const float* w_scales,
                                 const float* bias, const void* residual, uint64_t residual_stride, int out_type, void* out,
                                 uint64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    int st = tokens_status(T, K, type, x, x_stride, norm_w, eps);
    if (!st) st = product_status(T, N, K, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out, out_stride);
    if (st || T == 0 || N == 0) return st;
    const LinearSpace l = linear_space(T, N, K);
    if (!workspace || off(workspace, 256) || workspace_bytes < l.bytes) return ANE_ERR_WORKSPACE;
    int8_t* q = static_cast<int8_t*>(workspace);
    float* qs = reinterpret_cast<float*>(q + l.scales);
    GemmParams p = product(T, N, K, q, row_bytes(K), qs, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out,
                           out_stride);
    if (l.plan.split > 1) {
        p.counts = reinterpret_cast<uint32_t*>(q + l.counts);
        p.planes = reinterpret_cast<int32_t*>(q + l.planes);
    }
    const QuantArgs a{x, x_stride, row_bytes(K), norm_w, q, qs, T, K, eps, p.counts};
    // (the one launch reads x in every workgroup, so an output in its place takes two)
    const uintptr_t xa = (uintptr_t)x, oa = (uintptr_t)out;
    const bool apart = xa + K * item_size(type) <= oa || oa + N * item_size(out_type) <= xa;
    if (const uint32_t runs = apart ? linear_one_runs(p, K) : 0) {
        type == ANE_TYPE_F32 ? launch_one<float>(a, p, runs, (hipStream_t)stream) : launch_one<_Float16>(a, p, runs, (hipStream_t)stream);
        ANE_HIP_CHECK_LAUNCH();
        return ANE_OK;
    }
    st = quantize(type, a, (hipStream_t)stream);
    return st ? st : launch_gemm_scaled(p, l.plan, (hipStream_t)stream);
}
