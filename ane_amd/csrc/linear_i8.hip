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
};

// NW waves a token; thread i takes the values 8 i .. 8 i + 7 of every run of
// 512 NW, of which R stay in registers between the passes (sum of squares,
// maximum, output); a token of more runs (R = 0) is read again in each.
template <class T, int NW, int R>
__global__ void __launch_bounds__(256) k_quantize_tokens(QuantArgs a) {
    constexpr uint32_t kPer = 256 / (64 * NW), kRun = 512 * NW;
    __shared__ double sums[4];
    __shared__ uint32_t tops[4];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t t = blockIdx.x * kPer + wave / NW, i0 = (wave % NW * 64 + lane) * 8;
    if (NW == 1 && t >= a.T) return;  // (whole waves, and nothing below waits for another one)
    const T* x = static_cast<const T*>(a.x) + (uint64_t)t * a.x_stride;
    const uint32_t runs = R ? R : (a.K + kRun - 1) / kRun;
    float v[R ? R : 1][8];
    auto load = [&](uint32_t r, float(&y)[8]) {
        const uint32_t k = r * kRun + i0;
        if (k + 8 <= a.K) {
            load8<T>(x + k, y);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) y[e] = k + e < a.K ? (float)x[k + e] : 0.0f;
        }
    };
    auto norm = [&](uint32_t r, float(&y)[8], float inv) {
        const uint32_t k = r * kRun + i0;
        float w[8];
        if (k + 8 <= a.K) {
            load8<float>(a.norm_w + k, w);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) w[e] = k + e < a.K ? a.norm_w[k + e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = __fmul_rn(__fmul_rn(y[e], inv), w[e]);
    };
#pragma unroll
    for (uint32_t r = 0; r < R; r++) load(r, v[r]);

    float inv = 1.0f;
    if (a.norm_w) {
        double ss = 0.0;
        auto add = [&](const float(&y)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e++) ss = __builtin_fma((double)y[e], (double)y[e], ss);
        };
        if constexpr (R) {
#pragma unroll
            for (int r = 0; r < R; r++) add(v[r]);
        } else {
            for (uint32_t r = 0; r < runs; r++) load(r, v[0]), add(v[0]);
        }
        ss = tree64_f64(ss);
        if constexpr (NW > 1) {
            if (lane == 0) sums[wave] = ss;
            __syncthreads();
            ss = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        }
        inv = rms_inv(ss, a.K, a.eps);
    }
    uint32_t top = 0;
    auto most = [&](const float(&y)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, abs_key(y[e]));
    };
    if constexpr (R) {
#pragma unroll
        for (uint32_t r = 0; r < R; r++) {
            if (a.norm_w) norm(r, v[r], inv);
            most(v[r]);
        }
    } else {
        for (uint32_t r = 0; r < runs; r++) {
            load(r, v[0]);
            if (a.norm_w) norm(r, v[0], inv);
            most(v[0]);
        }
    }
    top = wave_max_u32(top);
    if constexpr (NW > 1) {
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    // (a maximum below 2^-96 is brought up first: its reciprocal would not be finite)
    const float up = top < 0x0f800000u ? 0x1p96f : 1.0f, m = __uint_as_float(top) * up;
    const float scale = top == 0 ? up : m / 127.0f, per = top == 0 ? 127.0f : __fmul_rn(1.0f / m, 127.0f);
    if (wave % NW == 0 && lane == 0) a.scales[t] = scale / up;
    const uint32_t Kp = (a.K + 15) & ~15u;  // zeros up to here
    auto put = [&](uint32_t r, const float(&y)[8]) {
        const uint32_t k = r * kRun + i0;
        if (k >= Kp) return;
        uint2 o = make_uint2(0, 0);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            o.x |= (uint32_t)(quant1(y[e] * up, per) & 0xff) << (8 * e);
            o.y |= (uint32_t)(quant1(y[4 + e] * up, per) & 0xff) << (8 * e);
        }
        *reinterpret_cast<uint2*>(a.q + (uint64_t)t * a.q_stride + k) = o;
    };
    if constexpr (R) {
#pragma unroll
        for (uint32_t r = 0; r < R; r++) put(r, v[r]);
    } else {
        for (uint32_t r = 0; r < runs; r++) {
            load(r, v[0]);
            if (a.norm_w) norm(r, v[0], inv);
            put(r, v[0]);
        }
    }
}

constexpr uint32_t kMaxK = (1u << 17) - 1;      // |sum| <= K 2^14 < 2^31
constexpr uint32_t kMaxRows = 65535u * 128;     // of x and of w: workgroups of 128 in a launch's y

template <class T>
void launch_quantize(const QuantArgs& a, hipStream_t s) {
    if (a.K <= 512) {
        hipLaunchKernelGGL((k_quantize_tokens<T, 1, 1>), dim3((a.T + 3) / 4), dim3(256), 0, s, a);
        return;
    }
    const auto fn = a.K <= 2048    ? k_quantize_tokens<T, 4, 1>
                    : a.K <= 4096  ? k_quantize_tokens<T, 4, 2>
                    : a.K <= 8192  ? k_quantize_tokens<T, 4, 4>
                    : a.K <= 16384 ? k_quantize_tokens<T, 4, 8>
                                   : k_quantize_tokens<T, 4, 0>;
    hipLaunchKernelGGL(fn, dim3(a.T), dim3(256), 0, s, a);
}

uint64_t item_size(int type) { return type == ANE_TYPE_F32 ? 4 : 2; }
bool known_type(int type) { return type == ANE_TYPE_F32 || type == ANE_TYPE_F16; }
bool off(const void* p, uint64_t n) { return ((uintptr_t)p) % n != 0; }

int tokens_status(uint32_t T, uint32_t K, int type, const void* x, uint64_t x_stride, const float* norm_w, float eps) {
    if (T > kMaxRows || K == 0 || K > kMaxK || !known_type(type) || !(eps >= 0.0f) || !(eps < 1e30f)) return ANE_ERR_INVALID_ARG;
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

int product(uint32_t T, uint32_t N, uint32_t K, const int8_t* q, uint64_t q_stride, const float* q_scales, const int8_t* w,
            uint64_t w_stride, const float* w_scales, const float* bias, const void* residual, uint64_t residual_stride,
            int out_type, void* out, uint64_t out_stride, hipStream_t s) {
    GemmParams p{};
    p.A = q, p.lda = q_stride, p.rowsA = T, p.Mout = T;
    p.B = w, p.ldb = w_stride, p.colsB = N, p.Nout = N;
    p.Kp = (uint32_t)ceil_to(K, 16);
    p.rs = q_scales, p.cs = w_scales, p.bias = bias;
    p.res = residual, p.ldr = residual ? residual_stride : out_stride;
    p.half = out_type == ANE_TYPE_F16;
    p.C = static_cast<float*>(out), p.ldc = out_stride;
    return launch_gemm_rows(p, s);
}

}  // namespace
}  // namespace ane

using namespace ane;

extern "C" int ane_hip_quantize_tokens(uint32_t T, uint32_t K, int type, const void* x, uint64_t x_stride,
                                       const float* norm_w, float eps, int8_t* q, uint64_t q_stride, float* scales,
                                       void* stream) {
    const int st = tokens_status(T, K, type, x, x_stride, norm_w, eps);
    if (st || T == 0) return st;
    if (!q || !scales) return ANE_ERR_BAD_POINTER;
    if (off(q, 16) || q_stride % 16 || q_stride < K || off(scales, 4)) return ANE_ERR_INVALID_ARG;
    const QuantArgs a{x, x_stride, q_stride, norm_w, q, scales, T, K, eps};
    type == ANE_TYPE_F32 ? launch_quantize<float>(a, (hipStream_t)stream) : launch_quantize<_Float16>(a, (hipStream_t)stream);
    ANE_HIP_CHECK_LAUNCH();
    return ANE_OK;
}

extern "C" int ane_hip_dense_i8_scaled(uint32_t T, uint32_t N, uint32_t K, const int8_t* q, uint64_t q_stride,
                                       const float* q_scales, const int8_t* w, uint64_t w_stride, const float* w_scales,
                                       const float* bias, const void* residual, uint64_t residual_stride, int out_type,
                                       void* out, uint64_t out_stride, void* stream) {
    const int st = product_status(T, N, K, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out, out_stride);
    if (st || T == 0 || N == 0) return st;
    if (!q || !q_scales) return ANE_ERR_BAD_POINTER;
    if (off(q, 16) || q_stride % 16 || q_stride < K || q_stride >= (1ull << 31) || off(q_scales, 4)) return ANE_ERR_INVALID_ARG;
    return product(T, N, K, q, q_stride, q_scales, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out,
                   out_stride, (hipStream_t)stream);
}

extern "C" size_t ane_hip_linear_i8_workspace_size(uint32_t T, uint32_t N, uint32_t K) {
    if (T == 0 || T > kMaxRows || N == 0 || N > kMaxRows || K == 0 || K > kMaxK) return 0;
    return q_bytes(T, K) + ceil_to((uint64_t)T * 4, 256);
}

extern "C" int ane_hip_linear_i8(uint32_t T, uint32_t N, uint32_t K, int type, const void* x, uint64_t x_stride,
                                 const float* norm_w, float eps, const int8_t* w, uint64_t w_stride, const float* w_scales,
                                 const float* bias, const void* residual, uint64_t residual_stride, int out_type, void* out,
                                 uint64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    int st = tokens_status(T, K, type, x, x_stride, norm_w, eps);
    if (!st) st = product_status(T, N, K, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out, out_stride);
    if (st || T == 0 || N == 0) return st;
    if (!workspace || off(workspace, 256) || workspace_bytes < ane_hip_linear_i8_workspace_size(T, N, K)) return ANE_ERR_WORKSPACE;
    int8_t* q = static_cast<int8_t*>(workspace);
    float* qs = reinterpret_cast<float*>(q + q_bytes(T, K));
    st = ane_hip_quantize_tokens(T, K, type, x, x_stride, norm_w, eps, q, row_bytes(K), qs, stream);
    if (st) return st;
    return product(T, N, K, q, row_bytes(K), qs, w, w_stride, w_scales, bias, residual, residual_stride, out_type, out,
                   out_stride, (hipStream_t)stream);
}
