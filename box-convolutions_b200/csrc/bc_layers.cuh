// What the layers around a box convolution share (pointwise.cu, pointwise_mma.cu, group_norm.cu): storage types,
// activations, vectors of values, launchers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <type_traits>

#include "bc_common.cuh"
#include "bc_smem_walk.cuh"

namespace bc {

// ---- storage types: every value is widened to float as it is read and rounded once as it is written
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit values of a word, and back.
__device__ __forceinline__ void widen2(uint32_t w, float &a, float &b, __nv_bfloat16)
{
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void widen2(uint32_t w, float &a, float &b, __half)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    a = f.x;
    b = f.y;
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half)
{
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// 16 bytes of values.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &w, float (&v)[kVec<T>])
{
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(w.x);
        v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z);
        v[3] = __uint_as_float(w.w);
    } else {
        widen2(w.x, v[0], v[1], T());
        widen2(w.y, v[2], v[3], T());
        widen2(w.z, v[4], v[5], T());
        widen2(w.w, v[6], v[7], T());
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[kVec<T>])
{
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else
        return make_uint4(narrow2(v[0], v[1], T()), narrow2(v[2], v[3], T()), narrow2(v[4], v[5], T()), narrow2(v[6], v[7], T()));
}

// ---- activations (BC_ACT_*).  A NaN stays one in all of them; the ReLU's slope at zero and at NaN is 0, as PyTorch's.
// The exponential and the quotients are CUDA's own in full precision for float tensors.  16-bit tensors take the fast
// forms: their errors, some 2^-21 for arguments that matter, are far below the rounding at the end (2^-9, 2^-12).
template <typename T>
__device__ __forceinline__ float exp_of(float v) { return sizeof(T) == 4 ? expf(v) : __expf(v); }
template <typename T>
__device__ __forceinline__ float quotient(float a, float b) { return sizeof(T) == 4 ? a / b : __fdividef(a, b); }

// The normal distribution function, and its density times sqrt(2 pi).  Float tensors: CUDA's error function.  16-bit ones:
// Abramowitz and Stegun's 7.1.26, five terms of 1 / (1 + 0.3275911 |x|) times exp(-x^2), x = z / sqrt(2), off by 7.5e-8 at
// most: a third of the instructions, and the exponential serves the density too.
template <typename T>
__device__ __forceinline__ float normal(float z, float &density)
{
    if constexpr (sizeof(T) == 4) {
        density = expf(-0.5f * z * z);
        return 0.5f * (1.f + erff(z * 0.70710678118654752f));
    } else {
        density = __expf(-0.5f * z * z);
        const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
        float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
        p = fmaf(p, t, 0.5f * 1.421413741f);
        p = fmaf(p, t, 0.5f * -0.284496736f);
        p = fmaf(p, t, 0.5f * 0.254829592f) * t * density;      // the smaller of the two tails
        return z < 0.f ? p : 1.f - p;
    }
}

template <int ACT, typename T>
__device__ __forceinline__ float activate(float z)
{
    if constexpr (ACT == BC_ACT_RELU) return z <= 0.f ? 0.f : z;
    if constexpr (ACT == BC_ACT_SILU) return quotient<T>(z, 1.f + exp_of<T>(-z));
    if constexpr (ACT == BC_ACT_GELU) {
        float density;
        return z * normal<T>(z, density);
    }
    return z;
}
template <int ACT, typename T>
__device__ __forceinline__ float slope(float z)
{
    if constexpr (ACT == BC_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == BC_ACT_SILU) {
        const float s = quotient<T>(1.f, 1.f + exp_of<T>(-z));
        return s * (1.f + z * (1.f - s));
    }
    if constexpr (ACT == BC_ACT_GELU) {
        float density;
        const float p = normal<T>(z, density);
        return fmaf(z * 0.39894228040143268f, density, p);
    }
    return 1.f;
}

// A runtime activation as a template argument: f(std::integral_constant<int, ACT>).
template <typename F>
inline int with_activation(int act, F &&f)
{
    switch (act) {
        case BC_ACT_NONE: return f(std::integral_constant<int, BC_ACT_NONE>());
        case BC_ACT_RELU: return f(std::integral_constant<int, BC_ACT_RELU>());
        case BC_ACT_SILU: return f(std::integral_constant<int, BC_ACT_SILU>());
        case BC_ACT_GELU: return f(std::integral_constant<int, BC_ACT_GELU>());
        default: return BC_ERR_UNSUPPORTED;
    }
}
// The same for a storage type (BC_IO_*): f(T()).
template <typename F>
inline int with_type(int io_kind, F &&f)
{
    switch (io_kind) {
        case BC_IO_F32: return f(float());
        case BC_IO_F16: return f(__half());
        case BC_IO_BF16: return f(__nv_bfloat16());
        default: return BC_ERR_UNSUPPORTED;
    }
}

// ---- launchers
inline int io_size(int io_kind) { return io_kind == BC_IO_F32 ? 4 : 2; }

struct NormShape {
    int N, C, G;             // G groups of C / G channels
    int64_t P;               // pixels of a plane
    bool last;               // channels last: (N, P, C); planes (N, C, P) otherwise
    int io_kind, act;
    float eps;
};
size_t group_norm_workspace(const NormShape &s, int need_mask);
int launch_group_norm_forward(const NormShape &s, const void *x, const void *weight, const void *bias, void *out, float *stats,
                              void *ws, cudaStream_t stream);
int launch_group_norm_backward(const NormShape &s, const void *x, const void *weight, const void *bias, const float *stats,
                               const void *grad, int need_mask, void *grad_input, void *grad_weight, void *grad_bias, void *ws,
                               cudaStream_t stream);

struct PointwiseShape {
    int N, Ci, Co;
    int64_t P;
    bool last;
    int io_kind, act;
};
size_t pointwise_workspace(const PointwiseShape &s, int need_mask);
int launch_pointwise_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual, void *out,
                             cudaStream_t stream);
int launch_pointwise_backward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                              const void *grad, int need_mask, void *grad_input, void *grad_weight, void *grad_bias,
                              void *grad_residual, void *ws, cudaStream_t stream);

}  // namespace bc
