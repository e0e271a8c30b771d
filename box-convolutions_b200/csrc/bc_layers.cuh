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

// The same as pairs for the packed arithmetic of two floats an instruction.
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4 &w, f2_t (&v)[kVec<T> / 2])
{
    float f[kVec<T>];
    unpack<T>(w, f);
#pragma unroll
    for (int j = 0; j < kVec<T> / 2; ++j) v[j] = pack2(f[2 * j], f[2 * j + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const f2_t (&v)[kVec<T> / 2])
{
    float f[kVec<T>];
#pragma unroll
    for (int j = 0; j < kVec<T> / 2; ++j) unpack2(v[j], f[2 * j], f[2 * j + 1]);
    return pack<T>(f);
}
__device__ __forceinline__ f2_t both(float v) { return pack2(v, v); }

// What a rounding to 16 bits leaves of a value; of one whose rounding is not finite, nothing.
template <typename T>
__device__ __forceinline__ float left_by_rounding(float v, T rounded)
{
    const float left = v - to_float(rounded);
    return fabsf(left) < INFINITY ? left : 0.f;
}
template <typename T>
__device__ __forceinline__ uint4 left_by_rounding(const f2_t (&v)[kVec<T> / 2], const uint4 &rounded)
{
    f2_t r[kVec<T> / 2];
    unpack_pairs<T>(rounded, r);
#pragma unroll
    for (int j = 0; j < kVec<T> / 2; ++j) {
        float a, b;
        unpack2(sub2(v[j], r[j]), a, b);
        r[j] = pack2(fabsf(a) < INFINITY ? a : 0.f, fabsf(b) < INFINITY ? b : 0.f);
    }
    return pack_pairs<T>(r);
}

// ---- activations (BC_ACT_*), of two values at a time.  A NaN stays one in all of them; the ReLU's slope at zero and at NaN
// is 0, as PyTorch's.  Exponentials and quotients are the hardware's powers of two and reciprocals (2^-22 and 2^-23): with
// CUDA's own functions a normalisation of float planes with SiLU was bound by instructions, (256,32,64,128) forward 148 us.
// Float tensors carry the rounding of the exponent along; 16-bit ones, whose results are rounded to 2^-9 or 2^-12, do not.
// Their normal distribution function, below zero, is exp(-z^2 / 2) times t (c1 + ... + c6 t^5), t = 1 / (1 + 0.29 |z|): the form of
// Abramowitz and Stegun's 7.1.26 with a term more, its coefficients fitted by weighted least squares (Lawson's iteration) to errors of
// 4.8e-8 or, in the tail down to -13, 2^-13 of the function.  (7.1.26 itself is off by 7.5e-8, and by 4 % of the tail.)  With the
// arithmetic's errors it is off by 2.5e-7 and 10^-4 at most over all 16-bit arguments.
__device__ __forceinline__ float power_of_two(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocal(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
template <typename F>
__device__ __forceinline__ f2_t of_each(f2_t v, F &&f)
{
    float a, b;
    unpack2(v, a, b);
    return pack2(f(a), f(b));
}
template <typename F>
__device__ __forceinline__ f2_t of_each2(f2_t v, f2_t w, F &&f)
{
    float a, b, c, d;
    unpack2(v, a, b);
    unpack2(w, c, d);
    return pack2(f(a, c), f(b, d));
}
// Of two values: exp(-|z|) = e k, `a` = 1 / (1 + exp(-|z|)).  Their logistic function is `a` from zero on and e k a below, where it
// so keeps its relative accuracy: to the smallest float for float (k = 2^-64 below -42, where e would soon be no normal number, 1 elsewhere), for bfloat16
// down to -96, below which z times it is no normal number, for float16 down to 2^-126, which is far below its smallest.  16-bit tensors:
// one reciprocal for two, 1 / a = b / (a b), since reciprocals and powers of two are what their normalisations wait for; a
// value then depends on its neighbour in its 22nd bit (not on a NaN, which is taken for a large number here).  An exp(-z) that ended at
// 2^60 made 0 of what lies below -41.6; (256,32,64,128) f32 forward took 113 us with it, 119 now, backward 181 and 190.
template <typename T>
__device__ __forceinline__ void logistic_parts2(f2_t z, f2_t &e, f2_t &k, f2_t &a)
{
    k = both(1.f);
    if constexpr (sizeof(T) == 4) {
        // (infinities and NaN have no rounding to carry along)
        const f2_t size = of_each(z, [](float v) { return fminf(fabsf(v), 1e4f); }), t = mul2(size, both(-1.44269504f));
        e = of_each2(z, t, [](float v, float w) { return power_of_two(v < -42.f ? w + 64.f : w); });      // (an exact sum: multiples of 2^-18)
        k = of_each(z, [](float v) { return v < -42.f ? 0x1p-64f : 1.f; });
        // minus the exponent's rounding and what 1.44269504f lacks of log2(e)
        const f2_t rest = fma2(size, both(1.9259629911e-8f), fma2(size, both(1.44269504f), t));
        e = fma2(e, mul2(rest, both(-0.69314718f)), e);
        a = of_each(fma2(e, k, both(1.f)), reciprocal);
    } else {
        const f2_t size = of_each(z, [](float v) { return fminf(fabsf(v), 1e4f); });
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {      // (a square: the power of two itself ends at 2^-126)
            e = of_each(mul2(size, both(-0.5f * 1.44269504f)), power_of_two);
            e = mul2(e, e);
        } else {
            e = of_each(mul2(size, both(-1.44269504f)), power_of_two);
        }
        float x, y;
        unpack2(add2(e, both(1.f)), x, y);
        const float r = reciprocal(x * y);
        a = pack2(y * r, x * r);
    }
}
// v where z is below zero, 1 elsewhere
__device__ __forceinline__ f2_t below_zero(f2_t z, f2_t v)
{
    return of_each2(z, v, [](float a, float b) { return a < 0.f ? b : 1.f; });
}
// The normal distribution function, and exp(-z^2 / 2).
template <typename T>
__device__ __forceinline__ f2_t normal2(f2_t z, f2_t &density)
{
    if constexpr (sizeof(T) == 4) {
        density = of_each(z, [](float v) { return expf(-0.5f * v * v); });
        // (off by 2^-24 of 1, so that the tail's digits are lost from -3 on, as PyTorch's; with erfcf in its place, or below -2.5
        // alone, (256,32,64,128) planes took 166 to 175 us forward instead of 138, and 326 to 331 backward instead of 244)
        return of_each(z, [](float v) { return 0.5f * (1.f + erff(v * 0.70710678118654752f)); });
    }
    density = of_each(mul2(mul2(z, z), both(-0.5f * 1.4426950408889634f)), power_of_two);
    const f2_t size = of_each(z, [](float v) { return fabsf(v); });
    const f2_t t = of_each(fma2(size, both(0.29f), both(1.f)), reciprocal);
    f2_t p = fma2(both(-0.0896348559f), t, both(0.287845366f));
    p = fma2(p, t, both(-0.0973541001f));
    p = fma2(p, t, both(0.182338251f));
    p = fma2(p, t, both(0.0998317281f));
    p = fma2(p, t, both(0.116973562f));
    p = mul2(mul2(p, t), density);      // the smaller of the two tails
    float z0, z1, p0, p1;
    unpack2(z, z0, z1);
    unpack2(p, p0, p1);
    return pack2(z0 < 0.f ? p0 : 1.f - p0, z1 < 0.f ? p1 : 1.f - p1);
}

template <int ACT, typename T>
__device__ __forceinline__ f2_t activate2(f2_t z)
{
    if constexpr (ACT == BC_ACT_RELU) return of_each(z, [](float v) { return v <= 0.f ? 0.f : v; });
    if constexpr (ACT == BC_ACT_SILU) {
        f2_t e, k, a;
        logistic_parts2<T>(z, e, k, a);
        if constexpr (sizeof(T) == 2) return mul2(z, mul2(a, below_zero(z, e)));
        return mul2(mul2(mul2(z, below_zero(z, e)), a), k);      // (k last: a product that underflows is rounded once)
    }
    if constexpr (ACT == BC_ACT_GELU) {
        f2_t density;
        return mul2(z, normal2<T>(z, density));
    }
    return z;
}
// g times the activation's slope
template <int ACT, typename T>
__device__ __forceinline__ f2_t times_slope2(f2_t g, f2_t z)
{
    if constexpr (ACT == BC_ACT_RELU) {
        float g0, g1, z0, z1;
        unpack2(g, g0, g1);
        unpack2(z, z0, z1);
        return pack2(z0 > 0.f ? g0 : 0.f, z1 > 0.f ? g1 : 0.f);
    }
    if constexpr (ACT == BC_ACT_SILU) {
        f2_t e, k, a;
        logistic_parts2<T>(z, e, k, a);
        if constexpr (sizeof(T) == 2) {
            const f2_t s = mul2(a, below_zero(z, e)), u = fma2(s, both(-1.f), both(1.f));
            return mul2(mul2(g, s), fma2(z, u, both(1.f)));
        }
        // logistic(z) (1 + z logistic(-z))
        const f2_t below = below_zero(z, e), other = mul2(a, of_each2(z, mul2(e, k), [](float v, float w) { return v < 0.f ? 1.f : w; }));
        return mul2(mul2(mul2(mul2(g, below), a), fma2(z, other, both(1.f))), k);
    }
    if constexpr (ACT == BC_ACT_GELU) {
        f2_t density;
        const f2_t p = normal2<T>(z, density);
        return mul2(g, fma2(mul2(z, both(0.39894228040143268f)), density, p));
    }
    return g;
}
template <int ACT, typename T>
__device__ __forceinline__ float activate(float z)
{
    float a, b;
    unpack2(activate2<ACT, T>(pack2(z, 0.f)), a, b);
    return a;
}
template <int ACT, typename T>
__device__ __forceinline__ float times_slope(float g, float z)
{
    float a, b;
    unpack2(times_slope2<ACT, T>(pack2(g, 0.f), pack2(z, 0.f)), a, b);
    return a;
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
// A 16-bit dz = grad * slope is two tensors, its rounding and `rest`, the rounding of what that leaves (null: one tensor is all of dz).
// The products on the tensor cores (pointwise_mma.cu): 16-bit types, rows and arrays on 16 bytes.
bool pointwise_mma_suits(const PointwiseShape &s, bool input);
bool pointwise_mma_aligned(const void *a, const void *b, const void *c = nullptr, const void *d = nullptr, const void *e = nullptr);
int launch_pointwise_mma_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                                 void *out, cudaStream_t stream);
// sums: pointwise_mma_sums_rows() rows of Co floats, sums of dz to be added, or null
int pointwise_mma_sums_rows(const PointwiseShape &s);
int launch_pointwise_mma_slope(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                               const void *grad, void *dz, void *rest, float *sums, cudaStream_t stream);
int launch_pointwise_mma_input(const PointwiseShape &s, const void *dz, const void *rest, const void *weight, void *grad_input,
                               cudaStream_t stream);
// Floats of a row of partial sums of grad_weight, Co * Ci and the Co of grad_bias: whole vectors, so that every row starts on one.
__host__ __device__ inline int64_t pointwise_partial_stride(int Co, int Ci) { return ((int64_t)Co * Ci + Co + 3) / 4 * 4; }
// rows of partial sums (0: not for this kernel)
int pointwise_mma_weight_splits(const PointwiseShape &s);
int launch_pointwise_mma_weight(const PointwiseShape &s, const void *dz, const void *rest, const void *x, float *partial, bool sums,
                                cudaStream_t stream);
int read_wait_timeouts_mma(int *count);

// The same with operands made by threads (pointwise_split.cu): floats as sums of bf16, rows of any alignment.
bool pointwise_split_suits(const PointwiseShape &s, bool input);
int pointwise_split_sums_rows(const PointwiseShape &s);
int launch_pointwise_split_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                                   void *out, cudaStream_t stream);
int launch_pointwise_split_slope(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                                 const void *grad, void *dz, void *rest, float *sums, cudaStream_t stream);
int launch_pointwise_split_input(const PointwiseShape &s, const void *dz, const void *rest, const void *weight, void *grad_input,
                                 cudaStream_t stream);
int pointwise_split_weight_splits(const PointwiseShape &s, bool rest);      // (no more with `rest` than without)
int launch_pointwise_split_weight(const PointwiseShape &s, const void *dz, const void *rest, const void *x, float *partial, bool sums,
                                  cudaStream_t stream);
int read_wait_timeouts_split(int *count);

size_t pointwise_workspace(const PointwiseShape &s, int need_mask);
int launch_pointwise_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual, void *out,
                             cudaStream_t stream);
int launch_pointwise_backward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                              const void *grad, int need_mask, void *grad_input, void *grad_weight, void *grad_bias,
                              void *grad_residual, void *ws, cudaStream_t stream);

}  // namespace bc
