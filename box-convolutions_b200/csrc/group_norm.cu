// Group normalisation with an activation: out = act(weight * (x - mean) * rstd + bias), mean and variance over a sample's
// group of D = C / G channels and P pixels, L = D * P values.
//
// This file: which kernels serve a call (vectors of 16 bytes: group_norm_planes.cu, group_norm_last.cu), the general ones, and
// the channels' sums over the samples.
//
// General forward, one CTA a group: the mean, then the squares about it (a sum of squares minus a squared mean loses every digit
// where the mean is large), then the outputs.  Backward, with xhat = (x - mean) * rstd and dz = grad * act'(weight xhat + bias):
//   S1 = sum dz and S2 = sum dz * xhat for each channel,
//   grad_input = rstd * (weight dz - (sum_c weight S1 + xhat * sum_c weight S2) / L),
//   grad_weight = sum_n S2,  grad_bias = sum_n S1.
#include "bc_norm.cuh"

namespace bc {

namespace {

constexpr int kThreads = 256;

// Sum over the CTA, the same value in all threads; `scratch` holds a word per warp.
__device__ __forceinline__ double block_sum(double v, double *scratch)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0;
    for (int i = 0; i < kThreads / 32; ++i) t += scratch[i];
    return t;
}

// Walks a group's values: f(offset from the tensor's start, channel of the group).
template <bool LAST, typename F>
__device__ __forceinline__ void walk(int64_t n, int g, int D, int C, int64_t P, F &&f)
{
    const int64_t L = D * P;
    if (LAST) {
        const int64_t base = n * P * C + (int64_t)g * D;
        for (int64_t e = threadIdx.x; e < L; e += kThreads) {
            const int64_t p = e / D;
            const int d = (int)(e - p * D);
            f(base + p * C + d, d);
        }
    } else {
        const int64_t base = (n * C + (int64_t)g * D) * P;
        for (int64_t e = threadIdx.x; e < L; e += kThreads) f(base + e, (int)(e / P));
    }
}

template <typename T, int ACT, bool LAST>
__global__ void __launch_bounds__(kThreads) norm_forward_kernel(const T *__restrict__ x, const T *__restrict__ weight,
                                                                const T *__restrict__ bias, T *__restrict__ out, float *__restrict__ stats,
                                                                NormShape s)
{
    __shared__ double scratch[kThreads / 32];
    const int64_t n = blockIdx.x / s.G;
    const int g = (int)(blockIdx.x - n * s.G), D = s.C / s.G;
    grid_dependency_wait();
    double sum = 0;
    walk<LAST>(n, g, D, s.C, s.P, [&](int64_t at, int) { sum += to_float(x[at]); });
    const float mean = (float)(block_sum(sum, scratch) / ((double)D * s.P));
    double squares = 0;
    walk<LAST>(n, g, D, s.C, s.P, [&](int64_t at, int) {
        const float d = to_float(x[at]) - mean;
        squares += d * d;
    });
    const float rstd = rsqrtf((float)(block_sum(squares, scratch) / ((double)D * s.P)) + s.eps);
    if (stats && threadIdx.x == 0) {
        stats[2 * (int64_t)blockIdx.x] = mean;
        stats[2 * (int64_t)blockIdx.x + 1] = rstd;
    }
    walk<LAST>(n, g, D, s.C, s.P, [&](int64_t at, int d) {
        const float w = weight ? to_float(weight[g * D + d]) : 1.f, b = bias ? to_float(bias[g * D + d]) : 0.f;
        out[at] = from_float<T>(activate<ACT, T>((to_float(x[at]) - mean) * rstd * w + b));
    });
}

template <typename T, int ACT, bool LAST>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(const T *__restrict__ x, const T *__restrict__ weight,
                                                                 const T *__restrict__ bias, const float *__restrict__ stats,
                                                                 const T *__restrict__ grad, T *__restrict__ grad_input,
                                                                 float *__restrict__ sums, NormShape s)
{
    __shared__ double scratch[kThreads / 32];
    const int64_t n = blockIdx.x / s.G;
    const int g = (int)(blockIdx.x - n * s.G), D = s.C / s.G;
    grid_dependency_wait();
    const float mean = stats[2 * (int64_t)blockIdx.x], rstd = stats[2 * (int64_t)blockIdx.x + 1];
    double all1 = 0, all2 = 0;
    for (int d = 0; d < D; ++d) {
        const int c = g * D + d;
        const float w = weight ? to_float(weight[c]) : 1.f, b = bias ? to_float(bias[c]) : 0.f;
        double s1 = 0, s2 = 0;
        for (int64_t p = threadIdx.x; p < s.P; p += kThreads) {
            const int64_t at = LAST ? (n * s.P + p) * s.C + c : (n * s.C + c) * s.P + p;
            const float unit = (to_float(x[at]) - mean) * rstd, dz = times_slope<ACT, T>(to_float(grad[at]), unit * w + b);
            s1 += dz;
            s2 += dz * unit;
        }
        s1 = block_sum(s1, scratch);
        s2 = block_sum(s2, scratch);
        if (threadIdx.x == 0) {
            sums[2 * (n * s.C + c)] = (float)s1;
            sums[2 * (n * s.C + c) + 1] = (float)s2;
        }
        all1 += w * s1;
        all2 += w * s2;
    }
    if (!grad_input) return;
    const float a1 = (float)(all1 / ((double)D * s.P)), a2 = (float)(all2 / ((double)D * s.P));
    walk<LAST>(n, g, D, s.C, s.P, [&](int64_t at, int d) {
        const float w = weight ? to_float(weight[g * D + d]) : 1.f, b = bias ? to_float(bias[g * D + d]) : 0.f;
        const float unit = (to_float(x[at]) - mean) * rstd, dz = times_slope<ACT, T>(to_float(grad[at]), unit * w + b);
        grad_input[at] = from_float<T>(rstd * (w * dz - a1 - unit * a2));
    });
}

// The rows' S1 and S2 added up in a fixed order: a lane a channel, 32 rows at a time.
constexpr int kFinish = 1024;
template <typename T>
__global__ void __launch_bounds__(kFinish) norm_finish_kernel(const float *__restrict__ sums, T *__restrict__ grad_weight,
                                                             T *__restrict__ grad_bias, int rows, int C)
{
    __shared__ float2 part[kFinish / 32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    grid_dependency_wait();
    float2 t = make_float2(0.f, 0.f);
    if (c < C) {
        const float2 *from = reinterpret_cast<const float2 *>(sums) + c;
#pragma unroll 8
        for (int i = warp; i < rows; i += kFinish / 32) {
            const float2 v = from[(int64_t)i * C];
            t.x += v.x;
            t.y += v.y;
        }
    }
    part[warp][lane] = t;
    __syncthreads();
    // a warp a channel
    float2 v = part[lane][warp];
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    const int mine = blockIdx.x * 32 + warp;
    if (lane == 0 && mine < C) {
        if (grad_bias) grad_bias[mine] = from_float<T>(v.x);
        if (grad_weight) grad_weight[mine] = from_float<T>(v.y);
    }
}

// f(T(), activation, layout) for the shape's.
template <typename F>
int dispatch(const NormShape &s, F &&f)
{
    return with_type(s.io_kind, [&](auto t) {
        return with_activation(s.act, [&](auto act) {
            return s.last ? f(t, act, std::true_type()) : f(t, act, std::false_type());
        });
    });
}

// How a call runs: planes of vectors, rows of vectors, or (channels last with more than 1024 places of a vector among the
// channels; arrays off a vector's boundary) a CTA a group, value by value.
struct Route {
    bool planes = false, rows = false;
    NormPlanes p{};
    NormRows r{};
    Route(const NormShape &s, bool aligned)
    {
        if (!aligned) return;
        if (s.last) {
            rows = plan_rows(s, &r);
        } else {
            plan_planes(s, &p);
            planes = true;
        }
    }
    int64_t sums(const NormShape &s) const { return (int64_t)s.N * (rows ? r.k : planes ? p.k : 1); }      // rows of S1, S2
};

bool aligned(const void *a, const void *b, const void *c = nullptr)
{
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}

}  // namespace

size_t group_norm_workspace(const NormShape &s, int need_mask)
{
    // (the larger of the vectors' and the general way's: the query does not know the arrays)
    const Route q(s, true);
    const size_t general = need_mask ? (size_t)s.N * s.C * 8 : 0;
    return std::max(general, q.rows ? rows_sums_bytes(s, q.r, need_mask != 0) : q.planes ? planes_sums_bytes(s, q.p, need_mask != 0) : 0);
}

int launch_group_norm_forward(const NormShape &s, const void *x, const void *weight, const void *bias, void *out, float *stats,
                              void *ws, cudaStream_t stream)
{
    const int64_t groups = (int64_t)s.N * s.G;
    if (groups > INT32_MAX) return BC_ERR_BAD_SHAPE;
    const Route q(s, aligned(x, out));
    if (q.rows) return launch_norm_rows_forward(s, q.r, x, weight, bias, out, stats, ws, stream);
    if (q.planes) return launch_norm_planes_forward(s, q.p, x, weight, bias, out, stats, ws, stream);
    return dispatch(s, [&](auto t, auto act, auto last) {
        using T = decltype(t);
        const LaunchScope scope(KID_NORM_FORWARD, stream);
        launch_overlapped(norm_forward_kernel<T, act(), last()>, (unsigned)groups, kThreads, 0, stream, (const T *)x, (const T *)weight,
                          (const T *)bias, (T *)out, stats, s);
        return check_launch("norm_forward_kernel");
    });
}

int launch_group_norm_backward(const NormShape &s, const void *x, const void *weight, const void *bias, const float *stats,
                               const void *grad, int need_mask, void *grad_input, void *grad_weight, void *grad_bias, void *ws,
                               cudaStream_t stream)
{
    const int64_t groups = (int64_t)s.N * s.G;
    if (groups > INT32_MAX) return BC_ERR_BAD_SHAPE;
    void *gx = (need_mask & BC_NEED_GN_INPUT) ? grad_input : nullptr;
    const Route q(s, aligned(x, grad, gx));
    if (q.sums(s) > INT32_MAX) return BC_ERR_BAD_SHAPE;
    int e;
    if (q.rows) e = launch_norm_rows_backward(s, q.r, x, weight, bias, stats, grad, gx, (float *)ws, stream);
    else if (q.planes) e = launch_norm_planes_backward(s, q.p, x, weight, bias, stats, grad, gx, (float *)ws, stream);
    else e = dispatch(s, [&](auto t, auto act, auto last) {
        using T = decltype(t);
        const LaunchScope scope(KID_NORM_BACKWARD, stream);
        launch_overlapped(norm_backward_kernel<T, act(), last()>, (unsigned)groups, kThreads, 0, stream, (const T *)x, (const T *)weight,
                          (const T *)bias, stats, (const T *)grad, (T *)gx, (float *)ws, s);
        return check_launch("norm_backward_kernel");
    });
    if (e || !(need_mask & (BC_NEED_GN_WEIGHT | BC_NEED_GN_BIAS))) return e;
    return with_type(s.io_kind, [&](auto t) {
        using T = decltype(t);
        const LaunchScope scope(KID_NORM_FINISH, stream);
        launch_overlapped(norm_finish_kernel<T>, (unsigned)((s.C + 31) / 32), kFinish, 0, stream, (const float *)ws, 
                          (need_mask & BC_NEED_GN_WEIGHT) ? (T *)grad_weight : nullptr,
                          (need_mask & BC_NEED_GN_BIAS) ? (T *)grad_bias : nullptr, (int)q.sums(s), s.C);
        return check_launch("norm_finish_kernel");
    });
}

}  // namespace bc
