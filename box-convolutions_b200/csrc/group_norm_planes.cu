// Group normalisation of planes, a unit being a sample's group: C / G adjacent planes (bc_norm.cuh).
//
// A unit's planes are cut into pieces of at most kPiece vectors, a CTA's pieces dealt out to its warps: a warp has one
// channel's weight and bias at a time and one channel's sums.  Vectors lie on 16-byte boundaries of the tensor; the values in
// front of a piece's first whole vector and behind its last go to a lane each, so planes of odd sizes are read like others.
#include "bc_norm.cuh"

namespace bc {

namespace {

constexpr int kPiece = 256;            // vectors: eight a lane
constexpr int kMostPieces = 2048;      // of a CTA: their sums are kept in shared memory
// Bytes that are worth a CTA.  A CTA a group, or a cluster of two where a group is longer than that; 256 samples, 8 groups, SiLU, f32,
// us forward and backward by the size of a group:
//     128 KB  119 + 191 (one), 156 + 201 (two)     136 KB  185 + 308, 256 + 355     192 KB  176 + 312, 215 + 307
//     256 KB  243 + 407 (one), 245 + 403 (two)     384 KB  366 + 622 (two), 366 + 622 (four), 435 + 615 (eight)
// and bf16, 160 KB, 178 + 328 and 235 + 348: up to 256 KB one is as fast or faster, beyond they are alike.
constexpr int64_t kPlaneSlice = 256 << 10;
// Bytes of a CTA up to which a cluster of eight serves a group where that leaves SMs without work: (2,64,256,512) bf16, 8 groups of
// 2 MB, SiLU: 41 us forward and 61 backward with 256 KB a CTA; in two launches over the whole GPU 22 + 22 and 31 + 31, each timed
// by itself, of which some 5 are the timing.
constexpr int64_t kClusterSlice = 128 << 10;

// Where a piece lies: values [a, b) of the tensor, whole vectors [v0, v1) of those.
template <typename T>
struct Piece {
    static constexpr int V = kVec<T>;
    int64_t a, b, v0, v1;
    int channel;              // of the unit
    __device__ __forceinline__ Piece(const NormShape &s, const NormPlanes &plan, int64_t first_plane, int piece)
    {
        channel = (unsigned)piece / (unsigned)plan.chunks;
        const int64_t from = (int64_t)(piece - channel * plan.chunks) * plan.chunk;
        a = (first_plane + channel) * s.P + from;
        b = a + min((int64_t)plan.chunk, s.P - from);
        v0 = min((a + V - 1) & ~(int64_t)(V - 1), b);
        v1 = max(b & ~(int64_t)(V - 1), v0);
    }
    // The lane's single value, or -1.
    __device__ __forceinline__ int64_t edge(int lane) const
    {
        const int head = (int)(v0 - a);
        return lane < head ? a + lane : lane - head < (int)(b - v1) ? v1 + lane - head : -1;
    }
    // f(how many, offset of the first): U vectors of the lane at a time, 32 vectors apart.
    template <int U, typename F>
    __device__ __forceinline__ void each(int lane, F &&f) const
    {
        int64_t at = v0 + lane * V;
        for (; at + (U - 1) * 32 * V < v1; at += U * 32 * V) f(std::integral_constant<int, U>(), at);
        for (; at < v1; at += 32 * V) f(std::integral_constant<int, 1>(), at);
    }
};

template <typename T, int ACT, int STEP>
__global__ void __launch_bounds__(512, 2) norm_planes_forward_kernel(const T *__restrict__ x, const T *__restrict__ weight,
                                                                     const T *__restrict__ bias, T *__restrict__ out,
                                                                     float *__restrict__ stats, float *__restrict__ ws, NormShape s,
                                                                     NormPlanes plan)
{
    constexpr int V = kVec<T>;
    __shared__ float warp_moments[16][3], own[3];
    __shared__ float2 result;
    const int D = s.C / s.G, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned index = blockIdx.x / (unsigned)plan.k;
    const int64_t unit = index, first_plane = unit * D;
    const int rank = (int)(blockIdx.x - index * plan.k);
    const int begin = rank * plan.per, end = min(D * plan.chunks, begin + plan.per);
    grid_dependency_wait();

    if (STEP != NORM_RESULTS) {
        Moments m{0.f, 0.f, 0.f};
        for (int i = begin + warp; i < end; i += warps) {
            const Piece<T> piece(s, plan, first_plane, i);
            piece.template each<4>(lane, [&](auto many, int64_t at) {
                constexpr int M = decltype(many)::value;
                uint4 raw[M];
#pragma unroll
                for (int u = 0; u < M; ++u) raw[u] = *reinterpret_cast<const uint4 *>(x + at + u * 32 * V);
#pragma unroll
                for (int u = 0; u < M; ++u) {
                    f2_t v[V / 2], sum, squares = both(0.f);
                    float a, b;
                    unpack_pairs<T>(raw[u], v);
                    sum = v[0];
#pragma unroll
                    for (int j = 1; j < V / 2; ++j) sum = add2(sum, v[j]);
                    unpack2(sum, a, b);
                    const float mean = (a + b) * (1.f / V);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {
                        const f2_t d = sub2(v[j], both(mean));
                        squares = fma2(d, d, squares);
                    }
                    unpack2(squares, a, b);
                    m = merged(m, {(float)V, mean, (a + b) * (1.f / V)});
                }
            });
            const int64_t at = piece.edge(lane);
            if (at >= 0) m = merged(m, {1.f, to_float(x[at]), 0.f});
        }
        m = warp_merged(m);
        if (lane == 0) {
            warp_moments[warp][0] = m.n;
            warp_moments[warp][1] = m.mean;
            warp_moments[warp][2] = m.var;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < warps; ++i) m = merged(m, {warp_moments[i][0], warp_moments[i][1], warp_moments[i][2]});
            float *to = STEP == NORM_SUMS ? ws + (unit * plan.k + rank) * 3 : own;
            to[0] = m.n;
            to[1] = m.mean;
            to[2] = m.var;
        }
        if (STEP == NORM_SUMS) return;
    }
    if (STEP == NORM_WHOLE) {
        if (plan.k > 1) cluster_sync();
        if (threadIdx.x == 0) {
            Moments m{own[0], own[1], own[2]};
            if (plan.k > 1) {
                m = {0.f, 0.f, 0.f};
                for (int i = 0; i < plan.k; ++i) {
                    const uint32_t at = cluster_map(smem_u32(own), i);
                    m = merged(m, {cluster_load(at), cluster_load(at + 4), cluster_load(at + 8)});
                }
            }
            result = make_float2(m.mean, rsqrtf(m.var + s.eps));
        }
        if (plan.k > 1) cluster_sync();      // (nobody leaves while its moments are read)
        else __syncthreads();
    } else {
        if (warp == 0) {
            Moments m{0.f, 0.f, 0.f};
            for (int i = lane; i < plan.k; i += 32) {
                const float *from = ws + (unit * plan.k + i) * 3;
                m = merged(m, {__ldg(from), __ldg(from + 1), __ldg(from + 2)});
            }
            m = warp_merged(m);
            if (lane == 0) result = make_float2(m.mean, rsqrtf(m.var + s.eps));
        }
        __syncthreads();
    }
    const float mean = result.x, rstd = result.y;
    if (stats && rank == 0 && threadIdx.x == 0) reinterpret_cast<float2 *>(stats)[unit] = make_float2(mean, rstd);
    const int c0 = (int)(index % (unsigned)s.G) * D;
    for (int i = begin + warp; i < end; i += warps) {
        const Piece<T> piece(s, plan, first_plane, i);
        const float a = weight ? rstd * to_float(weight[c0 + piece.channel]) : rstd, b = bias ? to_float(bias[c0 + piece.channel]) : 0.f;
        piece.template each<4>(lane, [&](auto many, int64_t at) {
            constexpr int M = decltype(many)::value;
            uint4 raw[M];
#pragma unroll
            for (int u = 0; u < M; ++u) raw[u] = *reinterpret_cast<const uint4 *>(x + at + u * 32 * V);
#pragma unroll
            for (int u = 0; u < M; ++u) {
                f2_t v[V / 2];
                unpack_pairs<T>(raw[u], v);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) v[j] = activate2<ACT, T>(fma2(sub2(v[j], both(mean)), both(a), both(b)));
                *reinterpret_cast<uint4 *>(out + at + u * 32 * V) = pack_pairs<T>(v);
            }
        });
        const int64_t at = piece.edge(lane);
        if (at >= 0) out[at] = from_float<T>(activate<ACT, T>(fmaf(to_float(x[at]) - mean, a, b)));
    }
}

// Backward: as in group_norm_last.cu, with d = x - mean, a = weight rstd, z = a d + bias and dz = grad * slope(z).
template <typename T, int ACT, int STEP>
__global__ void __launch_bounds__(512, 2) norm_planes_backward_kernel(const T *__restrict__ x, const T *__restrict__ weight,
                                                                      const T *__restrict__ bias, const float *__restrict__ stats,
                                                                      const T *__restrict__ grad, T *__restrict__ grad_input,
                                                                      float *__restrict__ sums, NormShape s, NormPlanes plan)
{
    constexpr int V = kVec<T>, U = 4;
    __shared__ float2 pieces[kMostPieces];
    __shared__ float2 of_warp[16], own, result;
    const int D = s.C / s.G, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned index = blockIdx.x / (unsigned)plan.k, sample = index / (unsigned)s.G;
    const int64_t unit = index, first_plane = unit * D, n = sample;
    const int rank = (int)(blockIdx.x - index * plan.k), c0 = (int)(index - sample * s.G) * D;
    const int begin = rank * plan.per, end = min(D * plan.chunks, begin + plan.per);
    const float count = (float)D * (float)s.P;
    grid_dependency_wait();
    const float mean = stats[2 * unit], rstd = stats[2 * unit + 1];
    auto affine = [&](int channel, float &a, float &b) {
        a = weight ? rstd * to_float(weight[c0 + channel]) : rstd;
        b = ACT != BC_ACT_NONE && bias ? to_float(bias[c0 + channel]) : 0.f;
    };

    if (STEP != NORM_RESULTS) {
        for (int i = begin + warp; i < end; i += warps) {
            const Piece<T> piece(s, plan, first_plane, i);
            float a, b;
            f2_t p1 = both(0.f), p2 = both(0.f);
            affine(piece.channel, a, b);
            piece.template each<U>(lane, [&](auto many, int64_t at) {
                constexpr int M = decltype(many)::value;
                uint4 rx[M], rg[M];
#pragma unroll
                for (int u = 0; u < M; ++u) {
                    rx[u] = *reinterpret_cast<const uint4 *>(x + at + u * 32 * V);
                    rg[u] = *reinterpret_cast<const uint4 *>(grad + at + u * 32 * V);
                }
#pragma unroll
                for (int u = 0; u < M; ++u) {
                    f2_t v[V / 2], g[V / 2];
                    unpack_pairs<T>(rx[u], v);
                    unpack_pairs<T>(rg[u], g);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) {
                        const f2_t d = sub2(v[j], both(mean)), dz = times_slope2<ACT, T>(g[j], fma2(d, both(a), both(b)));
                        p1 = add2(p1, dz);
                        p2 = fma2(dz, d, p2);
                    }
                }
            });
            float s1, s2, other;
            unpack2(p1, s1, other);
            s1 += other;
            unpack2(p2, s2, other);
            s2 += other;
            const int64_t at = piece.edge(lane);
            if (at >= 0) {
                const float d = to_float(x[at]) - mean, dz = times_slope<ACT, T>(to_float(grad[at]), fmaf(d, a, b));
                s1 += dz;
                s2 = fmaf(dz, d, s2);
            }
            s1 = warp_sum(s1);
            s2 = warp_sum(s2);
            if (lane == 0) pieces[i - begin] = make_float2(s1, s2 * rstd);
        }
        __syncthreads();
        // channels' sums over the CTA's pieces in order (none: zeros), and the group's weighted ones
        float t1 = 0.f, t2 = 0.f;
        for (int c = threadIdx.x; c < D; c += blockDim.x) {
            float2 t = make_float2(0.f, 0.f);
            for (int i = max(begin, c * plan.chunks); i < min(end, (c + 1) * plan.chunks); ++i) {
                t.x += pieces[i - begin].x;
                t.y += pieces[i - begin].y;
            }
            reinterpret_cast<float2 *>(sums)[(n * plan.k + rank) * s.C + c0 + c] = t;
            const float w = weight ? to_float(weight[c0 + c]) : 1.f;
            t1 = fmaf(w, t.x, t1);
            t2 = fmaf(w, t.y, t2);
        }
        if (STEP == NORM_SUMS) return;
        t1 = warp_sum(t1);
        t2 = warp_sum(t2);
        if (lane == 0) of_warp[warp] = make_float2(t1, t2);
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < warps; ++i) {
                t1 += of_warp[i].x;
                t2 += of_warp[i].y;
            }
            own = make_float2(t1, t2);
        }
        if (plan.k > 1) cluster_sync();
        if (threadIdx.x == 0) {
            float2 t = own;
            if (plan.k > 1) {
                t = make_float2(0.f, 0.f);
                for (int i = 0; i < plan.k; ++i) {
                    const uint32_t at = cluster_map(smem_u32(&own), i);
                    t.x += cluster_load(at);
                    t.y += cluster_load(at + 4);
                }
            }
            result = make_float2(__fdiv_rn(t.x, count), __fdiv_rn(t.y, count));
        }
        if (plan.k > 1) cluster_sync();
        else __syncthreads();
    } else {
        float t1 = 0.f, t2 = 0.f;
        for (int64_t i = threadIdx.x; i < (int64_t)plan.k * D; i += blockDim.x) {
            const int64_t at = i / D;
            const int c = c0 + (int)(i - at * D);
            const float2 v = __ldg(reinterpret_cast<const float2 *>(sums) + (n * plan.k + at) * s.C + c);
            const float w = weight ? to_float(weight[c]) : 1.f;
            t1 = fmaf(w, v.x, t1);
            t2 = fmaf(w, v.y, t2);
        }
        t1 = warp_sum(t1);
        t2 = warp_sum(t2);
        if (lane == 0) of_warp[warp] = make_float2(t1, t2);
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < warps; ++i) {
                t1 += of_warp[i].x;
                t2 += of_warp[i].y;
            }
            result = make_float2(__fdiv_rn(t1, count), __fdiv_rn(t2, count));
        }
        __syncthreads();
    }
    const float k1 = rstd * result.x, k2 = rstd * rstd * result.y;
    for (int i = begin + warp; i < end; i += warps) {
        const Piece<T> piece(s, plan, first_plane, i);
        float a, b;
        affine(piece.channel, a, b);
        piece.template each<U>(lane, [&](auto many, int64_t at) {
            constexpr int M = decltype(many)::value;
            uint4 rx[M], rg[M];
#pragma unroll
            for (int u = 0; u < M; ++u) {
                rx[u] = *reinterpret_cast<const uint4 *>(x + at + u * 32 * V);
                rg[u] = *reinterpret_cast<const uint4 *>(grad + at + u * 32 * V);
            }
#pragma unroll
            for (int u = 0; u < M; ++u) {
                f2_t v[V / 2], g[V / 2];
                unpack_pairs<T>(rx[u], v);
                unpack_pairs<T>(rg[u], g);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const f2_t d = sub2(v[j], both(mean)), dz = times_slope2<ACT, T>(g[j], fma2(d, both(a), both(b)));
                    v[j] = fma2(d, both(-k2), fma2(both(a), dz, both(-k1)));
                }
                *reinterpret_cast<uint4 *>(grad_input + at + u * 32 * V) = pack_pairs<T>(v);
            }
        });
        const int64_t at = piece.edge(lane);
        if (at >= 0) {
            const float d = to_float(x[at]) - mean, dz = times_slope<ACT, T>(to_float(grad[at]), fmaf(d, a, b));
            grad_input[at] = from_float<T>(fmaf(-d, k2, fmaf(a, dz, -k1)));
        }
    }
}

template <typename F>
int dispatch(const NormShape &s, F &&f)
{
    return with_type(s.io_kind, [&](auto t) { return with_activation(s.act, [&](auto act) { return f(t, act); }); });
}

template <typename... K, typename... A>
int launch(int kid, const char *name, void (*kernel)(K...), int64_t grid, int threads, int cluster, cudaStream_t stream, A... args)
{
    if (grid > INT32_MAX) return BC_ERR_BAD_SHAPE;
    const LaunchScope scope(kid, stream);
    launch_overlapped_cluster(kernel, (unsigned)grid, (unsigned)threads, 0, (unsigned)cluster, stream, args...);
    return check_launch(name);
}

}  // namespace

void plan_planes(const NormShape &s, NormPlanes *plan)
{
    const int size = io_size(s.io_kind), V = 16 / size, D = s.C / s.G;
    NormPlanes r{};
    const int64_t most = (int64_t)kPiece * V, units = (int64_t)s.N * s.G, bytes = s.P * D * size;
    r.chunk = (int)(norm_ceil(norm_ceil(s.P, norm_ceil(s.P, most)), V) * V);
    r.chunks = (int)norm_ceil(s.P, r.chunk);
    const int64_t pieces = (int64_t)D * r.chunks;
    int64_t k = norm_ceil(bytes, kPlaneSlice);
    if (units * k < kNormFill) k = norm_ceil(kNormFill, units);
    k = std::min(k, norm_ceil(bytes, (int64_t)8 << 10));
    if (k > kNormCluster && (units * kNormCluster >= 148 || bytes <= kNormCluster * kClusterSlice)) k = kNormCluster;
    k = std::max<int64_t>(1, std::min(k, pieces));
    if (k <= kNormCluster) {
        int p = 1;
        while (2 * p <= k) p *= 2;
        k = p;
    }
    k = std::max(k, norm_ceil(pieces, kMostPieces));
    r.per = (int)norm_ceil(pieces, k);
    r.k = (int)k;
    r.threads = 512;
    while (r.threads > 32 && r.threads / 32 / 2 >= r.per) r.threads /= 2;
    *plan = r;
}

size_t planes_sums_bytes(const NormShape &s, const NormPlanes &plan, bool backward)
{
    if (backward) return (size_t)s.N * plan.k * s.C * 8;
    return plan.k > kNormCluster ? (size_t)s.N * s.G * plan.k * 12 : 0;
}

int launch_norm_planes_forward(const NormShape &s, const NormPlanes &plan, const void *x, const void *weight, const void *bias, void *out,
                               float *stats, void *ws, cudaStream_t stream)
{
    return dispatch(s, [&](auto t, auto act) {
        using T = decltype(t);
        const int64_t grid = (int64_t)s.N * s.G * plan.k;
        auto go = [&](auto kernel, int cluster) {
            return launch(KID_NORM_FORWARD, "norm_planes_forward_kernel", kernel, grid, plan.threads, cluster, stream, (const T *)x,
                          (const T *)weight, (const T *)bias, (T *)out, stats, (float *)ws, s, plan);
        };
        if (plan.k <= kNormCluster) return go(norm_planes_forward_kernel<T, act(), NORM_WHOLE>, plan.k);
        if (const int e = go(norm_planes_forward_kernel<T, BC_ACT_NONE, NORM_SUMS>, 1)) return e;
        return go(norm_planes_forward_kernel<T, act(), NORM_RESULTS>, 1);
    });
}

int launch_norm_planes_backward(const NormShape &s, const NormPlanes &plan, const void *x, const void *weight, const void *bias,
                                const float *stats, const void *grad, void *grad_input, float *sums, cudaStream_t stream)
{
    return dispatch(s, [&](auto t, auto act) {
        using T = decltype(t);
        const int64_t grid = (int64_t)s.N * s.G * plan.k;
        auto go = [&](auto kernel, int cluster) {
            return launch(KID_NORM_BACKWARD, "norm_planes_backward_kernel", kernel, grid, plan.threads, cluster, stream, (const T *)x,
                          (const T *)weight, (const T *)bias, stats, (const T *)grad, (T *)grad_input, sums, s, plan);
        };
        if (plan.k <= kNormCluster && grad_input) return go(norm_planes_backward_kernel<T, act(), NORM_WHOLE>, plan.k);
        if (const int e = go(norm_planes_backward_kernel<T, act(), NORM_SUMS>, 1)) return e;
        return grad_input ? go(norm_planes_backward_kernel<T, act(), NORM_RESULTS>, 1) : (int)BC_OK;
    });
}

}  // namespace bc
