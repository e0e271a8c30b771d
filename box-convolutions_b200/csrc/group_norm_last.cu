// Group normalisation of channels-last tensors, a unit being `width` channels of a sample (bc_norm.cuh).
//
// A thread reads a vector at a fixed place among the channels and steps by whole rows of threads: the sums of its channels
// stay in its registers.  Channels that are no multiple of a vector: threads count vectors of the whole sample, and their
// number is a multiple of the vectors after which the places repeat (60 channels: 15 vectors of 8 are 2 pixels).  The
// values in front of a slice's first whole vector and behind its last are dealt with one by one.
//
// Position q of a CTA's vectors (thread q / V, value q % V) holds channel (phase + q) % width: reductions walk positions.
//
#include "bc_norm.cuh"

namespace bc {

namespace {

constexpr int kUnroll = 4;
constexpr size_t kMostShared = 200 << 10;

template <typename T>
struct Rows {
    static constexpr int V = kVec<T>;
    int64_t first;            // element of the thread's first vector
    int64_t step;             // elements between its vectors
    int count;                // vectors
    int channel;              // of the first value, in the unit
    int phase;                // of position 0
    int edges;                // single values around the vectors
    int64_t e0, e1, v0, v1;   // elements of the slice; of its whole vectors
    __device__ __forceinline__ Rows(const NormShape &s, const NormRows &r, int64_t n, int slab, int rank)
    {
        const int64_t p0 = min(s.P, (int64_t)rank * r.per), p1 = min(s.P, p0 + r.per);
        const int t = threadIdx.x;
        if (r.slabs > 1) {      // aligned vectors of a part of the channels
            const int cols = r.width / V, row = t / cols, rows = r.active / cols;
            channel = (t - row * cols) * V;
            first = (n * s.P + p0 + row) * s.C + slab * r.width + channel;
            step = (int64_t)rows * s.C;
            count = t < r.active && p0 + row < p1 ? (int)((p1 - p0 - row + rows - 1) / rows) : 0;
            phase = edges = 0;
            e0 = e1 = v0 = v1 = 0;
        } else {
            e0 = (n * s.P + p0) * s.C;
            e1 = (n * s.P + p1) * s.C;
            v0 = min((e0 + V - 1) / V * V, e1);
            v1 = max(e1 / V * V, v0);
            edges = (int)(v0 - e0 + e1 - v1);
            first = v0 + (int64_t)t * V;
            step = (int64_t)r.active * V;
            count = t < r.active && first < v1 ? (int)((v1 - first + step - 1) / step) : 0;
            phase = (int)(v0 - e0) % s.C;
            channel = (phase + t * V) % s.C;
        }
    }
    __device__ __forceinline__ int channel_of(int j, int width) const      // of the thread's value j, in the unit
    {
        int c = channel + j;
        while (c >= width) c -= width;
        return c;
    }
    // The i-th single value and its channel (one slab).
    __device__ __forceinline__ int64_t edge(int i, int C, int &c) const
    {
        const int64_t at = i < v0 - e0 ? e0 + i : v1 + (i - (v0 - e0));
        c = (int)((at - e0) % C);
        return at;
    }
    // Position of channel c in the pp-th repetition.
    __device__ __forceinline__ int position(int pp, int c, int width, int active) const
    {
        const int q = pp * width + c - phase;
        return q < 0 ? q + active * V : q;
    }
};

// f(vectors that are there, offset of each): kUnroll vectors of a thread at a time.
template <typename T, typename F>
__device__ __forceinline__ void each(const Rows<T> &r, F &&f)
{
    int64_t at = r.first;
    int i = 0;
    for (; i + kUnroll <= r.count; i += kUnroll, at += kUnroll * r.step) f(std::integral_constant<int, kUnroll>(), at);
    for (; i < r.count; ++i, at += r.step) f(std::integral_constant<int, 1>(), at);
}

// Shared memory: positions (pairs), counts of threads, groups' moments and results.
struct Layout {
    int active_v, threads, groups;
    __host__ __device__ size_t pairs() const { return 0; }
    __host__ __device__ size_t counts() const { return (size_t)active_v * 8; }
    __host__ __device__ size_t moments() const { return counts() + (size_t)threads * 4; }
    __host__ __device__ size_t results() const { return (moments() + (size_t)groups * 12 + 7) / 8 * 8; }
    __host__ __device__ size_t edges() const { return results() + (size_t)groups * 8; }
    __host__ __device__ size_t bytes() const { return edges() + 16 * 8; }
};

template <typename T, int ACT, int STEP, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_rows_forward_kernel(const T *__restrict__ x, const T *__restrict__ weight, const T *__restrict__ bias,
                                         T *__restrict__ out, float *__restrict__ stats, float *__restrict__ ws, NormShape s, NormRows plan)
{
    constexpr int V = kVec<T>;
    extern __shared__ __align__(16) char smem[];
    const int D = s.C / s.G, groups = plan.width / D, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Layout lay{plan.active * V, (int)blockDim.x, groups};
    float2 *pairs = reinterpret_cast<float2 *>(smem + lay.pairs());
    float *counts = reinterpret_cast<float *>(smem + lay.counts());
    float *moments = reinterpret_cast<float *>(smem + lay.moments());
    float2 *results = reinterpret_cast<float2 *>(smem + lay.results());
    float2 *edges = reinterpret_cast<float2 *>(smem + lay.edges());
    const int64_t unit = blockIdx.x / plan.k, n = unit / plan.slabs;
    const int rank = (int)(blockIdx.x - unit * plan.k), slab = (int)(unit - n * plan.slabs);
    const Rows<T> r(s, plan, n, slab, rank);
    grid_dependency_wait();

    if (STEP != NORM_RESULTS) {
        float mean[V] = {}, m2[V] = {}, have = 0.f;
        each(r, [&](auto many, int64_t at) {
            constexpr int M = decltype(many)::value;
            uint4 raw[M];
#pragma unroll
            for (int u = 0; u < M; ++u) raw[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
#pragma unroll
            for (int u = 0; u < M; ++u) {
                float v[V];
                unpack<T>(raw[u], v);
                have += 1.f;
                const float share = __fdividef(1.f, have);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - mean[j];
                    mean[j] = fmaf(d, share, mean[j]);
                    m2[j] = fmaf(d, v[j] - mean[j], m2[j]);
                }
            }
        });
        if (threadIdx.x < plan.active) {
#pragma unroll
            for (int j = 0; j < V; ++j) pairs[threadIdx.x * V + j] = make_float2(mean[j], m2[j]);
            counts[threadIdx.x] = have;
        }
        if (threadIdx.x < r.edges) {
            int c;
            const int64_t at = r.edge(threadIdx.x, s.C, c);
            edges[threadIdx.x] = make_float2(to_float(x[at]), (float)c);
        }
        __syncthreads();
        const int repeats = plan.active * V / plan.width;
        for (int g = warp; g < groups; g += warps) {
            Moments m{0.f, 0.f, 0.f};
            for (int i = lane; i < repeats * D; i += 32) {
                const int pp = i / D, q = r.position(pp, g * D + i - pp * D, plan.width, plan.active);
                const float2 v = pairs[q];
                m = merged(m, {counts[q / V], v.x, v.y});
            }
            m = warp_merged(m);
            for (int i = 0; i < r.edges; ++i)
                if ((int)edges[i].y / D == g) m = merged(m, {1.f, edges[i].x, 0.f});
            if (lane == 0) {
                float *to = STEP == NORM_SUMS ? ws + ((unit * plan.k + rank) * groups + g) * 3 : moments + 3 * g;
                to[0] = m.n;
                to[1] = m.mean;
                to[2] = m.m2;
            }
        }
        if (STEP == NORM_SUMS) return;
    }

    if (STEP == NORM_WHOLE) {
        if (plan.k > 1) cluster_sync();
        else __syncthreads();
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            Moments m{0.f, 0.f, 0.f};
            for (int i = 0; i < plan.k; ++i) {
                const uint32_t at = cluster_map(smem_u32(moments + 3 * g), plan.k > 1 ? i : 0);
                if (plan.k > 1) m = merged(m, {cluster_load(at), cluster_load(at + 4), cluster_load(at + 8)});
                else m = {moments[3 * g], moments[3 * g + 1], moments[3 * g + 2]};
            }
            results[g] = make_float2(m.mean, rsqrtf(__fdiv_rn(m.m2, m.n) + s.eps));
        }
        if (plan.k > 1) cluster_sync();      // (nobody leaves while its moments are read)
        else __syncthreads();
    } else {
        for (int g = warp; g < groups; g += warps) {
            Moments m{0.f, 0.f, 0.f};
            for (int i = lane; i < plan.k; i += 32) {
                const float *from = ws + ((unit * plan.k + i) * groups + g) * 3;
                m = merged(m, {__ldg(from), __ldg(from + 1), __ldg(from + 2)});
            }
            m = warp_merged(m);
            if (lane == 0) results[g] = make_float2(m.mean, rsqrtf(__fdiv_rn(m.m2, m.n) + s.eps));
        }
        __syncthreads();
    }
    if (stats && rank == 0)
        for (int g = threadIdx.x; g < groups; g += blockDim.x)
            reinterpret_cast<float2 *>(stats)[n * s.G + slab * groups + g] = results[g];

    float mean[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = r.count ? r.channel_of(j, plan.width) : 0, all = slab * plan.width + c;
        const float2 st = results[c / D];
        mean[j] = st.x;
        a[j] = weight ? st.y * to_float(weight[all]) : st.y;
        b[j] = bias ? to_float(bias[all]) : 0.f;
    }
    each(r, [&](auto many, int64_t at) {
        constexpr int M = decltype(many)::value;
        uint4 raw[M];
#pragma unroll
        for (int u = 0; u < M; ++u) raw[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
#pragma unroll
        for (int u = 0; u < M; ++u) {
            float v[V];
            unpack<T>(raw[u], v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = activate<ACT, T>(fmaf(v[j] - mean[j], a[j], b[j]));
            *reinterpret_cast<uint4 *>(out + at + u * r.step) = pack<T>(v);
        }
    });
    if (threadIdx.x < r.edges) {
        int c;
        const int64_t at = r.edge(threadIdx.x, s.C, c);
        const float2 st = results[c / D];
        const float w = weight ? st.y * to_float(weight[c]) : st.y;
        out[at] = from_float<T>(activate<ACT, T>(fmaf(to_float(x[at]) - st.x, w, bias ? to_float(bias[c]) : 0.f)));
    }
}

// Backward: with d = x - mean, a = weight rstd and z = a d + bias, dz = grad * slope(z),
//   S1 = sum dz, S2 = rstd * sum dz d,   A1 = sum_c weight S1 / L, A2 = sum_c weight S2 / L over the group,
//   grad_input = a dz - rstd A1 - d rstd^2 A2.
// `sums`: a row of C pairs (S1, S2) per (sample, rank).
// Shared memory: positions' pairs, partial sums of the channels, channels' pairs, groups' sums (twice), edges.
struct BackLayout {
    int active_v, threads, width, groups;
    __host__ __device__ size_t pairs() const { return 0; }
    __host__ __device__ size_t parts() const { return (size_t)active_v * 8; }
    __host__ __device__ size_t channels() const { return parts() + (size_t)(threads > width ? threads : width) * 8; }
    __host__ __device__ size_t sums() const { return channels() + (size_t)width * 8; }
    __host__ __device__ size_t results() const { return sums() + (size_t)groups * 8; }
    __host__ __device__ size_t edges() const { return results() + (size_t)groups * 8; }
    __host__ __device__ size_t bytes() const { return edges() + 16 * 12; }
};

template <typename T, int ACT, int STEP, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_rows_backward_kernel(const T *__restrict__ x, const T *__restrict__ weight, const T *__restrict__ bias,
                                          const float *__restrict__ stats, const T *__restrict__ grad, T *__restrict__ grad_input,
                                          float *__restrict__ sums, NormShape s, NormRows plan)
{
    constexpr int V = kVec<T>, U = 2;
    extern __shared__ __align__(16) char smem[];
    const int D = s.C / s.G, groups = plan.width / D, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const BackLayout lay{plan.active * V, (int)blockDim.x, plan.width, groups};
    float2 *pairs = reinterpret_cast<float2 *>(smem + lay.pairs()), *parts = reinterpret_cast<float2 *>(smem + lay.parts());
    float2 *channels = reinterpret_cast<float2 *>(smem + lay.channels()), *own = reinterpret_cast<float2 *>(smem + lay.sums());
    float2 *results = reinterpret_cast<float2 *>(smem + lay.results());
    float *edges = reinterpret_cast<float *>(smem + lay.edges());
    const int64_t unit = blockIdx.x / plan.k, n = unit / plan.slabs;
    const int rank = (int)(blockIdx.x - unit * plan.k), slab = (int)(unit - n * plan.slabs);
    const Rows<T> r(s, plan, n, slab, rank);
    grid_dependency_wait();

    const float2 *of_group = reinterpret_cast<const float2 *>(stats) + n * s.G + slab * groups;
    float mean[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = r.count ? r.channel_of(j, plan.width) : 0, all = slab * plan.width + c;
        const float2 st = of_group[c / D];
        mean[j] = st.x;
        a[j] = weight ? st.y * to_float(weight[all]) : st.y;
        b[j] = ACT != BC_ACT_NONE && bias ? to_float(bias[all]) : 0.f;
    }
    auto both = [&](auto &&f) {      // U vectors of x and of grad at a time
        int64_t at = r.first;
        int i = 0;
        for (; i + U <= r.count; i += U, at += U * r.step) f(std::integral_constant<int, U>(), at);
        for (; i < r.count; ++i, at += r.step) f(std::integral_constant<int, 1>(), at);
    };
    auto edge_slope = [&](int64_t at, int c, float &d) {      // dz of a single value
        const float2 st = of_group[c / D];
        const float w = weight ? st.y * to_float(weight[c]) : st.y;
        d = to_float(x[at]) - st.x;
        return to_float(grad[at]) * slope<ACT, T>(fmaf(d, w, ACT != BC_ACT_NONE && bias ? to_float(bias[c]) : 0.f));
    };

    if (STEP != NORM_RESULTS) {
        float s1[V] = {}, s2[V] = {};
        both([&](auto many, int64_t at) {
            constexpr int M = decltype(many)::value;
            uint4 rx[M], rg[M];
#pragma unroll
            for (int u = 0; u < M; ++u) {
                rx[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
                rg[u] = *reinterpret_cast<const uint4 *>(grad + at + u * r.step);
            }
#pragma unroll
            for (int u = 0; u < M; ++u) {
                float v[V], g[V];
                unpack<T>(rx[u], v);
                unpack<T>(rg[u], g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[j] - mean[j], dz = g[j] * slope<ACT, T>(fmaf(d, a[j], b[j]));
                    s1[j] += dz;
                    s2[j] = fmaf(dz, d, s2[j]);
                }
            }
        });
        if (threadIdx.x < plan.active)
#pragma unroll
            for (int j = 0; j < V; ++j) pairs[threadIdx.x * V + j] = make_float2(s1[j], s2[j]);
        if (threadIdx.x < r.edges) {
            int c;
            float d;
            const int64_t at = r.edge(threadIdx.x, s.C, c);
            const float dz = edge_slope(at, c, d);
            edges[3 * threadIdx.x] = dz;
            edges[3 * threadIdx.x + 1] = dz * d;
            edges[3 * threadIdx.x + 2] = (float)c;
        }
        __syncthreads();
        // a channel's positions: over as many threads as there are, then over those
        const int repeats = plan.active * V / plan.width, shares = max(1, (int)blockDim.x / plan.width);
        for (int i = threadIdx.x; i < shares * plan.width; i += blockDim.x) {
            const int share = i / plan.width, c = i - share * plan.width;
            float2 t = make_float2(0.f, 0.f);
            for (int pp = share; pp < repeats; pp += shares) {
                const float2 v = pairs[r.position(pp, c, plan.width, plan.active)];
                t.x += v.x;
                t.y += v.y;
            }
            parts[i] = t;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < plan.width; c += blockDim.x) {
            float2 t = make_float2(0.f, 0.f);
            for (int i = 0; i < shares; ++i) {
                t.x += parts[i * plan.width + c].x;
                t.y += parts[i * plan.width + c].y;
            }
            for (int i = 0; i < r.edges; ++i)
                if ((int)edges[3 * i + 2] == c) {
                    t.x += edges[3 * i];
                    t.y += edges[3 * i + 1];
                }
            t.y *= of_group[c / D].y;
            reinterpret_cast<float2 *>(sums)[(n * plan.k + rank) * s.C + slab * plan.width + c] = t;
            const float w = weight ? to_float(weight[slab * plan.width + c]) : 1.f;
            channels[c] = make_float2(w * t.x, w * t.y);
        }
        if (STEP == NORM_SUMS) return;
        __syncthreads();
        for (int g = warp; g < groups; g += warps) {
            float t1 = 0.f, t2 = 0.f;
            for (int d = lane; d < D; d += 32) {
                t1 += channels[g * D + d].x;
                t2 += channels[g * D + d].y;
            }
            t1 = warp_sum(t1);
            t2 = warp_sum(t2);
            if (lane == 0) own[g] = make_float2(t1, t2);
        }
        if (plan.k > 1) cluster_sync();
        else __syncthreads();
        const float count = (float)D * (float)s.P;
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            float2 t = own[g];
            if (plan.k > 1) {
                t = make_float2(0.f, 0.f);
                for (int i = 0; i < plan.k; ++i) {
                    const uint32_t at = cluster_map(smem_u32(own + g), i);
                    t.x += cluster_load(at);
                    t.y += cluster_load(at + 4);
                }
            }
            results[g] = make_float2(__fdiv_rn(t.x, count), __fdiv_rn(t.y, count));
        }
        if (plan.k > 1) cluster_sync();
        else __syncthreads();
    } else {
        // the ranks' rows, weighted: a warp a group
        const float count = (float)D * (float)s.P;
        for (int g = warp; g < groups; g += warps) {
            float t1 = 0.f, t2 = 0.f;
            for (int i = lane; i < plan.k * D; i += 32) {
                const int at = i / D, c = slab * plan.width + g * D + i - at * D;
                const float2 v = __ldg(reinterpret_cast<const float2 *>(sums) + (n * plan.k + at) * s.C + c);
                const float w = weight ? to_float(weight[c]) : 1.f;
                t1 = fmaf(w, v.x, t1);
                t2 = fmaf(w, v.y, t2);
            }
            t1 = warp_sum(t1);
            t2 = warp_sum(t2);
            if (lane == 0) results[g] = make_float2(__fdiv_rn(t1, count), __fdiv_rn(t2, count));
        }
        __syncthreads();
    }

    float k1[V], k2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int g = (r.count ? r.channel_of(j, plan.width) : 0) / D;
        const float rstd = of_group[g].y;
        k1[j] = rstd * results[g].x;
        k2[j] = rstd * rstd * results[g].y;
    }
    both([&](auto many, int64_t at) {
        constexpr int M = decltype(many)::value;
        uint4 rx[M], rg[M];
#pragma unroll
        for (int u = 0; u < M; ++u) {
            rx[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
            rg[u] = *reinterpret_cast<const uint4 *>(grad + at + u * r.step);
        }
#pragma unroll
        for (int u = 0; u < M; ++u) {
            float v[V], g[V];
            unpack<T>(rx[u], v);
            unpack<T>(rg[u], g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - mean[j], dz = g[j] * slope<ACT, T>(fmaf(d, a[j], b[j]));
                v[j] = fmaf(-d, k2[j], fmaf(a[j], dz, -k1[j]));
            }
            *reinterpret_cast<uint4 *>(grad_input + at + u * r.step) = pack<T>(v);
        }
    });
    if (threadIdx.x < r.edges) {
        int c;
        float d;
        const int64_t at = r.edge(threadIdx.x, s.C, c);
        const float dz = edge_slope(at, c, d), rstd = of_group[c / D].y;
        const float w = weight ? rstd * to_float(weight[c]) : rstd;
        grad_input[at] = from_float<T>(fmaf(-d, rstd * rstd * results[c / D].y, fmaf(w, dz, -rstd * results[c / D].x)));
    }
}

template <typename F>
int dispatch(const NormShape &s, F &&f)
{
    return with_type(s.io_kind, [&](auto t) { return with_activation(s.act, [&](auto act) { return f(t, act); }); });
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

template <typename... K, typename... A>
int launch(int kid, const char *name, void (*kernel)(K...), int64_t grid, int threads, size_t smem, int cluster, cudaStream_t stream, A... args)
{
    if (grid > INT32_MAX) return BC_ERR_BAD_SHAPE;
    if (smem > 48 << 10)
        if (const int e = raise_smem_limit((const void *)kernel, kMostShared)) return e;
    const LaunchScope scope(kid, stream);
    launch_overlapped_cluster(kernel, (unsigned)grid, (unsigned)threads, smem, (unsigned)cluster, stream, args...);
    return check_launch(name);
}

}  // namespace

// Whether these kernels serve the shape, and how: a CTA's threads repeat the channels' places in vectors.
bool plan_rows(const NormShape &s, NormRows *plan)
{
    const int size = io_size(s.io_kind), V = 16 / size, D = s.C / s.G;
    NormRows r{};
    r.width = s.C;
    r.slabs = 1;
    const int64_t sample = s.P * s.C * size;
    // Few samples: parts of the channels as units of their own, down to two sectors of 32 bytes a pixel.
    while ((s.N * r.slabs * kNormCluster < kNormFill || sample / r.slabs > kNormCluster * kNormSlice) && r.width % 2 == 0 &&
           r.width / 2 % D == 0 && r.width / 2 * size % 64 == 0) {
        r.width /= 2;
        r.slabs *= 2;
    }
    const int period = r.slabs > 1 ? r.width / V : s.C / gcd(s.C, V);      // vectors after which the places repeat
    if (period > 1024) return false;
    r.threads = period > 512 ? 1024 : 512;
    const int64_t units = (int64_t)s.N * r.slabs, bytes = sample / r.slabs;
    // slices that fill the GPU, of a vector a thread at least
    int64_t k = norm_ceil(bytes, kNormSlice);
    if (units * k < kNormFill) k = norm_ceil(kNormFill, units);
    k = std::min(k, norm_ceil(bytes, (int64_t)r.threads * 16));
    if (k > kNormCluster && (units * kNormCluster >= 148 || bytes <= kNormCluster * kNormSlice)) k = kNormCluster;
    if (k <= kNormCluster) {
        int p = 1;
        while (p < k) p *= 2;
        k = p;
    }
    // small slices: no more threads than vectors
    const int64_t vectors = norm_ceil(norm_ceil(bytes, k), 16);
    while (r.threads > 64 && r.threads / 2 >= period && r.threads / 2 >= vectors) r.threads /= 2;
    r.active = r.threads / period * period;
    r.per = (int)norm_ceil(s.P, k);
    r.k = (int)k;
    *plan = r;
    const int groups = r.width / D;
    return std::max(Layout{r.active * V, r.threads, groups}.bytes(), BackLayout{r.active * V, r.threads, r.width, groups}.bytes()) <= kMostShared;
}

size_t rows_sums_bytes(const NormShape &s, const NormRows &plan, bool backward)
{
    if (backward) return (size_t)s.N * plan.k * s.C * 8;
    return plan.k > kNormCluster ? (size_t)s.N * plan.k * s.G * 12 : 0;
}

int launch_norm_rows_forward(const NormShape &s, const NormRows &plan, const void *x, const void *weight, const void *bias, void *out,
                             float *stats, void *ws, cudaStream_t stream)
{
    return dispatch(s, [&](auto t, auto act) {
        using T = decltype(t);
        const int64_t grid = (int64_t)s.N * plan.slabs * plan.k;
        const size_t smem = Layout{plan.active * kVec<T>, plan.threads, plan.width / (s.C / s.G)}.bytes();
        auto go = [&](auto kernel, int cluster) {
            return launch(KID_NORM_FORWARD, "norm_rows_forward_kernel", kernel, grid, plan.threads, smem, cluster, stream, (const T *)x,
                          (const T *)weight, (const T *)bias, (T *)out, stats, (float *)ws, s, plan);
        };
        auto run = [&](auto most) {
            constexpr int THREADS = decltype(most)::value;
            if (plan.k <= kNormCluster) return go(norm_rows_forward_kernel<T, act(), NORM_WHOLE, THREADS>, plan.k);
            if (const int e = go(norm_rows_forward_kernel<T, BC_ACT_NONE, NORM_SUMS, THREADS>, 1)) return e;
            return go(norm_rows_forward_kernel<T, act(), NORM_RESULTS, THREADS>, 1);
        };
        return plan.threads > 512 ? run(std::integral_constant<int, 1024>()) : run(std::integral_constant<int, 512>());
    });
}

int launch_norm_rows_backward(const NormShape &s, const NormRows &plan, const void *x, const void *weight, const void *bias,
                              const float *stats, const void *grad, void *grad_input, float *sums, cudaStream_t stream)
{
    return dispatch(s, [&](auto t, auto act) {
        using T = decltype(t);
        const int64_t grid = (int64_t)s.N * plan.slabs * plan.k;
        const size_t smem = BackLayout{plan.active * kVec<T>, plan.threads, plan.width, plan.width / (s.C / s.G)}.bytes();
        auto go = [&](auto kernel, int cluster) {
            return launch(KID_NORM_BACKWARD, "norm_rows_backward_kernel", kernel, grid, plan.threads, smem, cluster, stream, (const T *)x,
                          (const T *)weight, (const T *)bias, stats, (const T *)grad, (T *)grad_input, sums, s, plan);
        };
        auto run = [&](auto most) {
            constexpr int THREADS = decltype(most)::value;
            if (plan.k <= kNormCluster && grad_input) return go(norm_rows_backward_kernel<T, act(), NORM_WHOLE, THREADS>, plan.k);
            if (const int e = go(norm_rows_backward_kernel<T, act(), NORM_SUMS, THREADS>, 1)) return e;
            return grad_input ? go(norm_rows_backward_kernel<T, act(), NORM_RESULTS, THREADS>, 1) : (int)BC_OK;
        };
        return plan.threads > 512 ? run(std::integral_constant<int, 1024>()) : run(std::integral_constant<int, 512>());
    });
}

}  // namespace bc
