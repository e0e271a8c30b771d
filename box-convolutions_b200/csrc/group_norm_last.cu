// Group normalisation of channels-last tensors, a unit being `width` channels of a sample (bc_norm.cuh).
//
// A thread reads a vector at a fixed place among the channels and steps by whole rows of threads: the sums of its channels
// stay in its registers.  Channels that are no multiple of a vector: threads count vectors of the whole sample, and their
// number is a multiple of the vectors after which the places repeat (60 channels: 15 vectors of 8 are 2 pixels).  The
// values in front of a slice's first whole vector and behind its last are dealt with one by one.
//
// Measured on B200, (16,128,64,128) bf16 with SiLU: forward 30 us, backward 43 (the bytes at the copy bandwidth: 10 and 15).  256 CTAs of
// 256 threads are fewer than two an SM: what a reading waits for has little beside it, nor has the exchange of the clusters.
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
            const unsigned cols = r.width / V, row = (unsigned)t / cols, rows = (unsigned)r.active / cols;
            channel = (t - row * cols) * V;
            first = (n * s.P + p0 + row) * s.C + slab * r.width + channel;
            step = (int64_t)rows * s.C;
            count = t < r.active && p0 + row < p1 ? (int)(((unsigned)(p1 - p0) - row + rows - 1) / rows) : 0;
            phase = edges = 0;
            e0 = e1 = v0 = v1 = 0;
        } else {
            e0 = (n * s.P + p0) * s.C;
            e1 = (n * s.P + p1) * s.C;
            v0 = min((e0 + V - 1) & ~(int64_t)(V - 1), e1);
            v1 = max(e1 & ~(int64_t)(V - 1), v0);
            edges = (int)(v0 - e0 + e1 - v1);
            first = v0 + (int64_t)t * V;
            step = (int64_t)r.active * V;
            count = 0;
            if (t < r.active && first < v1) {
                const int64_t more = v1 - first + step - 1;
                count = more >> 32 ? (int)(more / step) : (int)((unsigned)more / (unsigned)step);
            }
            phase = (int)(v0 - e0) % s.C;
            channel = (phase + t * V) % s.C;
        }
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

// Channels' factors in shared memory, made once a CTA: rows of `width` floats.
struct Affine {
    float *base;
    int width;
    __device__ __forceinline__ void put(int c, int row, float v) const { base[row * width + c] = v; }
    __device__ __forceinline__ float at(int c, int row) const { return base[row * width + c]; }
    // Those of a thread's vector.
    template <int V, typename R>
    __device__ __forceinline__ void get(int row, const R &r, f2_t (&v)[V / 2]) const
    {
        int c = r.channel;
        const float *from = base + row * width;
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const float a = from[c];
            c = c + 1 < width ? c + 1 : 0;
            const float b = from[c];
            c = c + 1 < width ? c + 1 : 0;
            v[j] = pack2(a, b);
        }
    }
};

// Shared memory: positions (pairs), counts of threads, groups' moments and results.
struct Layout {
    int active_v, threads, width, groups;
    __host__ __device__ size_t pairs() const { return 0; }
    __host__ __device__ size_t counts() const { return (size_t)(active_v > 2 * width ? active_v : 2 * width) * 8; }      // (or three rows of channels)
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
    const Layout lay{plan.active * V, (int)blockDim.x, plan.width, groups};
    float2 *pairs = reinterpret_cast<float2 *>(smem + lay.pairs());
    float *counts = reinterpret_cast<float *>(smem + lay.counts());
    float *moments = reinterpret_cast<float *>(smem + lay.moments());
    float2 *results = reinterpret_cast<float2 *>(smem + lay.results());
    float2 *edges = reinterpret_cast<float2 *>(smem + lay.edges());
    const unsigned index = blockIdx.x / (unsigned)plan.k, sample = index / (unsigned)plan.slabs;
    const int64_t unit = index, n = sample;
    const int rank = (int)(blockIdx.x - index * plan.k), slab = (int)(index - sample * plan.slabs);
    const Rows<T> r(s, plan, n, slab, rank);
    grid_dependency_wait();

    if (STEP != NORM_RESULTS) {
        f2_t mean[V / 2], m2[V / 2];
        float have = 0.f;
#pragma unroll
        for (int j = 0; j < V / 2; ++j) mean[j] = m2[j] = both(0.f);
        each(r, [&](auto many, int64_t at) {
            constexpr int M = decltype(many)::value;
            uint4 raw[M];
#pragma unroll
            for (int u = 0; u < M; ++u) raw[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
#pragma unroll
            for (int u = 0; u < M; ++u) {
                f2_t v[V / 2];
                unpack_pairs<T>(raw[u], v);
                have += 1.f;
                const f2_t share = both(reciprocal(have));
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const f2_t d = sub2(v[j], mean[j]);
                    mean[j] = fma2(d, share, mean[j]);
                    m2[j] = fma2(d, sub2(v[j], mean[j]), m2[j]);
                }
            }
        });
        // Neighbours of a group become one in the thread, where vectors and groups end together: their counts are equal.
        const int run = s.C % V == 0 && (D % V == 0 || V % D == 0) ? min(D, V) : 1;
        if (threadIdx.x < plan.active) {
            float mj[V], qj[V];      // means and variances
            const f2_t share = both(have > 0.f ? __frcp_rn(have) : 0.f);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                unpack2(mean[j / 2], mj[j], mj[j + 1]);
                unpack2(mul2(m2[j / 2], share), qj[j], qj[j + 1]);
            }
#pragma unroll
            for (int w = 1; w < V; w *= 2)
                if (run > w)
#pragma unroll
                    for (int j = 0; j < V; j += 2 * w) {
                        const float d = mj[j + w] - mj[j];
                        mj[j] = fmaf(0.5f, d, mj[j]);
                        qj[j] = fmaf(0.25f * d, d, 0.5f * (qj[j] + qj[j + w]));
                    }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j % run == 0) pairs[(threadIdx.x * V + j) / (unsigned)run] = make_float2(mj[j], qj[j]);
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
            const int each = D / run;
            for (int i = lane; i < repeats * each; i += 32) {
                const int pp = (unsigned)i / (unsigned)each;
                const int q = r.position(pp, g * D + (i - pp * each) * run, plan.width, plan.active);
                const float2 v = pairs[(unsigned)q / (unsigned)run];
                m = merged(m, {counts[q / V] * run, v.x, v.y});
            }
            m = warp_merged(m);
            for (int i = 0; i < r.edges; ++i)
                if ((int)edges[i].y / D == g) m = merged(m, {1.f, edges[i].x, 0.f});
            if (lane == 0) {
                float *to = STEP == NORM_SUMS ? ws + ((unit * plan.k + rank) * groups + g) * 3 : moments + 3 * g;
                to[0] = m.n;
                to[1] = m.mean;
                to[2] = m.var;
            }
        }
        if (STEP == NORM_SUMS) return;
    }

    if (STEP == NORM_WHOLE) {
        if (plan.k > 1) cluster_sync();
        else __syncthreads();
        // a lane a CTA, k lanes a group
        for (int i0 = 0; i0 < groups * plan.k; i0 += blockDim.x) {
            const int i = i0 + threadIdx.x, g = (unsigned)i / (unsigned)plan.k;
            Moments m{0.f, 0.f, 0.f};
            if (g < groups) {
                const uint32_t at = plan.k > 1 ? cluster_map(smem_u32(moments + 3 * g), i - g * plan.k) : smem_u32(moments + 3 * g);
                m = {cluster_load(at), cluster_load(at + 4), cluster_load(at + 8)};
            }
            for (int o = 1; o < plan.k; o *= 2)
                m = merged(m, {__shfl_down_sync(0xffffffffu, m.n, o), __shfl_down_sync(0xffffffffu, m.mean, o),
                               __shfl_down_sync(0xffffffffu, m.var, o)});
            if (g < groups && i == g * plan.k) results[g] = make_float2(m.mean, rsqrtf(m.var + s.eps));
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
            if (lane == 0) results[g] = make_float2(m.mean, rsqrtf(m.var + s.eps));
        }
        __syncthreads();
    }
    if (stats && rank == 0)
        for (int g = threadIdx.x; g < groups; g += blockDim.x)
            reinterpret_cast<float2 *>(stats)[n * s.G + slab * groups + g] = results[g];

    const Affine table{reinterpret_cast<float *>(smem + lay.pairs()), plan.width};      // (the positions have been read)
    __syncthreads();
    for (int c = threadIdx.x; c < plan.width; c += blockDim.x) {
        const float2 st = results[(unsigned)c / (unsigned)D];
        table.put(c, 0, st.x);
        table.put(c, 1, weight ? st.y * to_float(weight[slab * plan.width + c]) : st.y);
        table.put(c, 2, bias ? to_float(bias[slab * plan.width + c]) : 0.f);
    }
    __syncthreads();
    f2_t mean[V / 2], a[V / 2], b[V / 2];
    table.get<V>(0, r, mean);
    table.get<V>(1, r, a);
    table.get<V>(2, r, b);
    each(r, [&](auto many, int64_t at) {
        constexpr int M = decltype(many)::value;
        uint4 raw[M];
#pragma unroll
        for (int u = 0; u < M; ++u) raw[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
#pragma unroll
        for (int u = 0; u < M; ++u) {
            f2_t v[V / 2];
            unpack_pairs<T>(raw[u], v);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) v[j] = activate2<ACT, T>(fma2(sub2(v[j], mean[j]), a[j], b[j]));
            *reinterpret_cast<uint4 *>(out + at + u * r.step) = pack_pairs<T>(v);
        }
    });
    if (threadIdx.x < r.edges) {
        int c;
        const int64_t at = r.edge(threadIdx.x, s.C, c);
        out[at] = from_float<T>(activate<ACT, T>(fmaf(to_float(x[at]) - table.at(c, 0), table.at(c, 1), table.at(c, 2))));
    }
}

// Backward: with d = x - mean, a = weight rstd and z = a d + bias, dz = grad * slope(z),
//   S1 = sum dz, S2 = rstd * sum dz d,   A1 = sum_c weight S1 / L, A2 = sum_c weight S2 / L over the group,
//   grad_input = a dz - rstd A1 - d rstd^2 A2.
// `sums`: a row of C pairs (S1, S2) per (sample, rank).
// Shared memory: positions' pairs, partial sums of the channels, channels' pairs, groups' sums (twice), edges, channels' factors.
struct BackLayout {
    int active_v, threads, width, groups;
    __host__ __device__ size_t pairs() const { return 0; }
    __host__ __device__ size_t parts() const { return (size_t)active_v * 8; }
    __host__ __device__ size_t channels() const { return parts() + (size_t)(threads > width ? threads : width) * 8; }
    __host__ __device__ size_t sums() const { return channels() + (size_t)width * 8; }
    __host__ __device__ size_t results() const { return sums() + (size_t)groups * 8; }
    __host__ __device__ size_t edges() const { return results() + (size_t)groups * 8; }
    __host__ __device__ size_t affine() const { return edges() + 16 * 12; }
    __host__ __device__ size_t bytes() const { return affine() + (size_t)width * 20; }
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
    const unsigned index = blockIdx.x / (unsigned)plan.k, sample = index / (unsigned)plan.slabs;
    const int64_t n = sample;
    const int rank = (int)(blockIdx.x - index * plan.k), slab = (int)(index - sample * plan.slabs);
    const Rows<T> r(s, plan, n, slab, rank);
    grid_dependency_wait();

    const float2 *of_group = reinterpret_cast<const float2 *>(stats) + n * s.G + slab * groups;
    const Affine table{reinterpret_cast<float *>(smem + lay.affine()), plan.width};
    for (int c = threadIdx.x; c < plan.width; c += blockDim.x) {
        const float2 st = of_group[(unsigned)c / (unsigned)D];
        table.put(c, 0, st.x);
        table.put(c, 1, weight ? st.y * to_float(weight[slab * plan.width + c]) : st.y);
        table.put(c, 2, ACT != BC_ACT_NONE && bias ? to_float(bias[slab * plan.width + c]) : 0.f);
    }
    __syncthreads();
    f2_t mean[V / 2], a[V / 2], b[V / 2];
    table.get<V>(0, r, mean);
    table.get<V>(1, r, a);
    table.get<V>(2, r, b);
    auto each_both = [&](auto &&f) {      // U vectors of x and of grad at a time
        int64_t at = r.first;
        int i = 0;
        for (; i + U <= r.count; i += U, at += U * r.step) f(std::integral_constant<int, U>(), at);
        for (; i < r.count; ++i, at += r.step) f(std::integral_constant<int, 1>(), at);
    };
    auto edge_slope = [&](int64_t at, int c, float &d) {      // dz of a single value
        d = to_float(x[at]) - table.at(c, 0);
        return times_slope<ACT, T>(to_float(grad[at]), fmaf(d, table.at(c, 1), table.at(c, 2)));
    };

    if (STEP != NORM_RESULTS) {
        f2_t s1[V / 2], s2[V / 2];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) s1[j] = s2[j] = both(0.f);
        each_both([&](auto many, int64_t at) {
            constexpr int M = decltype(many)::value;
            uint4 rx[M], rg[M];
#pragma unroll
            for (int u = 0; u < M; ++u) {
                rx[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
                rg[u] = *reinterpret_cast<const uint4 *>(grad + at + u * r.step);
            }
#pragma unroll
            for (int u = 0; u < M; ++u) {
                f2_t v[V / 2], g[V / 2];
                unpack_pairs<T>(rx[u], v);
                unpack_pairs<T>(rg[u], g);
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const f2_t d = sub2(v[j], mean[j]), dz = times_slope2<ACT, T>(g[j], fma2(d, a[j], b[j]));
                    s1[j] = add2(s1[j], dz);
                    s2[j] = fma2(dz, d, s2[j]);
                }
            }
        });
        if (threadIdx.x < plan.active)
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                float p, q, u, v;
                unpack2(s1[j / 2], p, q);
                unpack2(s2[j / 2], u, v);
                *reinterpret_cast<float4 *>(pairs + threadIdx.x * V + j) = make_float4(p, u, q, v);
            }
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
        for (int i0 = 0; i0 < groups * plan.k; i0 += blockDim.x) {      // a lane a CTA, k lanes a group
            const int i = i0 + threadIdx.x, g = (unsigned)i / (unsigned)plan.k;
            float2 t = make_float2(0.f, 0.f);
            if (g < groups) {
                const uint32_t at = plan.k > 1 ? cluster_map(smem_u32(own + g), i - g * plan.k) : smem_u32(own + g);
                t = make_float2(cluster_load(at), cluster_load(at + 4));
            }
            for (int o = 1; o < plan.k; o *= 2) {
                t.x += __shfl_down_sync(0xffffffffu, t.x, o);
                t.y += __shfl_down_sync(0xffffffffu, t.y, o);
            }
            if (g < groups && i == g * plan.k) results[g] = make_float2(__fdiv_rn(t.x, count), __fdiv_rn(t.y, count));
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

    for (int c = threadIdx.x; c < plan.width; c += blockDim.x) {
        const int g = (unsigned)c / (unsigned)D;
        const float rstd = of_group[g].y;
        table.put(c, 3, -rstd * results[g].x);
        table.put(c, 4, -rstd * rstd * results[g].y);
    }
    __syncthreads();
    f2_t k1[V / 2], k2[V / 2];
    table.get<V>(3, r, k1);
    table.get<V>(4, r, k2);
    each_both([&](auto many, int64_t at) {
        constexpr int M = decltype(many)::value;
        uint4 rx[M], rg[M];
#pragma unroll
        for (int u = 0; u < M; ++u) {
            rx[u] = *reinterpret_cast<const uint4 *>(x + at + u * r.step);
            rg[u] = *reinterpret_cast<const uint4 *>(grad + at + u * r.step);
        }
#pragma unroll
        for (int u = 0; u < M; ++u) {
            f2_t v[V / 2], g[V / 2];
            unpack_pairs<T>(rx[u], v);
            unpack_pairs<T>(rg[u], g);
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const f2_t d = sub2(v[j], mean[j]), dz = times_slope2<ACT, T>(g[j], fma2(d, a[j], b[j]));
                v[j] = fma2(d, k2[j], fma2(a[j], dz, k1[j]));
            }
            *reinterpret_cast<uint4 *>(grad_input + at + u * r.step) = pack_pairs<T>(v);
        }
    });
    if (threadIdx.x < r.edges) {
        int c;
        float d;
        const int64_t at = r.edge(threadIdx.x, s.C, c);
        const float dz = edge_slope(at, c, d);
        grad_input[at] = from_float<T>(fmaf(d, table.at(c, 4), fmaf(table.at(c, 1), dz, table.at(c, 3))));
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
    // Parts of the channels as units of their own: down to 64 bytes a pixel where the GPU would not fill ((1,64,256,512) f32 forward
    // 17 us, 19 at 128 bytes), to 128 where slices would be long.  us forward + backward of that against no parts there, and
    // against 64 bytes there too: (16,128,64,128) bf16 35 + 48, 35 + 48, 41 + 54; f32 43 + 99, 58 + 101, 43 + 101; (24,256,64,128) bf16
    // 78 + 146, 132 + 177, 82 + 154; (64,64,64,128) bf16 68 + 103, 68 + 101, 62 + 105; (24,64,128,128) f32 56 + 199, 72 + 203, 66 + 170.
    while (r.width % 2 == 0 && r.width / 2 % D == 0 && r.width / 2 * size % 64 == 0 &&
           (s.N * r.slabs * kNormCluster < 148 || (sample / r.slabs > kNormCluster * kNormSlice && r.width / 2 * size % 128 == 0))) {
        r.width /= 2;
        r.slabs *= 2;
    }
    const int period = r.slabs > 1 ? r.width / V : s.C / gcd(s.C, V);      // vectors after which the places repeat
    if (period > 1024) return false;
    r.threads = period > 512 ? 1024 : period > 256 ? 512 : 256;
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
    return std::max(Layout{r.active * V, r.threads, r.width, groups}.bytes(), BackLayout{r.active * V, r.threads, r.width, groups}.bytes()) <= kMostShared;
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
        const size_t smem = Layout{plan.active * kVec<T>, plan.threads, plan.width, plan.width / (s.C / s.G)}.bytes();
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
