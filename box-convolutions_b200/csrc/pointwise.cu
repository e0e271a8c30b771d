// Pointwise convolution, out = act(W x + bias + residual) per pixel, and its gradients, with float multiply-adds:
// every size, layout, alignment and type.
//
// Three products, all of the form  D[m, n] = sum_k A[m, k] B[n, k]  with pixels and channels in turn:
//   forward      D[p, o] = sum_i x[i, p] W[o, i]           act(D + bias + residual) is stored
//   slope        the same product; grad * act'(D + bias + residual) = dz is stored
//   grad_input   D[p, i] = sum_o dz[o, p] W[o, i]
//   grad_weight  D[o, i] = sum_p dz[o, p] x[i, p]          split over the pixels; partial sums added in order
// A CTA makes a tile of D from slices of 16 k that pass through shared memory as floats; a thread keeps 8 x 8 (8 x 4)
// sums in registers, so that 16 (12) words read from shared memory feed 64 (32) multiply-adds.
#include "bc_layers.cuh"

namespace bc {

namespace {

enum { FORWARD, SLOPE, INPUT };
constexpr int kThreads = 128, kBM = 128, kBK = 16;

struct Product {
    const void *a, *w, *bias, *residual, *grad;
    void *out;
    int K, Cn;               // channels of A and of the output
    int wn, wk;              // strides of W along them
    int64_t P;               // pixels of a sample (of all of them together, channels last)
    int tiles_p, tiles_n;    // tiles of a sample's pixels, and of the output's channels
};

// D's tile: kBM pixels of a sample x BN channels.
template <typename T, int MODE, int ACT, bool LAST, int BN>
__global__ void __launch_bounds__(kThreads) pointwise_kernel(Product q)
{
    constexpr int TN = BN / 8;      // channels of a thread
    __shared__ __align__(16) float As[2][kBK][kBM + 4], Bs[2][kBK][BN + 4];
    const int tid = threadIdx.x, tm = tid & 15, tn = tid >> 4;
    const int64_t tile = blockIdx.x / q.tiles_n;
    const int n0 = (int)(blockIdx.x - tile * q.tiles_n) * BN;
    const int64_t sample = tile / q.tiles_p, p0 = (tile - sample * q.tiles_p) * kBM;
    const int pixels = (int)min((int64_t)kBM, q.P - p0);
    const T *a = static_cast<const T *>(q.a) + sample * q.K * q.P + (LAST ? p0 * q.K : p0);
    const T *w = static_cast<const T *>(q.w);
    grid_dependency_wait();

    float ra[kBM * kBK / kThreads], rb[BN * kBK / kThreads];
    auto load = [&](int k0) {
#pragma unroll
        for (int j = 0; j < kBM * kBK / kThreads; ++j) {
            const int k = k0 + (LAST ? tid & 15 : j), m = LAST ? (tid >> 4) + 8 * j : tid;
            ra[j] = k < q.K && m < pixels ? to_float(a[LAST ? (int64_t)m * q.K + k : k * q.P + m]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < BN * kBK / kThreads; ++j) {
            const int e = tid + kThreads * j;
            const int k = k0 + (MODE == INPUT ? e / BN : e % kBK), n = n0 + (MODE == INPUT ? e % BN : e / kBK);
            rb[j] = k < q.K && n < q.Cn ? to_float(w[(int64_t)n * q.wn + (int64_t)k * q.wk]) : 0.f;
        }
    };
    auto store = [&](int b) {
#pragma unroll
        for (int j = 0; j < kBM * kBK / kThreads; ++j) As[b][LAST ? tid & 15 : j][LAST ? (tid >> 4) + 8 * j : tid] = ra[j];
#pragma unroll
        for (int j = 0; j < BN * kBK / kThreads; ++j) {
            const int e = tid + kThreads * j;
            Bs[b][MODE == INPUT ? e / BN : e % kBK][MODE == INPUT ? e % BN : e / kBK] = rb[j];
        }
    };

    float acc[8][TN] = {};
    if (q.K) {
        load(0);
        store(0);
    }
    __syncthreads();
    for (int k0 = 0, b = 0; k0 < q.K; k0 += kBK, b ^= 1) {
        const bool more = k0 + kBK < q.K;
        if (more) load(k0 + kBK);
#pragma unroll
        for (int k = 0; k < kBK; ++k) {
            float av[8], bv[TN];
            *reinterpret_cast<float4 *>(av) = *reinterpret_cast<const float4 *>(&As[b][k][4 * tm]);
            *reinterpret_cast<float4 *>(av + 4) = *reinterpret_cast<const float4 *>(&As[b][k][64 + 4 * tm]);
#pragma unroll
            for (int j = 0; j < TN; j += 4) *reinterpret_cast<float4 *>(bv + j) = *reinterpret_cast<const float4 *>(&Bs[b][k][8 * j + 4 * tn]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
        if (more) store(b ^ 1);
        __syncthreads();
    }

    // pixel 64 * (i / 4) + 4 * tm + i % 4, channel 32 * (j / 4) + 4 * tn + j % 4 of the tile
    const int64_t base = sample * q.Cn * q.P + (LAST ? p0 * q.Cn : p0);
    const T *bias = static_cast<const T *>(q.bias), *residual = static_cast<const T *>(q.residual), *grad = static_cast<const T *>(q.grad);
    T *out = static_cast<T *>(q.out);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = n0 + 32 * (j / 4) + 4 * tn + j % 4;
        if (n >= q.Cn) continue;
        const float b = MODE != INPUT && bias ? to_float(bias[n]) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int m = 64 * (i / 4) + 4 * tm + i % 4;
            if (m >= pixels) continue;
            const int64_t at = base + (LAST ? (int64_t)m * q.Cn + n : n * q.P + m);
            float z = acc[i][j] + b;
            if (MODE != INPUT && residual) z += to_float(residual[at]);
            out[at] = from_float<T>(MODE == FORWARD ? activate<ACT, T>(z) : MODE == SLOPE ? times_slope<ACT, T>(to_float(grad[at]), z) : z);
        }
    }
}

struct WeightProduct {
    const void *dz, *x;
    float *partial;          // a row a split: Co * Ci sums, then Co sums of dz
    int N, Ci, Co;           // (N 1, channels last)
    int64_t P;
    int tiles_o, tiles_i;
    int chunk, chunks;       // a piece is `chunk` pixels of a sample, which has `chunks` of them
    int per;                 // pieces of a split
    bool sums;               // the sums of dz too
};

constexpr int kBO = 64, kBI = 64;

// D's tile: kBO x kBI weights, summed over a split's pixels.
template <typename T, bool LAST>
__global__ void __launch_bounds__(kThreads) pointwise_weight_kernel(WeightProduct q)
{
    __shared__ __align__(16) float As[2][kBK][kBO + 4], Bs[2][kBK][kBI + 4];
    const int tid = threadIdx.x, tm = tid & 7, tn = tid >> 3;      // 8 x 16 threads, 8 x 4 sums each
    const int tiles = q.tiles_o * q.tiles_i, split = blockIdx.x / tiles, t = blockIdx.x - split * tiles;
    const int o0 = t / q.tiles_i * kBO, i0 = t % q.tiles_i * kBI;
    const T *dz = static_cast<const T *>(q.dz), *x = static_cast<const T *>(q.x);
    grid_dependency_wait();
    float acc[8][4] = {}, sum = 0.f;
    const int64_t pieces = (int64_t)q.N * q.chunks, first = (int64_t)split * q.per, last = min(pieces, first + q.per);
    for (int64_t piece = first; piece < last; ++piece) {
        const int64_t sample = piece / q.chunks, p0 = (piece - sample * q.chunks) * q.chunk;
        const int pixels = (int)min((int64_t)q.chunk, q.P - p0);
        const T *a = dz + (sample * q.Co * q.P + (LAST ? p0 * q.Co : p0)), *b = x + (sample * q.Ci * q.P + (LAST ? p0 * q.Ci : p0));
        float ra[8], rb[8];
        auto load = [&](int k0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {      // LAST: channels run along the threads, pixels otherwise
                const int k = k0 + (LAST ? (tid >> 6) + 2 * j : tid & 15), c = LAST ? tid & 63 : (tid >> 4) + 8 * j;
                ra[j] = k < pixels && o0 + c < q.Co ? to_float(a[LAST ? (int64_t)k * q.Co + o0 + c : (o0 + c) * q.P + k]) : 0.f;
                rb[j] = k < pixels && i0 + c < q.Ci ? to_float(b[LAST ? (int64_t)k * q.Ci + i0 + c : (i0 + c) * q.P + k]) : 0.f;
            }
        };
        auto store = [&](int s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = LAST ? (tid >> 6) + 2 * j : tid & 15, c = LAST ? tid & 63 : (tid >> 4) + 8 * j;
                As[s][k][c] = ra[j];
                Bs[s][k][c] = rb[j];
            }
        };
        load(0);
        store(0);
        __syncthreads();
        for (int k0 = 0, s = 0; k0 < pixels; k0 += kBK, s ^= 1) {
            const bool more = k0 + kBK < pixels;
            if (more) load(k0 + kBK);
#pragma unroll
            for (int k = 0; k < kBK; ++k) {
                float av[8], bv[4];
                *reinterpret_cast<float4 *>(av) = *reinterpret_cast<const float4 *>(&As[s][k][4 * tm]);
                *reinterpret_cast<float4 *>(av + 4) = *reinterpret_cast<const float4 *>(&As[s][k][32 + 4 * tm]);
                *reinterpret_cast<float4 *>(bv) = *reinterpret_cast<const float4 *>(&Bs[s][k][4 * tn]);
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
            }
            if (q.sums && i0 == 0 && tid < kBO) {
#pragma unroll
                for (int k = 0; k < kBK; ++k) sum += As[s][k][tid];
            }
            if (more) store(s ^ 1);
            __syncthreads();
        }
    }
    float *partial = q.partial + split * pointwise_partial_stride(q.Co, q.Ci);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int o = o0 + 32 * (i / 4) + 4 * tm + i % 4;
        if (o >= q.Co) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + 4 * tn + j < q.Ci) partial[(int64_t)o * q.Ci + i0 + 4 * tn + j] = acc[i][j];
    }
    if (q.sums && i0 == 0 && tid < kBO && o0 + tid < q.Co) partial[(int64_t)q.Co * q.Ci + o0 + tid] = sum;
}

// Rows of partial sums, added in a fixed order, rounded once: `count` columns, `stride` floats from row to row.
struct Partials {
    const float *from;
    int64_t stride, count;
    int rows;
    void *to;
};
constexpr int kFinishRows = 8;
// A lane a column; eight rows at a time, then those eight.
template <typename T>
__global__ void __launch_bounds__(32 * kFinishRows) pointwise_finish_kernel(Partials weights, Partials sums, unsigned blocks)
{
    __shared__ float part[kFinishRows][32];
    const Partials &q = blockIdx.x < blocks ? weights : sums;
    const int64_t e = (int64_t)(blockIdx.x < blocks ? blockIdx.x : blockIdx.x - blocks) * 32 + threadIdx.x;
    grid_dependency_wait();
    float v = 0.f;
    if (e < q.count) {
#pragma unroll 8
        for (int i = threadIdx.y; i < q.rows; i += kFinishRows) v += q.from[i * q.stride + e];
    }
    part[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y || e >= q.count) return;
    for (int i = 1; i < kFinishRows; ++i) v += part[i][threadIdx.x];
    static_cast<T *>(q.to)[e] = from_float<T>(v);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align_up(size_t v) { return (v + 255) / 256 * 256; }

template <int MODE>
int launch_product(const PointwiseShape &s, Product q, cudaStream_t stream)
{
    const int samples = s.last ? 1 : s.N;
    q.P = s.last ? s.N * s.P : s.P;
    const int bn = q.Cn <= 32 ? 32 : 64;
    const int64_t tiles_p = ceil_div(q.P, kBM);
    q.tiles_n = (int)ceil_div(q.Cn, bn);
    if (tiles_p > INT32_MAX || (double)samples * tiles_p * q.tiles_n > INT32_MAX) return BC_ERR_BAD_SHAPE;
    q.tiles_p = (int)tiles_p;
    const unsigned grid = (unsigned)(samples * tiles_p * q.tiles_n);
    return with_type(s.io_kind, [&](auto t) {
        return with_activation(MODE == INPUT ? BC_ACT_NONE : s.act, [&](auto act) {
            using T = decltype(t);
            constexpr int ACT = MODE == INPUT ? BC_ACT_NONE : act();
            const LaunchScope scope(KID_POINTWISE, stream);
            if (s.last) bn == 32 ? launch_overlapped(pointwise_kernel<T, MODE, ACT, true, 32>, grid, kThreads, 0, stream, q)
                                 : launch_overlapped(pointwise_kernel<T, MODE, ACT, true, 64>, grid, kThreads, 0, stream, q);
            else bn == 32 ? launch_overlapped(pointwise_kernel<T, MODE, ACT, false, 32>, grid, kThreads, 0, stream, q)
                          : launch_overlapped(pointwise_kernel<T, MODE, ACT, false, 64>, grid, kThreads, 0, stream, q);
            return check_launch("pointwise_kernel");
        });
    });
}

// How the pixels of grad_weight are split: pieces of whole slices of k, about two CTAs an SM, at least 256 pixels each.
struct Splits {
    int chunk, chunks, per, splits;
};
Splits splits_of(const PointwiseShape &s)
{
    const int64_t P = s.last ? s.N * s.P : s.P, samples = s.last ? 1 : s.N;
    Splits v;
    v.chunk = (int)(P < 256 ? P : 256);
    v.chunks = (int)ceil_div(P, v.chunk);
    const int64_t pieces = samples * v.chunks, tiles = ceil_div(s.Co, kBO) * ceil_div(s.Ci ? s.Ci : 1, kBI);
    const int64_t wanted = tiles > 296 ? 1 : 296 / tiles;
    v.per = (int)ceil_div(pieces, wanted);
    v.splits = (int)ceil_div(pieces, v.per);
    return v;
}

size_t partial_bytes(const PointwiseShape &s)
{
    // (either kernel's: the query does not know the arrays)
    return align_up((size_t)std::max(splits_of(s).splits, pointwise_mma_weight_splits(s)) * pointwise_partial_stride(s.Co, s.Ci) * sizeof(float));
}
size_t sums_bytes(const PointwiseShape &s) { return align_up((size_t)pointwise_mma_sums_rows(s) * s.Co * sizeof(float)); }
// dz in memory, where it is neither grad_output itself nor asked for.
bool own_dz(const PointwiseShape &s, int need_mask) { return s.act != BC_ACT_NONE && !(need_mask & BC_NEED_PW_RESIDUAL); }

}  // namespace

int launch_pointwise_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual, void *out,
                             cudaStream_t stream)
{
    if (pointwise_mma_suits(s, false) && pointwise_mma_aligned(x, weight, residual, out))
        return launch_pointwise_mma_forward(s, x, weight, bias, residual, out, stream);
    return launch_product<FORWARD>(s, {x, weight, bias, residual, nullptr, out, s.Ci, s.Co, s.Ci, 1}, stream);
}

size_t pointwise_workspace(const PointwiseShape &s, int need_mask)
{
    size_t bytes = own_dz(s, need_mask) ? align_up((size_t)io_size(s.io_kind) * s.N * s.Co * s.P) : 0;
    if (need_mask & (BC_NEED_PW_WEIGHT | BC_NEED_PW_BIAS)) bytes += partial_bytes(s);
    if ((need_mask & BC_NEED_PW_BIAS) && s.act != BC_ACT_NONE && pointwise_mma_suits(s, false)) bytes += sums_bytes(s);
    return bytes;
}

int launch_pointwise_backward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                              const void *grad, int need_mask, void *grad_input, void *grad_weight, void *grad_bias,
                              void *grad_residual, void *ws, cudaStream_t stream)
{
    char *free_ws = static_cast<char *>(ws);
    auto take = [&](size_t bytes) {
        void *p = free_ws;
        free_ws += bytes;
        return p;
    };
    const bool want_weight = need_mask & BC_NEED_PW_WEIGHT, want_bias = need_mask & BC_NEED_PW_BIAS;
    const void *dz = grad;
    float *sums = nullptr;      // of dz as it was before its rounding
    if (s.act != BC_ACT_NONE) {
        void *to = own_dz(s, need_mask) ? take(align_up((size_t)io_size(s.io_kind) * s.N * s.Co * s.P)) : grad_residual;
        int e;
        if (pointwise_mma_suits(s, false) && pointwise_mma_aligned(x, weight, residual, grad, to)) {
            if (want_bias) sums = static_cast<float *>(take(sums_bytes(s)));
            e = launch_pointwise_mma_slope(s, x, weight, bias, residual, grad, to, sums, stream);
        } else {
            e = launch_product<SLOPE>(s, {x, weight, bias, residual, grad, to, s.Ci, s.Co, s.Ci, 1}, stream);
        }
        if (e) return e;
        dz = to;
    }
    if (need_mask & BC_NEED_PW_INPUT) {
        const int e = pointwise_mma_suits(s, true) && pointwise_mma_aligned(dz, weight, grad_input)
                          ? launch_pointwise_mma_input(s, dz, weight, grad_input, stream)
                          : launch_product<INPUT>(s, {dz, weight, nullptr, nullptr, nullptr, grad_input, s.Co, s.Ci, 1, s.Ci}, stream);
        if (e) return e;
    }
    if (!want_weight && !want_bias) return BC_OK;
    const int64_t weights = (int64_t)s.Co * s.Ci;
    Partials of_weights{}, of_sums{};
    if (sums) of_sums = {sums, s.Co, s.Co, pointwise_mma_sums_rows(s), grad_bias};
    if (want_weight || !sums) {
        float *partial = static_cast<float *>(take(partial_bytes(s)));
        int splits = pointwise_mma_weight_splits(s), e;
        if (splits && pointwise_mma_aligned(dz, x)) {
            e = launch_pointwise_mma_weight(s, dz, x, partial, want_bias && !sums, stream);
        } else {
            const Splits v = splits_of(s);
            splits = v.splits;
            WeightProduct q{dz, x, partial, s.last ? 1 : s.N, s.Ci, s.Co, s.last ? s.N * s.P : s.P, (int)ceil_div(s.Co, kBO),
                            (int)ceil_div(s.Ci ? s.Ci : 1, kBI), v.chunk, v.chunks, v.per, want_bias && !sums};
            const int64_t ctas = (int64_t)v.splits * q.tiles_o * q.tiles_i;
            if (ctas > INT32_MAX) return BC_ERR_BAD_SHAPE;
            e = with_type(s.io_kind, [&](auto t) {
                using T = decltype(t);
                const LaunchScope scope(KID_POINTWISE_WEIGHT, stream);
                if (s.last) launch_overlapped(pointwise_weight_kernel<T, true>, (unsigned)ctas, kThreads, 0, stream, q);
                else launch_overlapped(pointwise_weight_kernel<T, false>, (unsigned)ctas, kThreads, 0, stream, q);
                return check_launch("pointwise_weight_kernel");
            });
        }
        if (e) return e;
        if (want_weight) of_weights = {partial, pointwise_partial_stride(s.Co, s.Ci), weights, splits, grad_weight};
        if (want_bias && !sums) of_sums = {partial + weights, pointwise_partial_stride(s.Co, s.Ci), s.Co, splits, grad_bias};
    }
    const int64_t blocks = ceil_div(of_weights.count, 32), more = ceil_div(of_sums.count, 32);
    if (blocks + more > INT32_MAX) return BC_ERR_BAD_SHAPE;
    return with_type(s.io_kind, [&](auto t) {
        using T = decltype(t);
        const LaunchScope scope(KID_POINTWISE_FINISH, stream);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(blocks + more));
        cfg.blockDim = dim3(32, kFinishRows);
        cfg.stream = stream;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, pointwise_finish_kernel<T>, of_weights, of_sums, (unsigned)blocks);
        return check_launch("pointwise_finish_kernel");
    });
}

}  // namespace bc
