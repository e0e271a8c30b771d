// Pointwise convolution, out = act(W x + bias + residual) per pixel, and its gradients: which kernels serve a call, those of
// float multiply-adds for weights that the tensor cores' kernels (pointwise_mma.cu, pointwise_split.cu) do not hold, and the
// sums that end the weights' gradients.
//
// The products are of the form  D[m, n] = sum_k A[m, k] B[n, k]  with pixels and channels in turn:
//   forward      D[p, o] = sum_i x[i, p] W[o, i]           act(D + bias + residual) is stored
//   slope        the same product; grad * act'(D + bias + residual) = dz is stored
//   grad_input   D[p, i] = sum_o dz[o, p] W[o, i]
//   grad_weight  D[o, i] = sum_p dz[o, p] x[i, p]          split over the pixels; partial sums added in order
// By multiply-adds a CTA makes a tile of D from slices of 16 k that pass through shared memory as floats; a thread keeps 8 x 8 (8 x 4)
// sums in registers.
#include "bc_layers.cuh"

namespace bc {

namespace {

enum { FORWARD, SLOPE, INPUT };
constexpr int kThreads = 128, kBM = 128, kBK = 16;

struct Product {
    const void *a, *w, *bias, *residual, *grad;
    void *out;
    void *rest;              // INPUT: null, or what `a` lacks of dz; SLOPE: where that goes, or null
    int K, Cn;               // channels of A and of the output
    int wn, wk;              // strides of W along them
    int64_t P;               // pixels of a sample (of all of them together, channels last)
    int tiles_p, tiles_n;    // tiles of a sample's pixels, and of the output's channels
};

// Four values in a row, aligned.
template <typename T>
__device__ __forceinline__ float4 load4(const T *p)
{
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4 *>(p);
    } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        float4 v;
        widen2(w.x, v.x, v.y, T());
        widen2(w.y, v.z, v.w, T());
        return v;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4])
{
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(narrow2(v[0], v[1], T()), narrow2(v[2], v[3], T()));
}

// What becomes of four sums whose values lie in a row; `bias` four of them.
template <typename T, int MODE, int ACT, bool VEC>
__device__ __forceinline__ void finish4(const Product &q, int64_t at, float (&z)[4], const float (&bias)[4])
{
    const T *residual = static_cast<const T *>(q.residual) + at, *grad = static_cast<const T *>(q.grad) + at;
    T *out = static_cast<T *>(q.out) + at;
    if (MODE != INPUT) {
        float r[4] = {}, g[4];
        if (q.residual) *reinterpret_cast<float4 *>(r) = load4(residual);
        if (MODE == SLOPE) *reinterpret_cast<float4 *>(g) = load4(grad);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            z[i] += bias[i] + r[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const f2_t v = MODE == SLOPE ? times_slope2<ACT, T>(pack2(g[i], g[i + 1]), pack2(z[i], z[i + 1])) : activate2<ACT, T>(pack2(z[i], z[i + 1]));
            unpack2(v, z[i], z[i + 1]);
        }
    }
    store4<T>(out, z);
    if (MODE == SLOPE && q.rest) {
        float left[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) left[i] = left_by_rounding(z[i], from_float<T>(z[i]));
        store4<T>(static_cast<T *>(q.rest) + at, left);
    }
}

// D's tile: kBM pixels of a sample x BN channels.  VEC: rows and arrays allow vectors of four values; a thread's pixels are
// 4 tm + {0..3} and 64 + that.  Otherwise they are tm + 16 i, so that neighbouring lanes store neighbouring values.
// Multiply-adds go two pixels an instruction; the weights' slice holds every weight twice for that.
// Measured (f32, 128 -> 32, 16 x 64 x 128 planes): one value an instruction, scalar stores 40 us.
template <typename T, int MODE, int ACT, bool LAST, int BN, bool VEC>
__global__ void __launch_bounds__(kThreads, BN == 64 ? 3 : 4) pointwise_kernel(Product q)
{
    constexpr int TN = BN / 8;      // channels of a thread
    __shared__ __align__(16) float As[2][kBK][kBM + 4];
    __shared__ __align__(16) float2 Bs[2][kBK][BN + 2];
    const int tid = threadIdx.x, tm = tid & 15, tn = tid >> 4;
    const unsigned tile = blockIdx.x / (unsigned)q.tiles_n;
    const int n0 = (int)(blockIdx.x - tile * q.tiles_n) * BN;
    const int64_t sample = tile / (unsigned)q.tiles_p, p0 = (int64_t)(tile - (unsigned)sample * q.tiles_p) * kBM;
    const int pixels = (int)min((int64_t)kBM, q.P - p0);
    const T *a = static_cast<const T *>(q.a) + sample * q.K * q.P + (LAST ? p0 * q.K : p0);
    const T *w = static_cast<const T *>(q.w);
    const T *a_rest = MODE == INPUT && q.rest ? static_cast<const T *>(q.rest) + (a - static_cast<const T *>(q.a)) : nullptr;
    grid_dependency_wait();

    float ra[16], rb[BN / 8];
    auto load = [&](int k0) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = tid + kThreads * j, k = k0 + (LAST ? 4 * (e & 3) : e >> 5), m = LAST ? e >> 2 : 4 * (e & 31);
                const int64_t at = LAST ? (int64_t)m * q.K + k : k * q.P + m;
                const bool there = k < q.K && m < pixels;
                float4 v = there ? load4(a + at) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (MODE == INPUT && a_rest && there) {
                    const float4 u = load4(a_rest + at);
                    v = make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
                }
                *reinterpret_cast<float4 *>(ra + 4 * j) = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int k = k0 + (LAST ? tid & 15 : j), m = LAST ? (tid >> 4) + 8 * j : tid;
                const int64_t at = LAST ? (int64_t)m * q.K + k : k * q.P + m;
                ra[j] = k < q.K && m < pixels ? to_float(a[at]) + (MODE == INPUT && a_rest ? to_float(a_rest[at]) : 0.f) : 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < BN / 8; ++j) {
            const int e = tid + kThreads * j;
            const int k = k0 + (MODE == INPUT ? e / BN : e % kBK), n = n0 + (MODE == INPUT ? e % BN : e / kBK);
            rb[j] = k < q.K && n < q.Cn ? to_float(w[(int64_t)n * q.wn + (int64_t)k * q.wk]) : 0.f;
        }
    };
    auto store = [&](int b) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = tid + kThreads * j;
                if (LAST) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) As[b][4 * (e & 3) + i][e >> 2] = ra[4 * j + i];
                } else {
                    *reinterpret_cast<float4 *>(&As[b][e >> 5][4 * (e & 31)]) = *reinterpret_cast<const float4 *>(ra + 4 * j);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) As[b][LAST ? tid & 15 : j][LAST ? (tid >> 4) + 8 * j : tid] = ra[j];
        }
#pragma unroll
        for (int j = 0; j < BN / 8; ++j) {
            const int e = tid + kThreads * j;
            Bs[b][MODE == INPUT ? e / BN : e % kBK][MODE == INPUT ? e % BN : e / kBK] = make_float2(rb[j], rb[j]);
        }
    };

    // pairs of pixels: VEC, 4 tm + {0, 1}, {2, 3} and 64 + those; tm + 16 {2 i, 2 i + 1} otherwise
    f2_t acc[4][TN];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = both(0.f);
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
            f2_t av[4], bv[TN];
            if constexpr (VEC) {
                const ulonglong2 u = *reinterpret_cast<const ulonglong2 *>(&As[b][k][4 * tm]), v = *reinterpret_cast<const ulonglong2 *>(&As[b][k][64 + 4 * tm]);
                av[0] = u.x;
                av[1] = u.y;
                av[2] = v.x;
                av[3] = v.y;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) av[i] = pack2(As[b][k][tm + 32 * i], As[b][k][tm + 32 * i + 16]);
            }
            // channel 32 (j / 4) + 4 tn + j % 4
#pragma unroll
            for (int j = 0; j < TN; j += 2) {
                const ulonglong2 u = *reinterpret_cast<const ulonglong2 *>(&Bs[b][k][32 * (j / 4) + 4 * tn + j % 4]);
                bv[j] = u.x;
                bv[j + 1] = u.y;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = fma2(av[i], bv[j], acc[i][j]);
        }
        if (more) store(b ^ 1);
        __syncthreads();
    }

    const int64_t base = sample * q.Cn * q.P + (LAST ? p0 * q.Cn : p0);
    const T *bias = static_cast<const T *>(q.bias), *residual = static_cast<const T *>(q.residual), *grad = static_cast<const T *>(q.grad);
    T *out = static_cast<T *>(q.out);
#pragma unroll
    for (int j4 = 0; j4 < TN; j4 += 4) {
        const int n = n0 + 8 * j4 + 4 * tn;      // four channels from here
        float b4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b4[j] = MODE != INPUT && bias && n + j < q.Cn ? to_float(bias[n + j]) : 0.f;
        if constexpr (VEC && LAST) {
            if (n < q.Cn)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int m = 64 * (i / 4) + 4 * tm + i % 4;
                    if (m >= pixels) continue;
                    float z[4], other;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (i % 2) unpack2(acc[i / 2][j4 + j], other, z[j]);
                        else unpack2(acc[i / 2][j4 + j], z[j], other);
                    }
                    finish4<T, MODE, ACT, VEC>(q, base + (int64_t)m * q.Cn + n, z, b4);
                }
        } else if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n + j >= q.Cn) continue;
                const float bj[4] = {b4[j], b4[j], b4[j], b4[j]};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int m = 64 * h + 4 * tm;
                    if (m >= pixels) continue;
                    float z[4];
                    unpack2(acc[2 * h][j4 + j], z[0], z[1]);
                    unpack2(acc[2 * h + 1][j4 + j], z[2], z[3]);
                    finish4<T, MODE, ACT, VEC>(q, base + (n + j) * q.P + m, z, bj);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (n + j >= q.Cn) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float z[2];
                    unpack2(acc[i][j4 + j], z[0], z[1]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int m = tm + 32 * i + 16 * h;
                        if (m >= pixels) continue;
                        const int64_t at = base + (LAST ? (int64_t)m * q.Cn + n + j : (n + j) * q.P + m);
                        float v = z[h] + b4[j];
                        if (MODE != INPUT && residual) v += to_float(residual[at]);
                        v = MODE == FORWARD ? activate<ACT, T>(v) : MODE == SLOPE ? times_slope<ACT, T>(to_float(grad[at]), v) : v;
                        const T rounded = from_float<T>(v);
                        out[at] = rounded;
                        if (MODE == SLOPE && q.rest) static_cast<T *>(q.rest)[at] = from_float<T>(left_by_rounding(v, rounded));
                    }
                }
            }
        }
    }
}

// Rows of partial sums, added in a fixed order (in double: there may be thousands), rounded once: `count` columns, `stride` floats from row to row.
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
    __shared__ double part[kFinishRows][32];
    const Partials &q = blockIdx.x < blocks ? weights : sums;
    const int64_t e = (int64_t)(blockIdx.x < blocks ? blockIdx.x : blockIdx.x - blocks) * 32 + threadIdx.x;
    grid_dependency_wait();
    double v = 0;
    if (e < q.count) {
#pragma unroll 8
        for (int i = threadIdx.y; i < q.rows; i += kFinishRows) v += q.from[i * q.stride + e];
    }
    part[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y || e >= q.count) return;
    for (int i = 1; i < kFinishRows; ++i) v += part[i][threadIdx.x];
    static_cast<T *>(q.to)[e] = from_float<T>((float)v);
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
            auto go = [&](auto last, auto vec) {
                constexpr bool LAST = decltype(last)::value, VEC = decltype(vec)::value;
                bn == 32 ? launch_overlapped(pointwise_kernel<T, MODE, ACT, LAST, 32, VEC>, grid, kThreads, 0, stream, q)
                         : launch_overlapped(pointwise_kernel<T, MODE, ACT, LAST, 64, VEC>, grid, kThreads, 0, stream, q);
                return check_launch("pointwise_kernel");
            };
            const bool vec = (s.last ? q.K % 4 == 0 && q.Cn % 4 == 0 : q.P % 4 == 0) && pointwise_mma_aligned(q.a, q.residual, q.grad, q.out);
            if (s.last) return vec ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
            return vec ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
        });
    });
}

size_t partial_bytes(const PointwiseShape &s)
{
    // (whichever kernel's: the query does not know the arrays)
    return align_up((size_t)std::max(pointwise_mma_weight_splits(s), pointwise_split_weight_splits(s, false)) * pointwise_partial_stride(s.Co, s.Ci) * sizeof(float));
}
// Which kernel a product with pixels in the rows takes.
enum { BY_TMA, BY_SPLIT, BY_FMA };
int way_of(const PointwiseShape &s, bool input, bool aligned)
{
    if (aligned && pointwise_mma_suits(s, input)) return BY_TMA;
    return pointwise_split_suits(s, input) ? BY_SPLIT : BY_FMA;
}
int sums_rows(const PointwiseShape &s, int way)
{
    return way == BY_TMA ? pointwise_mma_sums_rows(s) : way == BY_SPLIT ? pointwise_split_sums_rows(s) : 0;
}
// (for either: the query does not know the arrays)
size_t sums_bytes(const PointwiseShape &s)
{
    return align_up((size_t)std::max(sums_rows(s, way_of(s, false, true)), sums_rows(s, way_of(s, false, false))) * s.Co * sizeof(float));
}
// dz in memory, where it is neither grad_output itself nor asked for.
bool own_dz(const PointwiseShape &s, int need_mask) { return s.act != BC_ACT_NONE && !(need_mask & BC_NEED_PW_RESIDUAL); }
// A 16-bit dz goes into its products as its rounding (grad_residual) and what that leaves, rounded: off by u^2 of it.  With
// the rounding alone grad_input and grad_weight were 1.4 times as far from their definition as one rounding puts them; a step of
// (64,256->256,64,128) bf16 last with GELU took 706 us, and takes 831 to 883.
bool keeps_rest(const PointwiseShape &s, int need_mask)
{
    return s.act != BC_ACT_NONE && s.io_kind != BC_IO_F32 && (need_mask & (BC_NEED_PW_INPUT | BC_NEED_PW_WEIGHT | BC_NEED_PW_BIAS));
}
size_t dz_bytes(const PointwiseShape &s) { return align_up((size_t)io_size(s.io_kind) * s.N * s.Co * s.P); }

}  // namespace

int launch_pointwise_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual, void *out,
                             cudaStream_t stream)
{
    const int way = way_of(s, false, pointwise_mma_aligned(x, weight, residual, out));
    if (way == BY_TMA) return launch_pointwise_mma_forward(s, x, weight, bias, residual, out, stream);
    if (way == BY_SPLIT) return launch_pointwise_split_forward(s, x, weight, bias, residual, out, stream);
    return launch_product<FORWARD>(s, {x, weight, bias, residual, nullptr, out, nullptr, s.Ci, s.Co, s.Ci, 1}, stream);
}

size_t pointwise_workspace(const PointwiseShape &s, int need_mask)
{
    size_t bytes = ((own_dz(s, need_mask) ? 1 : 0) + (keeps_rest(s, need_mask) ? 1 : 0)) * dz_bytes(s);
    if (need_mask & (BC_NEED_PW_WEIGHT | BC_NEED_PW_BIAS)) bytes += partial_bytes(s);
    if ((need_mask & BC_NEED_PW_BIAS) && s.act != BC_ACT_NONE) bytes += sums_bytes(s);
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
    void *rest = nullptr;
    float *sums = nullptr;      // rows of sums of dz as it was before its rounding
    int rows = 0;
    if (s.act != BC_ACT_NONE) {
        void *to = own_dz(s, need_mask) ? take(dz_bytes(s)) : grad_residual;
        if (keeps_rest(s, need_mask)) rest = take(dz_bytes(s));
        const int way = way_of(s, false, pointwise_mma_aligned(x, weight, residual, grad, to));
        if (want_bias && way != BY_FMA) {
            sums = static_cast<float *>(take(sums_bytes(s)));
            rows = sums_rows(s, way);
        }
        const int e = way == BY_TMA     ? launch_pointwise_mma_slope(s, x, weight, bias, residual, grad, to, rest, sums, stream)
                      : way == BY_SPLIT ? launch_pointwise_split_slope(s, x, weight, bias, residual, grad, to, rest, sums, stream)
                                        : launch_product<SLOPE>(s, {x, weight, bias, residual, grad, to, rest, s.Ci, s.Co, s.Ci, 1}, stream);
        if (e) return e;
        dz = to;
    }
    if (need_mask & BC_NEED_PW_INPUT) {
        const int way = way_of(s, true, pointwise_mma_aligned(dz, weight, grad_input));
        const int e = way == BY_TMA     ? launch_pointwise_mma_input(s, dz, rest, weight, grad_input, stream)
                      : way == BY_SPLIT ? launch_pointwise_split_input(s, dz, rest, weight, grad_input, stream)
                                        : launch_product<INPUT>(s, {dz, weight, nullptr, nullptr, nullptr, grad_input, rest, s.Co, s.Ci, 1, s.Ci}, stream);
        if (e) return e;
    }
    if (!want_weight && !want_bias) return BC_OK;
    const int64_t weights = (int64_t)s.Co * s.Ci;
    Partials of_weights{}, of_sums{};
    if (sums) of_sums = {sums, s.Co, s.Co, rows, grad_bias};
    if (want_weight || !sums) {
        float *partial = static_cast<float *>(take(partial_bytes(s)));
        int splits = pointwise_mma_aligned(dz, x) ? pointwise_mma_weight_splits(s) : 0;
        int e = BC_ERR_BAD_SHAPE;
        if (splits) e = launch_pointwise_mma_weight(s, dz, rest, x, partial, want_bias && !sums, stream);
        else if ((splits = pointwise_split_weight_splits(s, rest))) e = launch_pointwise_split_weight(s, dz, rest, x, partial, want_bias && !sums, stream);
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
