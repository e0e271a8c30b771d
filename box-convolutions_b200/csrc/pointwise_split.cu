// Pointwise convolutions on the tensor cores with operands that threads bring into shared memory: float tensors, and 16-bit
// ones whose rows TMA does not take (odd planes, channels that are no multiple of eight).  The products of pointwise.cu with
// pixels in the rows, built like pointwise_mma_kernel: persistent CTAs, weights in shared memory, two sets of accumulators.
//
// A float is the sum of three bf16 values: itself rounded, what is left rounded, and what is left then.  A product of floats is that
// of nine pairs; the six are made that reach above 2^-26 of it: the upper ones into one accumulator, the others into a second or a
// third, added at the end.  (An accumulator's additions round towards zero: the others stay 2^-8 of the first, which sees a
// sixth of the additions.)  Measured against multiply-adds, which wait for shared memory here ((16,128->32,64,128) planes: 38 us).
// With them 26 us forward, 34 with the slope, 35 grad_input, 42 grad_weight (13 to 15 at the copy bandwidth): an instruction takes
// some 90 cycles here whether it is 32 or 128 columns wide, and splitting the operands about as long as the products.
// Infinities and NaN have no such sum: a result that is not finite is computed again by multiply-adds.  (Parts end at 2^-133, bf16's
// smallest number: operands below 2^-110 lose digits.)
#include "bc_mma.cuh"

namespace bc {

namespace {

enum { FORWARD, SLOPE, INPUT };
constexpr int kEpilogue = 8, kGroups = 2, kGroupWarps = 4;
constexpr int kThreads = 32 * (kEpilogue + kGroups * kGroupWarps + 1);
constexpr int kPitch = 17;
constexpr uint32_t kPart = 16384;      // 128 pixels x 64 k
constexpr uint32_t kCopies = 32768;    // the same in floats
constexpr int kProducers = 32 * kGroups * kGroupWarps;
constexpr uint32_t kMostShared = 227 << 10;

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 1;

struct SplitProduct {
    const void *a, *w, *bias, *residual, *grad;
    void *out;
    void *rest;              // 16-bit.  INPUT: null, or what `a` lacks of dz; SLOPE: where that goes, or null
    float *sums;             // SLOPE: [CTA / tiles_n][Cn] sums of dz over the CTA's pixels, or null
    int64_t P;               // pixels of a sample (of all of them together, channels last)
    int K, Cn, samples;
    int wn, wk;              // strides of W along the output's and the operand's channels
    int tiles_p, tiles_n;
    int bn, stages, columns;
    bool merged;             // float: the weights' three parts are one operand, and three sets of sums lie side by side
    uint32_t instruction;
};

// Shared memory from a 1024-byte boundary on.
struct SplitLayout {
    int bn, stages, chunks, parts;
    bool last;
    __host__ __device__ uint32_t slice() const { return (uint32_t)bn * 128; }      // 64 k of one part of the weights
    __host__ __device__ uint32_t ring() const { return parts * chunks * slice(); }
    __host__ __device__ uint32_t copies() const { return ring() + stages * parts * kPart; }      // a slice of floats as they come
    __host__ __device__ uint32_t staging() const { return copies() + (parts == 3 ? kCopies : 0); }
    __host__ __device__ uint32_t bias() const { return staging() + (last ? kEpilogue * 32 * kPitch * 4 : 0); }
    __host__ __device__ uint32_t sums() const { return bias() + bn * 4; }
    __host__ __device__ uint32_t barriers() const { return (sums() + 4 * bn * 4 + 7) / 8 * 8; }
    __host__ __device__ uint32_t bytes() const { return barriers() + (2 * stages + 4) * 8 + 8 + 1024; }
};

// Floats, two and four of them, as bf16 parts.  (An infinity leaves a NaN behind: what comes of it is computed again.)
__device__ __forceinline__ void split2(float a, float b, uint32_t (&part)[3])
{
    f2_t x = pack2(a, b);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        float lo, hi;
        unpack2(x, lo, hi);
        part[p] = narrow2(lo, hi, __nv_bfloat16());
        if (p == 2) break;
        widen2(part[p], lo, hi, __nv_bfloat16());
        x = sub2(x, pack2(lo, hi));
    }
}
// Into their place of every part, `part` bytes apart.
__device__ __forceinline__ void place4(char *to, uint32_t part, const float4 &v)
{
    uint32_t lo[3], hi[3];
    split2(v.x, v.y, lo);
    split2(v.z, v.w, hi);
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<uint2 *>(to + p * part) = make_uint2(lo[p], hi[p]);
}
// Four of them on their way into the thread's own place in shared memory, zeros beyond n.
template <bool VEC>
__device__ __forceinline__ void copy4(uint32_t to, const float *from, int n, const float *base)
{
    if (VEC) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(n > 0 ? from : base), "r"(n > 0 ? 16 : 0) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4 * i), "l"(n > i ? from + i : base), "r"(n > i ? 4 : 0) : "memory");
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All of the thread's but the newest `slots - 1` groups have arrived.
__device__ __forceinline__ void copies_wait(int slots)
{
    if (slots > 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Eight 16-bit values from `from` on, of which `n` are there (zeros beyond); VEC: whole vectors, aligned.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const T *from, int n)
{
    if constexpr (VEC) return n > 0 ? *reinterpret_cast<const uint4 *>(from) : make_uint4(0, 0, 0, 0);
    const unsigned short *bits = reinterpret_cast<const unsigned short *>(from);
    uint32_t f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? bits[i] : 0;
    return make_uint4(f[0] | f[1] << 16, f[2] | f[3] << 16, f[4] | f[5] << 16, f[6] | f[7] << 16);
}

template <typename T, int MODE, int ACT, bool LAST, bool VEC>
__global__ void __launch_bounds__(kThreads, 1) pointwise_split_kernel(const SplitProduct q)
{
    constexpr int PARTS = kParts<T>;
    extern __shared__ char raw_smem[];
    const uint32_t raw = smem_u32(raw_smem), base = (raw + 1023) & ~1023u;
    char *smem = raw_smem + (base - raw);
    const int chunks = (q.K + 63) / 64, sources = PARTS == 1 && MODE == INPUT && q.rest ? 2 : 1;      // tensors that A is the sum of
    const SplitLayout lay{q.bn, q.stages, chunks, PARTS, LAST};
    float *bias_smem = reinterpret_cast<float *>(smem + lay.bias()), *sums_smem = reinterpret_cast<float *>(smem + lay.sums());
    const uint32_t full = base + lay.barriers(), empty = full + 8 * q.stages, ready = empty + 8 * q.stages, drained = ready + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + lay.barriers() + (2 * q.stages + 4) * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned walkers = gridDim.x / (unsigned)q.tiles_n, walker = blockIdx.x / (unsigned)q.tiles_n;
    const int n0 = (int)(blockIdx.x - walker * q.tiles_n) * q.bn;
    const unsigned tiles = (unsigned)q.samples * (unsigned)q.tiles_p;      // (below 2^31)
    const uint32_t set_columns = q.merged ? q.columns : (PARTS > 1 ? 2 : 1) * q.columns;
    const T *w_all = static_cast<const T *>(q.w), *a_all = static_cast<const T *>(q.a);

    if (threadIdx.x == 0) {
        for (int i = 0; i < q.stages; ++i) {
            mbar_init(full + 8 * i, PARTS == 3 ? kGroups * kGroupWarps : kGroupWarps);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(ready + 8 * i, 1);
            mbar_init(drained + 8 * i, kEpilogue);
        }
        fence_mbar_init();
    }
    __syncthreads();
    grid_dependency_wait();
    if (warp == kEpilogue + kGroups * kGroupWarps) tmem_alloc(tmem_slot, 2 * set_columns);
    for (int i = threadIdx.x; i < q.bn; i += kThreads)
        bias_smem[i] = MODE != INPUT && q.bias && n0 + i < q.Cn ? to_float(static_cast<const T *>(q.bias)[n0 + i]) : 0.f;
    for (int i = threadIdx.x; i < 4 * q.bn; i += kThreads) sums_smem[i] = 0.f;
    // A producer's way through this CTA's slices, the sources of a slice in turn.
    struct Cursor {
        unsigned tile;
        int c;
    };
    auto advance = [&](Cursor &at) {
        if (++at.c == sources * chunks) {
            at.c = 0;
            at.tile += walkers;
        }
    };
    // Producers of floats: a thread has eight vectors of four floats of a slice, copies them to a place of its own and splits them
    // from there, the next slice's on their way.
    const int t = (int)threadIdx.x - 32 * kEpilogue;
    const float *all = reinterpret_cast<const float *>(q.a);
    const char *own = smem + lay.copies() + 16 * t;
    // planes: four pixels of a k; last: four k of a pixel
    const int in = 4 * (LAST ? t & 15 : t & 31), outer0 = LAST ? t >> 4 : t >> 5, outer_step = LAST ? kProducers / 16 : kProducers / 32;
    const int64_t pitch = LAST ? (int64_t)q.K : q.P;
    Cursor ahead{walker, 0};
    auto copy = [&] {
        if (ahead.tile < tiles) {
            const unsigned sample = ahead.tile / (unsigned)q.tiles_p;
            const int64_t p0 = (int64_t)(ahead.tile - sample * q.tiles_p) * 128;
            const int pixels = (int)min((int64_t)128, q.P - p0), k_left = q.K - 64 * ahead.c;
            const float *a = all + (LAST ? p0 * q.K + 64 * ahead.c : ((int64_t)sample * q.K + 64 * ahead.c) * q.P + p0) + outer0 * pitch + in;
            const int inner = (LAST ? k_left : pixels) - in, outers = (LAST ? pixels : k_left) - outer0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                copy4<VEC>(smem_u32(own) + 4096 * j, a + j * outer_step * pitch, j * outer_step < outers ? inner : 0, all);
            advance(ahead);
        }
        copies_commit();
    };
    const bool produces = warp >= kEpilogue && warp < kEpilogue + kGroups * kGroupWarps;
    if (PARTS == 3 && produces) copy();      // (the first slice is on its way while the weights are placed)
    // the weights, K-major, eight k a thread
    {
        for (int e = threadIdx.x; e < q.bn * chunks * 8; e += kThreads) {
            // (along the weights' rows: k forward, channels for grad_input)
            const int n = MODE == INPUT ? e % q.bn : e / (chunks * 8), k8 = MODE == INPUT ? e / q.bn : e % (chunks * 8);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = 8 * k8 + j;
                v[j] = k < q.K && n0 + n < q.Cn ? to_float(w_all[(int64_t)(n0 + n) * q.wn + (int64_t)k * q.wk]) : 0.f;
            }
            char *to = smem + (k8 >> 3) * PARTS * lay.slice() + n * 128 + (((k8 & 7) ^ (n & 7)) << 4);
            if constexpr (PARTS == 3) {
                place4(to, lay.slice(), make_float4(v[0], v[1], v[2], v[3]));
                place4(to + 8, lay.slice(), make_float4(v[4], v[5], v[6], v[7]));
            } else {
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = narrow2(v[2 * j], v[2 * j + 1], T());
                *reinterpret_cast<uint4 *>(to) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        }
    }
    fence_proxy_async();
    tmem_release();
    __syncthreads();
    tmem_acquire();
    const uint32_t tmem = *tmem_slot;
    Waiter wait;

    if (PARTS == 3 && produces) {
        uint32_t stage = 0, phase = 0;
        for (Cursor at{walker, 0}; at.tile < tiles; advance(at)) {
            copies_wait(1);
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const float4 *>(own + 4096 * j);
            copy();
            if (__any_sync(0xffffffffu, !wait(empty + 8 * stage, phase ^ 1))) break;
            char *to = smem + lay.ring() + stage * PARTS * kPart + (in & 4) * 2;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int outer = outer0 + j * outer_step;
                place4(to + (LAST ? 0 : (in >> 6) * kBlockBytes) + outer * 128 + ((((in >> 3) & 7) ^ (outer & 7)) << 4), kPart, v[j]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * stage);
            if (++stage == (uint32_t)q.stages) {
                stage = 0;
                phase ^= 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= kEpilogue && warp < kEpilogue + kGroups * kGroupWarps) {
        // group g brings every second slice: while one waits for memory the other writes
        const int group = (warp - kEpilogue) / kGroupWarps, t = threadIdx.x - 32 * (kEpilogue + group * kGroupWarps);
        uint32_t stage = group, phase = 0;
        Cursor at{walker, 0};
        if (group) advance(at);
        for (; at.tile < tiles; advance(at), advance(at)) {
            const int c = sources == 2 ? at.c >> 1 : at.c;
            const unsigned sample = at.tile / (unsigned)q.tiles_p;
            const int64_t p0 = (int64_t)(at.tile - sample * q.tiles_p) * 128;
            const int pixels = (int)min((int64_t)128, q.P - p0), k_left = q.K - 64 * c, k_used = (k_left + 15) / 16 * 16;
            const T *a = (sources == 2 && (at.c & 1) ? static_cast<const T *>(q.rest) : a_all) +
                         (LAST ? p0 * q.K + 64 * c : ((int64_t)sample * q.K + 64 * c) * q.P + p0);
            // a vector: planes, eight pixels of a k; last, eight k of a pixel.  `inner` of it are there.
            uint4 raw_v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = t + 128 * j, in = 8 * (LAST ? e & 7 : e & 15), outer = LAST ? e >> 3 : e >> 4;
                const int inner = outer < (LAST ? pixels : k_left) ? (LAST ? k_left : pixels) - in : 0;
                const T *from = a + outer * (LAST ? (int64_t)q.K : q.P) + in;
                if constexpr (PARTS == 1) raw_v[j] = load8<T, VEC>(from, inner);
            }
            if (__any_sync(0xffffffffu, !wait(empty + 8 * stage, phase ^ 1))) break;
            char *to = smem + lay.ring() + stage * PARTS * kPart;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = t + 128 * j;
                const uint32_t place = LAST ? (e >> 3) * 128 + (((e & 7) ^ (e >> 3 & 7)) << 4)
                                            : (e >> 3 & 1) * kBlockBytes + (e >> 4) * 128 + (((e & 7) ^ (e >> 4 & 7)) << 4);
                if ((LAST ? 8 * (e & 7) : e >> 4) >= k_used) continue;
                *reinterpret_cast<uint4 *>(to + place) = raw_v[j];
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * stage);
            if ((stage += kGroups) >= (uint32_t)q.stages) {
                stage -= q.stages;
                phase ^= 1;
            }
        }
    } else if (warp == kEpilogue + kGroups * kGroupWarps) {
        if (lane == 0) {
            const uint64_t ring = LAST ? k_major(base + lay.ring(), 0) : mn_major(base + lay.ring(), 0, kBlockBytes);
            const uint64_t weights = k_major(base, 0);
            uint32_t stage = 0, phase = 0, set = 0, set_phase = 0;
            for (unsigned tile = walker; tile < tiles; tile += walkers) {
                if (!wait(drained + 8 * set, set_phase ^ 1)) break;
                tmem_acquire();
                for (int piece = 0; piece < sources * chunks; ++piece) {
                    if (!wait(full + 8 * stage, phase)) break;
                    tmem_acquire();
                    const int c = sources == 2 ? piece >> 1 : piece;
                    const uint64_t a = further(ring, stage * PARTS * kPart);
                    const uint64_t w = further(weights, c * PARTS * lay.slice());
                    const int k_used = q.K - 64 * c;
                    const uint32_t d = tmem + set * set_columns;
#pragma unroll
                    for (int k = 0; k < 64; k += 16)
                        if (k < k_used) {
                            const uint64_t ak = further(a, (LAST ? 2 : 128) * k), wk = further(w, 2 * k);
                            if (PARTS == 3 && q.merged) {
                                // the weights' parts in a row are one operand: an instruction takes some 90 cycles at any width here
                                mma(d, ak, wk, q.instruction, piece || k);
                                mma(d + q.bn, further(ak, kPart), wk, q.instruction - (q.bn >> 3 << 17), true);
                                mma(d + 2 * q.bn, further(ak, 2 * kPart), wk, q.instruction - (2 * q.bn >> 3 << 17), true);
                            } else {
#pragma unroll
                                for (int i = 0; i < PARTS; ++i)
#pragma unroll
                                    for (int j = 0; j < PARTS - i; ++j)
                                        mma(i + j ? d + q.columns : d, further(ak, i * kPart), further(wk, j * lay.slice()), q.instruction,
                                            piece || k || i + j > 1 || i > 0);
                            }
                        }
                    mma_commit(empty + 8 * stage);
                    if (++stage == (uint32_t)q.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (wait.lost) break;
                mma_commit(ready + 8 * set);
                if (set ^= 1; set == 0) set_phase ^= 1;
            }
        }
    } else {
        float *staging = reinterpret_cast<float *>(smem + lay.staging()) + warp * 32 * kPitch;
        const int quarter = warp & 3, half = warp >> 2, blocks = q.bn / 16;
        const T *residual = static_cast<const T *>(q.residual), *grad = static_cast<const T *>(q.grad);
        T *out = static_cast<T *>(q.out), *rest = static_cast<T *>(q.rest);
        uint32_t set = 0, set_phase = 0;
        for (unsigned tile = walker; tile < tiles; tile += walkers) {
            const unsigned sample = tile / (unsigned)q.tiles_p;
            const int64_t p0 = (int64_t)(tile - sample * q.tiles_p) * 128 + quarter * 32;
            const int rows = (int)max((int64_t)0, min((int64_t)32, q.P - p0));
            // Blocks of 16 channels, 16 values a lane, coalesced: planes, the lane's pixel and channel i; last, pixel
            // 2 i + (lane >> 4) and channel lane & 15.  What the block reads is on its way before its sums are there.
            bool waited = false;
            for (int b = half; b < blocks || !waited; b += 2) {
                const int c0 = n0 + 16 * b, channels = min(16, q.Cn - c0);
                const int64_t at = LAST ? (p0 + (lane >> 4)) * q.Cn + c0 + (lane & 15) : ((int64_t)sample * q.Cn + c0) * q.P + p0 + lane;
                const int64_t step = LAST ? 2 * (int64_t)q.Cn : q.P;
                auto there = [&](int i) { return LAST ? 2 * i + (lane >> 4) < rows && (lane & 15) < channels : lane < rows && i < channels; };
                T res[16], g[16];
                if (b < blocks) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (MODE != INPUT && residual && there(i)) res[i] = residual[at + i * step];
                        if (MODE == SLOPE && there(i)) g[i] = grad[at + i * step];
                    }
                }
                if (!waited) {
                    waited = true;
                    wait(ready + 8 * set, set_phase);
                    __syncwarp();
                    tmem_acquire();
                    if (b >= blocks) break;
                }
                float v[16];
                const uint32_t from = tmem + set * set_columns + 16 * b + ((uint32_t)quarter << 21);
                accumulators16(from, v);
                if constexpr (PARTS == 3) {
                    float u[16], finite = 0.f;
                    if (q.merged) {
                        float u2[16];
                        accumulators16(from + q.bn, u);
                        accumulators16(from + 2 * q.bn, u2);
#pragma unroll
                        for (int j = 0; j < 16; ++j) u[j] += u2[j];
                    } else {
                        accumulators16(from + q.columns, u);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        v[j] += u[j];
                        finite = fmaf(v[j], 0.f, finite);
                    }
                    if (finite != 0.f && lane < rows) {      // (a NaN: some value is not finite)
#pragma unroll
                        for (int j = 0; j < 16; ++j) u[j] = 0.f;
                        for (int k = 0; k < q.K; ++k) {
                            const float x = to_float(a_all[LAST ? (p0 + lane) * q.K + k : ((int64_t)sample * q.K + k) * q.P + p0 + lane]);
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (j < channels) u[j] = fmaf(x, to_float(w_all[(int64_t)(c0 + j) * q.wn + (int64_t)k * q.wk]), u[j]);
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (!(fabsf(v[j]) < INFINITY)) v[j] = u[j];
                    }
                    __syncwarp();
                }
                if (LAST) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) staging[lane * kPitch + j] = v[j];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = staging[(2 * i + (lane >> 4)) * kPitch + (lane & 15)];
                    __syncwarp();
                }
                float total = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    if (MODE != INPUT) {
                        const float *bias = bias_smem + 16 * b;
                        float z[2], gg[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            z[h] = v[i + h] + bias[LAST ? lane & 15 : i + h];
                            if (residual && there(i + h)) z[h] += to_float(res[i + h]);
                            gg[h] = MODE == SLOPE && there(i + h) ? to_float(g[i + h]) : 0.f;
                        }
                        const f2_t zz = pack2(z[0], z[1]);
                        unpack2(MODE == SLOPE ? times_slope2<ACT, T>(pack2(gg[0], gg[1]), zz) : activate2<ACT, T>(zz), v[i], v[i + 1]);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (there(i + h)) {
                            const T rounded = from_float<T>(v[i + h]);
                            out[at + (i + h) * step] = rounded;
                            if (PARTS == 1 && MODE == SLOPE && rest) rest[at + (i + h) * step] = from_float<T>(left_by_rounding(v[i + h], rounded));
                        } else {
                            v[i + h] = 0.f;
                        }
                        if (LAST) total += v[i + h];
                    }
                }
                if (MODE == SLOPE && q.sums) {
                    if (LAST) {
                        total += __shfl_xor_sync(0xffffffffu, total, 16);
                    } else {      // sixteen channels over the lanes
                        fold(v, lane, 8, 8);
                        fold(v, lane, 4, 4);
                        fold(v, lane, 2, 2);
                        fold(v, lane, 1, 1);
                        total = v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
                    }
                    if (lane < 16) sums_smem[quarter * q.bn + 16 * b + lane] += total;
                }
            }
            tmem_release();
            __syncwarp();
            if (lane == 0) mbar_arrive(drained + 8 * set);
            if (__any_sync(0xffffffffu, wait.lost)) break;
            if (set ^= 1; set == 0) set_phase ^= 1;
        }
    }
    if (wait.lost) let_copies_land();
    __syncwarp();
    tmem_release();
    __syncthreads();
    if (warp == kEpilogue + kGroups * kGroupWarps) tmem_free(tmem, 2 * set_columns);
    if (MODE == SLOPE && q.sums)
        for (int i = threadIdx.x; i < q.bn; i += kThreads)
            if (n0 + i < q.Cn)
                q.sums[(int64_t)walker * q.Cn + n0 + i] = (sums_smem[i] + sums_smem[q.bn + i]) + (sums_smem[2 * q.bn + i] + sums_smem[3 * q.bn + i]);
}

// ---- grad_weight, D[o, i] = sum_p dz[o, p] x[i, p]: 128 x up to 256 (float 128) weights, split over the pixels; built like
// pointwise_weight_mma_kernel, slices of 64 pixels.  Planes are K-major operands, rows of 64 pixels; channels last MN-major.

constexpr int kWeightEpilogue = 4, kWeightThreads = 32 * (kWeightEpilogue + kGroups * kGroupWarps + 1);

struct WeightSplit {
    const void *dz, *rest, *x;      // (rest: 16-bit, what dz lacks, or null)
    float *partial;          // a row a split: Co * Ci sums, then Co sums of dz
    int64_t P;
    int per, slices;         // slices of a split; of a sample
    int samples, Ci, Co;
    int tiles_i;
    int rows, bn, stages, slots, columns;      // output and input channels of a tile; ring; floats' slices on their way
    SumColumns sums_at;
    bool sums;
    uint32_t instruction;
};

struct WeightSplitLayout {
    int rows, bn, stages, slots, parts, sources;      // (sources: tensors that dz is the sum of)
    bool last;
    __host__ __device__ uint32_t bytes_of(int channels) const { return last ? (uint32_t)((channels + 63) / 64) * kBlockBytes : (uint32_t)channels * 128; }
    // (M is 128 whatever there is of dz: what lies behind its rows is read as well, and leads nowhere)
    __host__ __device__ uint32_t dz_part() const { return bytes_of(rows); }
    __host__ __device__ uint32_t x_part() const { return bytes_of(bn); }
    __host__ __device__ uint32_t x_at() const { return parts * sources * dz_part(); }
    __host__ __device__ uint32_t stage() const { return (x_at() + parts * x_part() + 1023) / 1024 * 1024; }
    __host__ __device__ uint32_t copies() const { return stages * stage() + 2 * kBlockBytes; }
    __host__ __device__ int each() const { return ((rows + bn) * 16 + kProducers - 1) / kProducers; }      // vectors of a thread
    __host__ __device__ uint32_t barriers() const { return copies() + slots * each() * 16 * kProducers; }
    __host__ __device__ uint32_t bytes() const { return barriers() + (2 * stages + 4) * 8 + 8 + 1024; }
};

template <typename T, bool LAST, bool VEC>
__global__ void __launch_bounds__(kWeightThreads, 1) pointwise_weight_split_kernel(const WeightSplit q)
{
    constexpr int PARTS = kParts<T>;
    extern __shared__ char raw_smem[];
    __shared__ float sums_smem[kGroups][128];
    const uint32_t raw = smem_u32(raw_smem), base = (raw + 1023) & ~1023u;
    char *smem = raw_smem + (base - raw);
    const int sources = PARTS == 1 && q.rest ? 2 : 1;
    const WeightSplitLayout lay{q.rows, q.bn, q.stages, q.slots, PARTS, sources, LAST};
    const uint32_t full = base + lay.barriers(), empty = full + 8 * q.stages, ready = empty + 8 * q.stages, drained = ready + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + lay.barriers() + (2 * q.stages + 4) * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_o = (q.Co + q.rows - 1) / q.rows, tiles = tiles_o * q.tiles_i;
    const int split = (int)(blockIdx.x / (unsigned)tiles), t = (int)blockIdx.x - split * tiles;
    const int o0 = t / q.tiles_i * q.rows, i0 = (t - t / q.tiles_i * q.tiles_i) * q.bn;
    const int first = split * q.per, last = min(q.samples * q.slices, first + q.per);      // (all of them below 2^30)
    const bool sums = q.sums && i0 == 0;
    const uint32_t columns = (PARTS > 1 ? 2 : 1) * q.columns;
    const T *dz_all = static_cast<const T *>(q.dz), *x_all = static_cast<const T *>(q.x);

    if (threadIdx.x == 0) {
        for (int i = 0; i < q.stages; ++i) {
            mbar_init(full + 8 * i, PARTS == 3 ? kGroups * kGroupWarps : kGroupWarps);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(ready + 8 * i, 1);
            mbar_init(drained + 8 * i, kWeightEpilogue);
        }
        fence_mbar_init();
    }
    grid_dependency_wait();
    if (warp == kWeightEpilogue + kGroups * kGroupWarps) tmem_alloc(tmem_slot, q.sums_at.all);
    tmem_release();
    __syncthreads();
    tmem_acquire();
    const uint32_t tmem = *tmem_slot;
    Waiter wait;

    if (PARTS == 3 && warp >= kWeightEpilogue && warp < kWeightEpilogue + kGroups * kGroupWarps) {
        // as in the product's kernel: a thread's own vectors of four, copied `slots` slices ahead, eight of them at a time
        const int t = threadIdx.x - 32 * kWeightEpilogue;
        const int of_dz = q.rows * 16, total = of_dz + q.bn * 16;
        const uint32_t slot_bytes = lay.each() * 16 * kProducers;
        const char *own = smem + lay.copies() + 16 * t;
        // vector e of an operand of `wide` vectors a row: planes, four pixels of a channel; last, four channels of a pixel
        struct Spot {
            bool dz;
            int outer, in;
        };
        auto spot = [&](int e) {
            Spot v;
            v.dz = e < of_dz;
            const int f = v.dz ? e : e - of_dz, wide = LAST ? (v.dz ? q.rows : q.bn) / 4 : 16;
            v.outer = LAST ? (int)((unsigned)f / (unsigned)wide) : f >> 4;
            v.in = 4 * (LAST ? f - v.outer * wide : f & 15);
            return v;
        };
        auto copy = [&](int slice) {
            if (slice < last) {
                const int64_t sample = (unsigned)slice / (unsigned)q.slices, p0 = (slice - sample * q.slices) * 64;
                const int pixels = (int)min((int64_t)64, q.P - p0);
                const uint32_t to = smem_u32(own) + (q.slots > 1 ? (uint32_t)(slice - first & 1) * slot_bytes : 0);
                for (int j = 0, e = t; e < total; ++j, e += kProducers) {
                    const Spot v = spot(e);
                    const int C = v.dz ? q.Co : q.Ci, c = (v.dz ? o0 : i0) + (LAST ? v.in : v.outer), p = LAST ? v.outer : v.in;
                    const float *from = reinterpret_cast<const float *>(v.dz ? q.dz : q.x);
                    copy4<VEC>(to + 4096 * j, from + (LAST ? (p0 + p) * C + c : (sample * C + c) * q.P + p0 + p),
                               LAST ? (p < pixels ? C - c : 0) : (c < C ? pixels - p : 0), reinterpret_cast<const float *>(q.dz));
                }
            }
            copies_commit();
        };
        for (int i = 0; i < q.slots; ++i) copy(first + i);
        float sum[8] = {};      // planes: of the channel of vector t + 256 j; last: of the four channels of every vector of dz
        uint32_t stage = 0, phase = 0;
        for (int slice = first; slice < last; ++slice) {
            copies_wait(q.slots);
            if (__any_sync(0xffffffffu, !wait(empty + 8 * stage, phase ^ 1))) break;
            char *const dz_to = smem + stage * lay.stage(), *const x_to = dz_to + lay.x_at();
            const char *from = own + (q.slots > 1 ? (uint32_t)(slice - first & 1) * slot_bytes : 0);
            float here[4] = {};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float4 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (t + kProducers * (8 * half + j) < total) v[j] = *reinterpret_cast<const float4 *>(from + 4096 * (8 * half + j));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = t + kProducers * (8 * half + j);
                    if (e >= total) break;
                    const Spot w = spot(e);
                    char *to = (w.dz ? dz_to : x_to) + (LAST ? (w.in >> 6) * kBlockBytes : 0) + w.outer * 128 + ((((w.in >> 3) & 7) ^ (w.outer & 7)) << 4) +
                               (w.in & 4) * 2;
                    place4(to, w.dz ? lay.dz_part() : lay.x_part(), v[j]);
                    if (half == 0 && sums && w.dz) {      // (dz has 2048 vectors at most)
                        if (LAST) {      // (a slice's by itself first: fewer additions to a long sum)
                            here[0] += v[j].x;
                            here[1] += v[j].y;
                            here[2] += v[j].z;
                            here[3] += v[j].w;
                        } else {
                            sum[j] += (v[j].x + v[j].y) + (v[j].z + v[j].w);
                        }
                    }
                }
            }
            if (LAST)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] += here[i];
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * stage);
            copy(slice + q.slots);
            if (++stage == (uint32_t)q.stages) {
                stage = 0;
                phase ^= 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (sums) {
            // (rows are a power of two: a thread's vectors of dz are all at one place among the channels, or eight lanes' of a channel)
            if (LAST) {
                const int wide = q.rows / 4, place = t % wide;
                for (int turn = 0; turn < kProducers / wide; ++turn) {
                    if (t / wide == turn)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sums_smem[0][4 * place + i] = turn ? sums_smem[0][4 * place + i] + sum[i] : sum[i];
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float g = sum[j];
                    g += __shfl_xor_sync(0xffffffffu, g, 1);
                    g += __shfl_xor_sync(0xffffffffu, g, 2);
                    g += __shfl_xor_sync(0xffffffffu, g, 4);
                    g += __shfl_xor_sync(0xffffffffu, g, 8);
                    const int c = (t + kProducers * j) >> 4;
                    if ((lane & 15) == 0 && c < q.rows) sums_smem[0][c] = g;
                }
            }
        }
    } else if (warp >= kWeightEpilogue && warp < kWeightEpilogue + kGroups * kGroupWarps) {
        const int group = (warp - kWeightEpilogue) / kGroupWarps, me = threadIdx.x - 32 * (kWeightEpilogue + group * kGroupWarps);
        const int of_source = q.rows * 8, of_dz = sources * of_source, total = of_dz + q.bn * 8;      // vectors of a slice
        // planes: of the channel of vector me + 128 j of a source; last: of the channels of every vector of dz.  Of kSumSlices, of all.
        float sum[8] = {}, total_of[8] = {};
        for (int slice = first + group; slice < last; slice += kGroups) {
            const unsigned nth = slice - first, stage = nth % (unsigned)q.stages, phase = nth / (unsigned)q.stages & 1;
            const int64_t sample = (unsigned)slice / (unsigned)q.slices, p0 = (slice - sample * q.slices) * 64;
            const int pixels = (int)min((int64_t)64, q.P - p0);
            char *const dz_to = smem + stage * lay.stage(), *const x_to = dz_to + lay.x_at();
            bool waited = false;
            for (int v0 = me; v0 < total; v0 += 8 * 128) {
                uint4 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = v0 + 128 * j;
                    if (e >= total) break;
                    const bool dz = e < of_dz, more = dz && e >= of_source;
                    const int f = dz ? more ? e - of_source : e : e - of_dz, C = dz ? q.Co : q.Ci, c0 = dz ? o0 : i0, wide = (dz ? q.rows : q.bn) / 8;
                    const T *from = dz ? more ? static_cast<const T *>(q.rest) : dz_all : x_all;
                    if (LAST) {      // eight channels of a pixel
                        const int p = (unsigned)f / (unsigned)wide, c = c0 + 8 * (f - p * wide);
                        if constexpr (PARTS == 1) v[j] = load8<T, VEC>(from + (p0 + p) * C + c, p < pixels ? C - c : 0);
                    } else {         // eight pixels of a channel
                        const int c = c0 + (f >> 3), p = 8 * (f & 7);
                        if constexpr (PARTS == 1) v[j] = load8<T, VEC>(from + (sample * C + c) * q.P + p0 + p, c < C ? pixels - p : 0);
                    }
                }
                if (!waited) {
                    waited = true;
                    wait(empty + 8 * stage, phase ^ 1);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = v0 + 128 * j;
                    if (e >= total) break;
                    const bool dz = e < of_dz, more = dz && e >= of_source;
                    const int f = dz ? more ? e - of_source : e : e - of_dz, wide = (dz ? q.rows : q.bn) / 8;
                    const int outer = LAST ? (unsigned)f / (unsigned)wide : f >> 3, chunk = LAST ? f - outer * wide : f & 7;
                    char *to = (dz ? more ? dz_to + lay.dz_part() : dz_to : x_to) + (LAST ? (chunk >> 3) * kBlockBytes : 0) + outer * 128 + (((chunk & 7) ^ (outer & 7)) << 4);
                    *reinterpret_cast<uint4 *>(to) = v[j];
                    if (sums && dz) {
                        float g[8] = {};
                        if constexpr (PARTS == 1) unpack<T>(v[j], g);
                        if (LAST) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) sum[i] += g[i];
                        } else {
                            sum[j] += ((g[0] + g[1]) + (g[2] + g[3])) + ((g[4] + g[5]) + (g[6] + g[7]));
                        }
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * stage);
            if (sums && (nth % kSumSlices<T> >= kSumSlices<T> - kGroups || slice + kGroups >= last))
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    total_of[j] += sum[j];
                    sum[j] = 0.f;
                }
        }
        if (sums) {
            // (rows are a power of two: a thread's vectors of dz are all at one place among the channels, or eight lanes' of a channel)
            if (LAST) {
                // the threads of a place, in order, one at a time
                const int wide = q.rows / 8, place = me % wide;
                for (int turn = 0; turn < 128 / wide; ++turn) {
                    if (me / wide == turn)
#pragma unroll
                        for (int i = 0; i < 8; ++i) sums_smem[group][8 * place + i] = turn ? sums_smem[group][8 * place + i] + total_of[i] : total_of[i];
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
                }
            } else {
                // (rows of less than 128: the second source's vectors come as later j)
                if (sources == 2)
#pragma unroll
                    for (int j = 1; j < 8; j *= 2)
                        if (16 * j == q.rows)
#pragma unroll
                            for (int i = 0; i < j; ++i) total_of[i] += total_of[j + i];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float g = total_of[j];
                    g += __shfl_xor_sync(0xffffffffu, g, 1);
                    g += __shfl_xor_sync(0xffffffffu, g, 2);
                    g += __shfl_xor_sync(0xffffffffu, g, 4);
                    const int c = (me + 128 * j) >> 3;
                    if ((lane & 7) == 0 && c < q.rows) sums_smem[group][c] = g;
                }
            }
        }
    } else if (warp == kWeightEpilogue + kGroups * kGroupWarps) {
        if (lane == 0) {
            constexpr uint32_t step = LAST ? 128 : 2;      // bytes from k to k
            const uint64_t dz = LAST ? mn_major(base, 0, kBlockBytes) : k_major(base, 0), x = further(dz, lay.x_at());
            const uint32_t a_high = (uint32_t)(dz >> 32), b_high = (uint32_t)(x >> 32);
            uint32_t a[PARTS], b[PARTS];
            for (int i = 0; i < PARTS; ++i) {
                a[i] = (uint32_t)further(dz, i * lay.dz_part());
                b[i] = (uint32_t)further(x, i * lay.x_part());
            }
            uint32_t stage = 0, phase = 0, set = 0, set_phase = 0;
            int begin = first, end;      // a sum's slices
            do {
                end = min(last, begin + kSumSlices<T>);
                if (!wait(drained + 8 * set, set_phase ^ 1)) break;
                tmem_acquire();
                const uint32_t d = tmem + set * columns;
                for (int slice = begin; slice < end; ++slice) {
                    if (!wait(full + 8 * stage, phase)) break;
                    tmem_acquire();
                    const uint32_t at = stage * lay.stage() >> 4;
#pragma unroll
                    for (int k = 0; k < 64; k += 16) {
#pragma unroll
                        for (int i = 0; i < PARTS; ++i)
#pragma unroll
                            for (int j = 0; j < PARTS - i; ++j)
                                mma(i + j ? d + q.columns : d, a[i] + at + (step * k >> 4), a_high, b[j] + at + (step * k >> 4), b_high,
                                    q.instruction, slice > begin || k || i + j > 1 || i > 0);
                        if (PARTS == 1 && sources == 2)
                            mma(d, a[0] + at + (lay.dz_part() + step * k >> 4), a_high, b[0] + at + (step * k >> 4), b_high, q.instruction, true);
                    }
                    mma_commit(empty + 8 * stage);
                    if (++stage == (uint32_t)q.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (wait.lost) break;
                mma_commit(ready + 8 * set);
                if (++set == (uint32_t)q.sums_at.sets) {
                    set = 0;
                    set_phase ^= 1;
                }
            } while ((begin = end) < last);
        }
    } else {
        float *partial = q.partial + split * pointwise_partial_stride(q.Co, q.Ci);
        const int row = warp * 32 + lane, o = o0 + row;
        const bool mine = row < q.rows && o < q.Co;
        uint32_t set = 0, set_phase = 0;
        auto arrived = [&] {
            wait(ready + 8 * set, set_phase);
            __syncwarp();
            tmem_acquire();
        };
        auto sum16 = [&](int b, bool begun, float (&v)[16]) {
            const uint32_t at = tmem + b + ((uint32_t)warp << 21);
            accumulators16(at + set * columns, v);
            if (PARTS == 3) add16(at + set * columns + q.columns, v);
            if (begun) add16(at + q.sums_at.sets * columns, v);
        };
        int begin = first;
#pragma unroll 1
        for (; last - begin > kSumSlices<T>; begin += kSumSlices<T>) {
            arrived();
#pragma unroll 1
            for (int b = 0; b < q.bn; b += 16) {
                float v[16];
                sum16(b, begin > first, v);
                store16(tmem + q.sums_at.sets * columns + b + ((uint32_t)warp << 21), v);
            }
            tmem_wait_store();
            tmem_release();
            __syncwarp();
            if (lane == 0) mbar_arrive(drained + 8 * set);
            if (++set == (uint32_t)q.sums_at.sets) {
                set = 0;
                set_phase ^= 1;
            }
        }
        arrived();
        for (int b = 0; b < q.bn; b += 16) {
            float v[16];
            sum16(b, begin > first, v);
            if constexpr (PARTS == 3) {
                float u[16], finite = 0.f;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (i0 + b + j < q.Ci) finite = fmaf(v[j], 0.f, finite);
                if (finite != 0.f && mine) {      // (a NaN: some value is not finite)
#pragma unroll
                    for (int j = 0; j < 16; ++j) u[j] = 0.f;
                    for (int slice = first; slice < last; ++slice) {
                        const int64_t sample = (unsigned)slice / (unsigned)q.slices, p0 = (slice - sample * q.slices) * 64;
                        for (int64_t p = p0; p < min(p0 + 64, q.P); ++p) {
                            const float g = to_float(dz_all[LAST ? p * q.Co + o : (sample * q.Co + o) * q.P + p]);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const int c = i0 + b + j;
                                if (c < q.Ci) u[j] = fmaf(g, to_float(x_all[LAST ? p * q.Ci + c : (sample * q.Ci + c) * q.P + p]), u[j]);
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (!(fabsf(v[j]) < INFINITY)) v[j] = u[j];
                }
                __syncwarp();
            }
            if (mine)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (i0 + b + j < q.Ci) partial[(int64_t)o * q.Ci + i0 + b + j] = v[j];
        }
    }
    if (wait.lost) let_copies_land();
    __syncwarp();
    tmem_release();
    __syncthreads();
    if (warp == kWeightEpilogue + kGroups * kGroupWarps) tmem_free(tmem, q.sums_at.all);
    if (sums && (int)threadIdx.x < q.rows && o0 + (int)threadIdx.x < q.Co)
        q.partial[split * pointwise_partial_stride(q.Co, q.Ci) + (int64_t)q.Co * q.Ci + o0 + threadIdx.x] =
            PARTS == 1 && last - first > 1 ? sums_smem[0][threadIdx.x] + sums_smem[1][threadIdx.x] : sums_smem[0][threadIdx.x];
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct SplitPlan {
    int bn, tiles_n, stages, columns;
    bool merged;
    int64_t tiles_p;
    unsigned walkers;
    uint32_t smem;
};
bool plan_split(const PointwiseShape &s, int K, int Cn, SplitPlan *plan)
{
    const int parts = s.io_kind == BC_IO_F32 ? 3 : 1, chunks = (int)ceil_div(K, 64), samples = s.last ? 1 : s.N;
    const int64_t P = s.last ? s.N * s.P : s.P;
    if (K < 1 || Cn < 1) return false;
    SplitPlan r{};
    r.stages = parts == 3 ? 2 : 4;
    // channels of a tile: what shared memory holds of the weights, and tensor memory of the sums
    const uint32_t others = SplitLayout{16, r.stages, 0, parts, s.last}.bytes() + 8192;
    const int64_t most = std::min<int64_t>(parts == 3 ? 128 : 256, (int64_t)(kMostShared - others) / (parts * chunks * 128) / 16 * 16);
    // (every tile splits the operand again.  f32, 16 samples of 64 x 128 pixels, forward: 400 -> 400 channels in tiles of 32 641 us, by
    // multiply-adds 1168; 512 -> 512, where tiles would be of 16, by multiply-adds 1675)
    if (most < 32 && Cn > most) return false;
    if (most < 16) return false;
    r.tiles_n = (int)ceil_div(Cn, most);
    r.bn = (int)ceil_div(ceil_div(Cn, r.tiles_n), 16) * 16;
    r.tiles_n = (int)ceil_div(Cn, r.bn);
    r.merged = parts == 3 && 3 * r.bn <= 256;
    r.columns = 32;
    while (r.columns < (r.merged ? 3 : 1) * r.bn) r.columns *= 2;
    r.smem = SplitLayout{r.bn, r.stages, chunks, parts, s.last}.bytes();
    r.tiles_p = ceil_div(P, 128);
    const int64_t tiles = r.tiles_p * samples;
    if (r.smem > kMostShared || tiles > INT32_MAX) return false;
    r.walkers = (unsigned)std::min<int64_t>(tiles, std::max<int64_t>(1, 148 / r.tiles_n));
    *plan = r;
    return true;
}

template <int MODE>
int launch_split(const PointwiseShape &s, const SplitPlan &plan, SplitProduct q, cudaStream_t stream)
{
    q.samples = s.last ? 1 : s.N;
    q.P = s.last ? s.N * s.P : s.P;
    q.tiles_p = (int)plan.tiles_p;
    q.tiles_n = plan.tiles_n;
    q.bn = plan.bn;
    q.stages = plan.stages;
    q.columns = plan.columns;
    q.merged = plan.merged;
    q.instruction = mma_instruction(s.io_kind != BC_IO_F16, !s.last, false, (plan.merged ? 3 : 1) * plan.bn);
    const int each = 16 / io_size(s.io_kind);
    const bool vec = (s.last ? q.K : q.P) % each == 0 && pointwise_mma_aligned(q.a, nullptr);
    return with_type(s.io_kind, [&](auto t) {
        return with_activation(MODE == INPUT ? BC_ACT_NONE : s.act, [&](auto act) {
            using T = decltype(t);
            constexpr int ACT = MODE == INPUT ? BC_ACT_NONE : act();
            auto go = [&](auto kernel) {
                if (const int e = raise_smem_limit((const void *)kernel, kMostShared)) return e;
                const LaunchScope scope(KID_POINTWISE_SPLIT, stream);
                launch_overlapped(kernel, plan.walkers * plan.tiles_n, kThreads, plan.smem, stream, q);
                return check_launch("pointwise_split_kernel");
            };
            if (s.last) return vec ? go(pointwise_split_kernel<T, MODE, ACT, true, true>) : go(pointwise_split_kernel<T, MODE, ACT, true, false>);
            return vec ? go(pointwise_split_kernel<T, MODE, ACT, false, true>) : go(pointwise_split_kernel<T, MODE, ACT, false, false>);
        });
    });
}

}  // namespace

bool pointwise_split_suits(const PointwiseShape &s, bool input)
{
    SplitPlan plan;
    return plan_split(s, input ? s.Co : s.Ci, input ? s.Ci : s.Co, &plan);
}
int pointwise_split_sums_rows(const PointwiseShape &s)
{
    SplitPlan plan;
    return plan_split(s, s.Ci, s.Co, &plan) ? (int)plan.walkers : 0;
}
int launch_pointwise_split_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                                   void *out, cudaStream_t stream)
{
    SplitPlan plan;
    plan_split(s, s.Ci, s.Co, &plan);
    return launch_split<FORWARD>(s, plan, {x, weight, bias, residual, nullptr, out, nullptr, nullptr, 0, s.Ci, s.Co, 0, s.Ci, 1}, stream);
}
int launch_pointwise_split_slope(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                                 const void *grad, void *dz, void *rest, float *sums, cudaStream_t stream)
{
    SplitPlan plan;
    plan_split(s, s.Ci, s.Co, &plan);
    return launch_split<SLOPE>(s, plan, {x, weight, bias, residual, grad, dz, rest, sums, 0, s.Ci, s.Co, 0, s.Ci, 1}, stream);
}
int launch_pointwise_split_input(const PointwiseShape &s, const void *dz, const void *rest, const void *weight, void *grad_input,
                                 cudaStream_t stream)
{
    SplitPlan plan;
    plan_split(s, s.Co, s.Ci, &plan);
    return launch_split<INPUT>(s, plan, {dz, weight, nullptr, nullptr, nullptr, grad_input, const_cast<void *>(rest), nullptr, 0, s.Co, s.Ci, 0, 1, s.Ci}, stream);
}

// ---- grad_weight: rows of pointwise_partial_stride() floats, to be added
namespace {
struct WeightSplitPlan {
    int rows, tiles_o, tiles_i, bn, stages, slots, columns, splits;
    int64_t slices, per;
    uint32_t smem;
};
bool plan_weight_split(const PointwiseShape &s, int sources, WeightSplitPlan *plan)
{
    const int parts = s.io_kind == BC_IO_F32 ? 3 : 1, Ci = std::max(1, s.Ci);      // (no input channels: the sums of dz alone)
    const int64_t P = s.last ? s.N * s.P : s.P, samples = s.last ? 1 : s.N;
    WeightSplitPlan r{};
    r.rows = 16;
    while (r.rows < s.Co && r.rows < 128) r.rows *= 2;
    r.tiles_o = (int)ceil_div(s.Co, r.rows);
    // the widest tile that shared memory holds: 16-bit with a ring of two to four, float with two and one or two slices of copies
    for (int most = parts == 3 ? 128 : 256;; most /= 2) {
        if (most < 32) return false;
        r.tiles_i = (int)ceil_div(Ci, most);
        r.bn = (int)ceil_div(ceil_div(Ci, r.tiles_i), 16) * 16;
        r.tiles_i = (int)ceil_div(Ci, r.bn);
        auto fits = [&](int stages, int slots) {
            r.stages = stages;
            r.slots = slots;
            r.smem = WeightSplitLayout{r.rows, r.bn, stages, slots, parts, sources, s.last}.bytes();
            return r.smem <= kMostShared - 2048;
        };
        if (parts == 3 ? fits(2, 2) || fits(2, 1) : fits(4, 0) || fits(3, 0) || fits(2, 0)) break;
    }
    r.columns = 32;
    while (r.columns < r.bn) r.columns *= 2;
    r.slices = ceil_div(P, 64);
    const int64_t all = r.slices * samples, tiles = (int64_t)r.tiles_o * r.tiles_i;
    r.per = slices_of_split(all, tiles, parts == 3 ? kSumSlices<float> * kMostSums<float> : kSumSlices<__half> * kMostSums<__half>);
    r.splits = (int)ceil_div(all, r.per);
    if (all >= 1 << 30 || r.splits * tiles > INT32_MAX) return false;
    *plan = r;
    return true;
}
}  // namespace

int pointwise_split_weight_splits(const PointwiseShape &s, bool rest)
{
    WeightSplitPlan plan;
    return plan_weight_split(s, rest ? 2 : 1, &plan) ? plan.splits : 0;
}
int launch_pointwise_split_weight(const PointwiseShape &s, const void *dz, const void *rest, const void *x, float *partial, bool sums,
                                  cudaStream_t stream)
{
    WeightSplitPlan plan;
    plan_weight_split(s, rest ? 2 : 1, &plan);
    WeightSplit q{};
    q.dz = dz;
    q.rest = rest;
    q.x = x;
    q.partial = partial;
    q.P = s.last ? s.N * s.P : s.P;
    q.per = (int)plan.per;
    q.slices = (int)plan.slices;
    q.samples = s.last ? 1 : s.N;
    q.Ci = s.Ci;
    q.Co = s.Co;
    q.tiles_i = plan.tiles_i;
    q.rows = plan.rows;
    q.bn = plan.bn;
    q.stages = plan.stages;
    q.slots = plan.slots;
    q.columns = plan.columns;
    q.sums_at = s.io_kind == BC_IO_F32 ? sum_columns(plan.per > kSumSlices<float>, 2 * plan.columns, plan.bn)
                                       : sum_columns(plan.per > kSumSlices<__half>, plan.columns, plan.bn);
    q.sums = sums;
    q.instruction = mma_instruction(s.io_kind != BC_IO_F16, s.last, s.last, plan.bn);
    const int each = 16 / io_size(s.io_kind);
    const bool vec = (s.last ? s.Ci % each == 0 && s.Co % each == 0 : s.P % each == 0) && pointwise_mma_aligned(dz, x);
    return with_type(s.io_kind, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            if (const int e = raise_smem_limit((const void *)kernel, kMostShared - 2048)) return e;
            const LaunchScope scope(KID_POINTWISE_WEIGHT_SPLIT, stream);
            launch_overlapped(kernel, (unsigned)(plan.splits * plan.tiles_o * plan.tiles_i), kWeightThreads, plan.smem, stream, q);
            return check_launch("pointwise_weight_split_kernel");
        };
        if (s.last) return vec ? go(pointwise_weight_split_kernel<T, true, true>) : go(pointwise_weight_split_kernel<T, true, false>);
        return vec ? go(pointwise_weight_split_kernel<T, false, true>) : go(pointwise_weight_split_kernel<T, false, false>);
    });
}

int read_wait_timeouts_split(int *count) { return read_wait_timeouts_here(count); }

}  // namespace bc
