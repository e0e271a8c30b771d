// Pointwise convolutions of 16-bit tensors on the tensor cores: the products of pointwise.cu where rows start on 16 bytes.
//
// pointwise_mma_kernel, the products with pixels in the rows: D[p, c] = sum_k A[p, k] B[c, k], tiles of 128 pixels x up to 256
// channels.  The weights stay in shared memory; persistent CTAs walk over the pixels.  One thread brings slices of 64 k by
// TMA into a ring, one issues tcgen05.mma into one of two sets of accumulators in tensor memory, eight warps take the other set
// out.  Planes are an MN-major operand and channels last a K-major one: no transposition in either.
// A warp of the epilogue passes 32 x 32 sums through shared memory, so that it reads
// residuals and gradients and writes results 16 bytes a lane, 64 bytes in a row, along whichever index runs in memory.  Where a
// CTA has its SM to itself, the next block's are on their way while a block is dealt with.
//
// Measured on B200, (64,256->256,64,128) bf16 last: grad_input 97 us, 5.4 TB/s or 0.83 of the copy bandwidth, and 151 where dz is two
// tensors (5.3); forward with residual and GELU 182, slope that stores two tensors 291.  Those two wait for memory and shared memory with a
// CTA an SM: 0.41 and 0.47 instructions a cycle and scheduler, 1.5 and 1.4 times what their bytes take.
//
// pointwise_weight_mma_kernel: grad_weight, D[o, i] = sum_p dz[o, p] x[i, p], 128 x up to 256 weights, split over the pixels; 94 us there, 129
// of two tensors.
#include "bc_mma.cuh"

namespace bc {

namespace {

enum { FORWARD, SLOPE, INPUT };
constexpr int kEpilogue = 8;      // warps of the epilogue, or pairs of them
constexpr int kPitch = 33, kPitchLast = 36;      // words: columns, or vectors of rows, without bank conflicts
constexpr uint32_t kStage = 16384;      // 128 pixels x 64 k
constexpr size_t kMostShared = 227 << 10;

struct MmaProduct {
    CUtensorMap a, a_rest, w;      // INPUT: dz is the sum of two tensors
    const void *bias, *residual, *grad;
    void *out, *rest;        // rest: SLOPE, what the rounding of dz leaves, or null
    float *sums;             // SLOPE: [CTA / tiles_n][Cn] sums of dz over the CTA's pixels, or null
    int64_t P;               // pixels of a sample (of all of them together, channels last)
    int K, Cn, samples;
    int tiles_p, tiles_n;
    int bn, stages, columns; // channels of a tile; slices in the ring; columns of tensor memory for one set
    int parts;               // tensors that A is the sum of
    uint32_t instruction;
};

// Shared memory from a 1024-byte boundary on.
struct MmaLayout {
    int bn, stages, chunks, pair;
    bool input;
    // of one slice of 64 k of the weights
    __host__ __device__ uint32_t slice() const { return input ? (uint32_t)((bn + 63) / 64) * kBlockBytes : (uint32_t)bn * 128; }
    __host__ __device__ uint32_t ring() const { return (chunks * slice() + 1023) / 1024 * 1024; }
    __host__ __device__ uint32_t staging() const { return ring() + stages * kStage; }
    __host__ __device__ uint32_t bias() const { return staging() + kEpilogue * 32 * kPitchLast * 4; }
    __host__ __device__ uint32_t sums() const { return bias() + bn * 4; }
    __host__ __device__ uint32_t barriers() const { return (sums() + 4 * pair * bn * 4 + 7) / 8 * 8; }
    __host__ __device__ uint32_t bytes() const { return barriers() + (2 * stages + 5) * 8 + 8 + 1024; }
};

template <typename T, int MODE, int ACT, bool LAST, int PAIR>
__global__ void __launch_bounds__(32 * (kEpilogue * PAIR + 2), PAIR == 1 ? 2 : 1) pointwise_mma_kernel(const __grid_constant__ MmaProduct q)
{
    constexpr int WARPS = kEpilogue * PAIR, THREADS = 32 * (WARPS + 2), EACH = 4 / PAIR;
    extern __shared__ char raw_smem[];
    const uint32_t raw = smem_u32(raw_smem), base = (raw + 1023) & ~1023u;
    char *smem = raw_smem + (base - raw);
    const int chunks = (q.K + 63) / 64, parts = MODE == INPUT ? q.parts : 1;
    const MmaLayout lay{q.bn, q.stages, chunks, PAIR, MODE == INPUT};
    float *bias_smem = reinterpret_cast<float *>(smem + lay.bias()), *sums_smem = reinterpret_cast<float *>(smem + lay.sums());
    const uint32_t full = base + lay.barriers(), empty = full + 8 * q.stages, ready = empty + 8 * q.stages, drained = ready + 16,
                   weights_full = drained + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + lay.barriers() + (2 * q.stages + 5) * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned walkers = gridDim.x / (unsigned)q.tiles_n, walker = blockIdx.x / (unsigned)q.tiles_n;
    const int n0 = (int)(blockIdx.x - walker * q.tiles_n) * q.bn;
    const unsigned tiles = (unsigned)q.samples * (unsigned)q.tiles_p;      // (below 2^31)

    if (threadIdx.x == 0) {
        for (int i = 0; i < q.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(ready + 8 * i, 1);
            mbar_init(drained + 8 * i, WARPS);
        }
        mbar_init(weights_full, 1);
        fence_mbar_init();
        map_prefetch(&q.a);
        map_prefetch(&q.w);
    }
    grid_dependency_wait();
    if (warp == WARPS + 1) tmem_alloc(tmem_slot, 2 * q.columns);
    for (int i = threadIdx.x; i < q.bn; i += THREADS)
        bias_smem[i] = MODE != INPUT && q.bias && n0 + i < q.Cn ? to_float(static_cast<const T *>(q.bias)[n0 + i]) : 0.f;
    for (int i = threadIdx.x; i < 4 * PAIR * q.bn; i += THREADS) sums_smem[i] = 0.f;
    tmem_release();
    __syncthreads();
    tmem_acquire();
    const uint32_t tmem = *tmem_slot;
    Waiter wait;

    if (warp == WARPS) {
        if (lane == 0) {
            mbar_expect(weights_full, chunks * lay.slice());
            for (int c = 0; c < chunks; ++c) {
                if (MODE == INPUT)
                    for (int b = 0; b < (q.bn + 63) / 64; ++b)
                        tile_load(base + c * lay.slice() + b * kBlockBytes, &q.w, n0 + 64 * b, 64 * c, weights_full);
                else tile_load(base + c * lay.slice(), &q.w, 64 * c, n0, weights_full);
            }
            uint32_t stage = 0, phase = 0;
            for (unsigned tile = walker; tile < tiles; tile += walkers) {
                const unsigned sample = tile / (unsigned)q.tiles_p;
                const int64_t p0 = (int64_t)(tile - sample * q.tiles_p) * 128;
                for (int i = 0; i < parts * chunks; ++i) {      // (the parts of a slice in turn)
                    const int c = MODE == INPUT && parts == 2 ? i >> 1 : i;
                    const CUtensorMap *a = MODE == INPUT && parts == 2 && (i & 1) ? &q.a_rest : &q.a;
                    if (!wait(empty + 8 * stage, phase ^ 1)) break;
                    const uint32_t to = base + lay.ring() + stage * kStage, bar = full + 8 * stage;
                    mbar_expect(bar, kStage);
                    if (LAST) {
                        tile_load(to, a, 64 * c, (int)p0, bar);
                    } else {
                        tile_load(to, a, (int)p0, 64 * c, sample, bar);
                        tile_load(to + kBlockBytes, a, (int)p0 + 64, 64 * c, sample, bar);
                    }
                    if (++stage == (uint32_t)q.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (wait.lost) break;
            }
        }
    } else if (warp == WARPS + 1) {
        if (lane == 0) {
            wait(weights_full, 0);
            const uint64_t ring = LAST ? k_major(base + lay.ring(), 0) : mn_major(base + lay.ring(), 0, kBlockBytes);
            const uint64_t weights = MODE == INPUT ? mn_major(base, 0, kBlockBytes) : k_major(base, 0);
            uint32_t stage = 0, phase = 0, set = 0, set_phase = 0;
            for (unsigned tile = walker; tile < tiles; tile += walkers) {
                if (!wait(drained + 8 * set, set_phase ^ 1)) break;
                tmem_acquire();
                for (int i = 0; i < parts * chunks; ++i) {
                    if (!wait(full + 8 * stage, phase)) break;
                    tmem_acquire();
                    const int c = MODE == INPUT && parts == 2 ? i >> 1 : i;
                    const uint64_t a = further(ring, stage * kStage), w = further(weights, c * lay.slice());
                    const int k_used = q.K - 64 * c;
#pragma unroll
                    for (int k = 0; k < 64; k += 16)
                        if (k < k_used)
                            mma(tmem + set * q.columns, further(a, (LAST ? 2 : 128) * k), further(w, (MODE == INPUT ? 128 : 2) * k), q.instruction, i || k);
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
        const int quarter = warp & 3, member = PAIR == 2 ? warp >> 2 & 1 : 0, half = warp / (4 * PAIR), blocks = (q.bn + 31) / 32;
        float *staging = reinterpret_cast<float *>(smem + lay.staging()) + (4 * half + quarter) * 32 * kPitchLast;
        auto together = [&] {      // whoever shares the staging rows
            if (PAIR == 2) asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * half + quarter) : "memory");
            else __syncwarp();
        };
        // A lane's vectors of a block: planes, channel 8 i + outer and pixels from inner; last, that pixel and channels from
        // inner.  Every second block is a warp's, or two warps', two of the four vectors each.
        const int outer = (lane >> 2) + 8 * EACH * member, inner = 8 * (lane & 3);
        const T *residual = static_cast<const T *>(q.residual), *grad = static_cast<const T *>(q.grad);
        T *out = static_cast<T *>(q.out), *rest = static_cast<T *>(q.rest);
        struct Block {
            int64_t at;
            int there;                // bits
            uint4 res[MODE == INPUT ? 1 : EACH], grad[MODE == SLOPE ? EACH : 1];
        };
        uint32_t set = 0, set_phase = 0;
        for (unsigned tile = walker; tile < tiles; tile += walkers) {
            const unsigned sample = tile / (unsigned)q.tiles_p;
            const int64_t p0 = (int64_t)(tile - sample * q.tiles_p) * 128 + quarter * 32;
            auto fetch = [&](int b, Block &v) {
                const int64_t p = p0 + (LAST ? outer : inner);
                const int column = 32 * b + (LAST ? inner : outer), c = n0 + column;
                v.at = LAST ? p * q.Cn + c : ((int64_t)sample * q.Cn + c) * q.P + p;
                v.there = 0;
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    const bool there = LAST ? p + 8 * i < q.P && c < q.Cn && column < q.bn : p < q.P && c + 8 * i < q.Cn && column + 8 * i < q.bn;
                    const int64_t at = v.at + 8 * i * (LAST ? (int64_t)q.Cn : q.P);
                    v.there |= (int)there << i;
                    if (MODE != INPUT && residual && there) v.res[i] = *reinterpret_cast<const uint4 *>(residual + at);
                    if (MODE == SLOPE && there) v.grad[i] = *reinterpret_cast<const uint4 *>(grad + at);
                }
            };
            auto finish = [&](int b, const Block &now) {
#pragma unroll
                for (int part = member; part < 2; part += PAIR) {
                    float v[16];
                    accumulators16(tmem + set * q.columns + 32 * b + 16 * part + ((uint32_t)quarter << 21), v);
#pragma unroll
                    for (int j = 0; j < 16; j += LAST ? 4 : 1) {
                        if (LAST) *reinterpret_cast<float4 *>(staging + lane * kPitchLast + 16 * part + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        else staging[lane * kPitch + 16 * part + j] = v[j];
                    }
                }
                together();
                float total[8] = {};
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    const int row = 8 * i + outer;
                    const bool there = now.there >> i & 1;
                    f2_t z[4];
                    // four pairs, of a row or of a column
                    auto pairs = [](const float *from, int pitch, f2_t (&v)[4]) {
                        if (LAST) {
                            const ulonglong2 lo = *reinterpret_cast<const ulonglong2 *>(from), hi = *reinterpret_cast<const ulonglong2 *>(from + 4);
                            v[0] = lo.x;
                            v[1] = lo.y;
                            v[2] = hi.x;
                            v[3] = hi.y;
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[j] = pack2(from[2 * j * pitch], from[(2 * j + 1) * pitch]);
                        }
                    };
                    pairs(LAST ? staging + row * kPitchLast + inner : staging + inner * kPitch + row, kPitch, z);
                    if (MODE != INPUT && there) {
                        f2_t bias[4];
                        pairs(bias_smem + 32 * b + (LAST ? inner : row), 0, bias);
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = add2(z[j], bias[j]);
                        if (residual) {
                            f2_t r[4];
                            unpack_pairs<T>(now.res[i], r);
#pragma unroll
                            for (int j = 0; j < 4; ++j) z[j] = add2(z[j], r[j]);
                        }
                    }
                    if (MODE == SLOPE) {
                        f2_t g[4];
                        unpack_pairs<T>(there ? now.grad[i] : make_uint4(0, 0, 0, 0), g);
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = there ? times_slope2<ACT, T>(g[j], z[j]) : both(0.f);
                        if (q.sums) {
                            float s[8];
#pragma unroll
                            for (int j = 0; j < 4; ++j) unpack2(z[j], s[2 * j], s[2 * j + 1]);
                            if (LAST) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) total[j] += s[j];
                            } else {
                                float t = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
                                t += __shfl_xor_sync(0xffffffffu, t, 1);
                                t += __shfl_xor_sync(0xffffffffu, t, 2);
                                if ((lane & 3) == 0 && 32 * b + row < q.bn) sums_smem[(quarter + 4 * member) * q.bn + 32 * b + row] += t;
                            }
                        }
                    } else if (MODE == FORWARD) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = activate2<ACT, T>(z[j]);
                    }
                    if (there) {
                        const int64_t at = now.at + 8 * i * (LAST ? (int64_t)q.Cn : q.P);
                        const uint4 rounded = pack_pairs<T>(z);
                        *reinterpret_cast<uint4 *>(out + at) = rounded;
                        if (MODE == SLOPE && rest) *reinterpret_cast<uint4 *>(rest + at) = left_by_rounding<T>(z, rounded);
                    }
                }
                if (MODE == SLOPE && LAST && q.sums) {      // eight channels over the eight lanes of their vectors
                    fold(total, lane, 4, 4);
                    fold(total, lane, 8, 2);
                    fold(total, lane, 16, 1);
                    const int c = 32 * b + inner + (lane & 4 ? 4 : 0) + (lane & 8 ? 2 : 0) + (lane & 16 ? 1 : 0);
                    if (c < q.bn) sums_smem[(quarter + 4 * member) * q.bn + c] += total[0];
                }
                together();
            };
            Block one, two;
            fetch(half, one);
            wait(ready + 8 * set, set_phase);
            __syncwarp();
            tmem_acquire();
            for (int b = half; b < blocks; b += 4) {
                if (PAIR == 2) fetch(b + 2, two);
                finish(b, one);
                if (b + 2 >= blocks) break;
                if (PAIR == 2) fetch(b + 4, one);
                else fetch(b + 2, two);
                finish(b + 2, two);
                if (PAIR == 1 && b + 4 < blocks) fetch(b + 4, one);
            }
            tmem_release();
            __syncwarp();
            if (lane == 0) mbar_arrive(drained + 8 * set);
            if (set ^= 1; set == 0) set_phase ^= 1;
        }
    }
    if (wait.lost) let_copies_land();
    __syncwarp();
    tmem_release();
    __syncthreads();
    if (warp == WARPS + 1) tmem_free(tmem, 2 * q.columns);
    if (MODE == SLOPE && q.sums)
        for (int i = threadIdx.x; i < q.bn; i += THREADS)
            if (n0 + i < q.Cn) {
                float t = 0.f;
                for (int w = 0; w < 4 * PAIR; ++w) t += sums_smem[w * q.bn + i];
                q.sums[(int64_t)walker * q.Cn + n0 + i] = t;
            }
}

// ---- grad_weight

constexpr int kWeightThreads = 32 * 6, kMostStages = 8;

struct WeightMma {
    CUtensorMap dz, dz_rest, x;
    float *partial;          // a row a split: Co * Ci sums, then Co sums of dz
    int64_t per;             // slices of 64 pixels of a split
    int64_t slices;          // of a sample
    int samples, Ci, Co;
    int tiles_i;
    int bn, rows, stages, columns;      // input channels of a tile; rows of dz that are loaded (planes); ring; tensor memory of a set of sums
    SumColumns sums_at;
    bool sums;
    uint32_t instruction;
};

// Shared memory from a 1024-byte boundary on: slices of dz (128 channels of each part) and x (bn), then barriers.
struct WeightLayout {
    int bn, stages, parts;
    bool last;
    __host__ __device__ uint32_t x_bytes() const { return last ? (uint32_t)((bn + 63) / 64) * kBlockBytes : (uint32_t)bn * 128; }
    __host__ __device__ uint32_t x_at() const { return parts * 2 * kBlockBytes; }
    __host__ __device__ uint32_t stage() const { return x_at() + x_bytes(); }
    __host__ __device__ uint32_t barriers() const { return stages * stage(); }
    __host__ __device__ uint32_t bytes() const { return barriers() + (2 * stages + 4) * 8 + 8 + 1024; }
};

// Four warps of the epilogue also add up dz, from the slices as they pass, for grad_bias.  PARTS: tensors that dz is the sum of.
template <typename T, bool LAST, int PARTS>
__global__ void __launch_bounds__(kWeightThreads) pointwise_weight_mma_kernel(const __grid_constant__ WeightMma q)
{
    extern __shared__ char raw_smem[];
    __shared__ float part[128][9];
    const uint32_t raw = smem_u32(raw_smem), base = (raw + 1023) & ~1023u;
    char *smem = raw_smem + (base - raw);
    const WeightLayout lay{q.bn, q.stages, PARTS, LAST};
    const uint32_t full = base + lay.barriers(), empty = full + 8 * q.stages, ready = empty + 8 * q.stages, drained = ready + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + lay.barriers() + (2 * q.stages + 4) * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_o = (q.Co + 127) / 128, tiles = tiles_o * q.tiles_i;
    const int split = (int)(blockIdx.x / (unsigned)tiles), t = (int)blockIdx.x - split * tiles;
    const int o0 = t / q.tiles_i * 128, i0 = (t - t / q.tiles_i * q.tiles_i) * q.bn;
    const int64_t first = split * q.per, last = min((int64_t)q.samples * q.slices, first + q.per);
    const bool sums = q.sums && i0 == 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < q.stages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, sums ? 5 : 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(ready + 8 * i, 1);
            mbar_init(drained + 8 * i, 4);
        }
        fence_mbar_init();
        map_prefetch(&q.dz);
        map_prefetch(&q.x);
    }
    grid_dependency_wait();
    if (warp == 5) tmem_alloc(tmem_slot, q.sums_at.all);
    tmem_release();
    __syncthreads();
    tmem_acquire();
    const uint32_t tmem = *tmem_slot;
    Waiter wait;

    if (warp == 4) {
        if (lane == 0) {
            const int a_blocks = LAST ? (o0 + 64 < q.Co ? 2 : 1) : 0, b_blocks = (q.bn + 63) / 64;
            const uint32_t bytes = PARTS * (LAST ? a_blocks * kBlockBytes : (uint32_t)q.rows * 128) + lay.x_bytes();
            uint32_t stage = 0, phase = 0;
            for (int64_t slice = first; slice < last; ++slice) {
                if (!wait(empty + 8 * stage, phase ^ 1)) break;
                const int sample = (int)(slice / q.slices), p0 = (int)(slice - sample * q.slices) * 64;
                const uint32_t a = base + stage * lay.stage(), b = a + lay.x_at(), bar = full + 8 * stage;
                mbar_expect(bar, bytes);
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const CUtensorMap *dz = part ? &q.dz_rest : &q.dz;
                    const uint32_t to = a + part * 2 * kBlockBytes;
                    if (LAST)
                        for (int i = 0; i < a_blocks; ++i) tile_load(to + i * kBlockBytes, dz, o0 + 64 * i, p0, bar);
                    else tile_load(to, dz, p0, o0, sample, bar);
                }
                if (LAST)
                    for (int i = 0; i < b_blocks; ++i) tile_load(b + i * kBlockBytes, &q.x, i0 + 64 * i, p0, bar);
                else tile_load(b, &q.x, p0, i0, sample, bar);
                if (++stage == (uint32_t)q.stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 5) {
        if (lane == 0) {
            constexpr uint32_t step = LAST ? 128 : 2;      // bytes from k to k
            const uint64_t dz = LAST ? mn_major(base, 0, kBlockBytes) : k_major(base, 0), x = further(dz, lay.x_at());
            const uint32_t a_high = (uint32_t)(dz >> 32), b_high = (uint32_t)(x >> 32);
            uint32_t stage = 0, phase = 0, set = 0, set_phase = 0;
            int64_t begin = first, end;      // a sum's slices
            do {
                end = min(last, begin + kSumSlices<T>);
                if (!wait(drained + 8 * set, set_phase ^ 1)) break;
                const uint32_t d = tmem + set * q.columns;
                for (int64_t slice = begin; slice < end; ++slice) {
                    if (!wait(full + 8 * stage, phase)) break;
                    tmem_acquire();
                    const uint32_t at = stage * lay.stage() >> 4, a = (uint32_t)dz + at, b = (uint32_t)x + at;
#pragma unroll
                    for (int k = 0; k < 64; k += 16) {
                        mma(d, a + (step * k >> 4), a_high, b + (step * k >> 4), b_high, q.instruction, slice > begin || k);
                        if (PARTS == 2) mma(d, a + (2 * kBlockBytes + step * k >> 4), a_high, b + (step * k >> 4), b_high, q.instruction, true);
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
        const int o = o0 + warp * 32 + lane, group = threadIdx.x & 15, pixel = threadIdx.x >> 4;
        float total[8] = {};
        uint32_t stage = 0, phase = 0, set = 0, set_phase = 0;
        for (int64_t from = first; from < last; from += kSumSlices<T>) {
            // planes: a thread a channel, its 64 pixels.  last: a thread 8 channels of 8 pixels.
            float sum[8] = {};
            if (sums)
                for (int64_t slice = from; slice < min(last, from + kSumSlices<T>); ++slice) {
                    wait(full + 8 * stage, phase);
                    const char *a = smem + stage * lay.stage();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int k = 8 * j + pixel;
                        const char *at = LAST ? a + (group >> 3) * kBlockBytes + k * 128 + (((group & 7) ^ (k & 7)) << 4)
                                                : a + threadIdx.x * 128 + ((j ^ (threadIdx.x & 7)) << 4);
                        if (LAST ? o0 + 8 * group < q.Co : o0 + (int)threadIdx.x < q.Co)
#pragma unroll
                            for (int part = 0; part < PARTS; ++part) {
                                float v[8];
                                unpack<T>(*reinterpret_cast<const uint4 *>(at + part * 2 * kBlockBytes), v);
#pragma unroll
                                for (int i = 0; i < 8; ++i) sum[i] += v[i];
                            }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty + 8 * stage);
                    if (++stage == (uint32_t)q.stages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
#pragma unroll
            for (int i = 0; i < 8; ++i) total[i] += sum[i];
            wait(ready + 8 * set, set_phase);
            __syncwarp();
            tmem_acquire();
            const bool ends = last - from <= kSumSlices<T>;
            for (int b = 0; b < q.bn; b += 16) {
                const uint32_t at = tmem + b + ((uint32_t)warp << 21);
                const uint32_t total = at + q.sums_at.sets * q.columns;
                float v[16];
                accumulators16(at + set * q.columns, v);
                if (from > first) add16(total, v);
                if (!ends) store16(total, v);
                float *to = partial + (int64_t)o * q.Ci + i0 + b;
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    if (ends && o < q.Co && i0 + b + j < q.Ci) *reinterpret_cast<float4 *>(to + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            }
            if (ends) break;
            tmem_wait_store();
            tmem_release();
            __syncwarp();
            if (lane == 0) mbar_arrive(drained + 8 * set);
            if (++set == (uint32_t)q.sums_at.sets) {
                set = 0;
                set_phase ^= 1;
            }
        }
        if (sums) {
            if (LAST) {
#pragma unroll
                for (int i = 0; i < 8; ++i) part[8 * group + i][pixel] = total[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) part[threadIdx.x][i] = total[i];
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (o0 + (int)threadIdx.x < q.Co) {
                const float *v = part[threadIdx.x];
                partial[(int64_t)q.Co * q.Ci + o0 + threadIdx.x] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            }
        }
    }
    if (wait.lost) let_copies_land();
    __syncwarp();
    tmem_release();
    __syncthreads();
    if (warp == 5) tmem_free(tmem, q.sums_at.all);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Tiles, ring and grid of a product; false where the weights do not fit.
struct Plan {
    int bn, tiles_n, stages, columns, per_sm;
    int64_t tiles_p;
    unsigned walkers;
    uint32_t smem;
};
bool plan_product(const PointwiseShape &s, int K, int Cn, int mode, Plan *plan)
{
    const int samples = s.last ? 1 : s.N, chunks = (int)ceil_div(K, 64);
    const int64_t P = s.last ? s.N * s.P : s.P;
    const bool input = mode == INPUT;
    Plan r{};
    // channels of a tile: all of them up to 256, with weights of at most 128 KB
    const int64_t most = std::min<int64_t>(256, (int64_t)(128 << 10) / (chunks * 128) / 16 * 16);
    if (most < 32) return false;
    r.tiles_n = (int)ceil_div(Cn, most);
    r.bn = (int)ceil_div(ceil_div(Cn, r.tiles_n), 16) * 16;
    r.tiles_n = (int)ceil_div(Cn, r.bn);
    r.columns = 32;
    while (r.columns < r.bn) r.columns *= 2;
    r.tiles_p = ceil_div(P, 128);
    const int64_t tiles = r.tiles_p * samples;
    if (tiles > INT32_MAX || P > INT32_MAX - 256 || P * std::max(s.Ci, s.Co) >= (int64_t)1 << 38) return false;      // (coordinates, strides)
    // two CTAs an SM where both find room, or one with pairs of warps
    // ((32,32->128,64,128) f16 last with residual: 47 us alone with a ring of four, 43 with two CTAs and rings of three).  The
    // slope's epilogue does not fit the registers of two: alone ((32,128->64,64,128) bf16 last, SiLU: 43 us, 47 with two).
    r.per_sm = 2;
    for (r.stages = 4; r.stages > 2; --r.stages) {
        r.smem = MmaLayout{r.bn, r.stages, chunks, 1, input}.bytes();
        if (2 * (r.smem + 1024) <= 228 << 10) break;
    }
    if (r.columns > 128 || r.stages == 2 || mode == SLOPE) {
        r.per_sm = 1;
        r.stages = 4;
        while ((r.smem = MmaLayout{r.bn, r.stages, chunks, 2, input}.bytes()) > kMostShared)
            if (--r.stages < 2) return false;
    }
    r.walkers = (unsigned)std::min<int64_t>(tiles, std::max<int64_t>(1, 148 * r.per_sm / r.tiles_n));
    *plan = r;
    return true;
}

template <int MODE>
int launch_mma(const PointwiseShape &s, const Plan &plan, MmaProduct q, const void *a, const void *a_rest, const void *w, cudaStream_t stream)
{
    const bool bf16 = s.io_kind == BC_IO_BF16;
    q.samples = s.last ? 1 : s.N;
    q.P = s.last ? s.N * s.P : s.P;
    q.tiles_p = (int)plan.tiles_p;
    q.tiles_n = plan.tiles_n;
    q.bn = plan.bn;
    q.stages = plan.stages;
    q.columns = plan.columns;
    q.instruction = mma_instruction(bf16, !s.last, MODE == INPUT, plan.bn);
    {
        const uint64_t last_sizes[2] = {(uint64_t)q.K, (uint64_t)q.P}, last_strides[1] = {(uint64_t)q.K};
        const uint64_t sizes[3] = {(uint64_t)q.P, (uint64_t)q.K, (uint64_t)q.samples}, strides[2] = {(uint64_t)q.P, (uint64_t)q.P * q.K};
        const uint32_t last_box[2] = {64, 128}, box[3] = {64, 64, 1};
        auto map = [&](CUtensorMap *to, const void *from) {
            return s.last ? make_map(to, from, bf16, 2, last_sizes, last_strides, last_box) : make_map(to, from, bf16, 3, sizes, strides, box);
        };
        if (const int e = map(&q.a, a)) return e;
        q.parts = a_rest ? 2 : 1;
        if (a_rest)
            if (const int e = map(&q.a_rest, a_rest)) return e;
        const uint64_t w_sizes[2] = {(uint64_t)s.Ci, (uint64_t)s.Co}, w_strides[1] = {(uint64_t)s.Ci};
        const uint32_t w_box[2] = {64, MODE == INPUT ? 64u : (uint32_t)plan.bn};
        if (const int e = make_map(&q.w, w, bf16, 2, w_sizes, w_strides, w_box)) return e;
    }
    return with_activation(MODE == INPUT ? BC_ACT_NONE : s.act, [&](auto act) {
        constexpr int ACT = MODE == INPUT ? BC_ACT_NONE : act();
        auto go = [&](auto kernel) {
            if (const int e = raise_smem_limit((const void *)kernel, kMostShared)) return e;
            const LaunchScope scope(KID_POINTWISE_MMA, stream);
            launch_overlapped(kernel, plan.walkers * plan.tiles_n, 32 * (kEpilogue * (plan.per_sm == 1 ? 2 : 1) + 2), plan.smem, stream, q);
            return check_launch("pointwise_mma_kernel");
        };
        auto of_type = [&](auto t, auto pair) {
            using T = decltype(t);
            constexpr int PAIR = decltype(pair)::value;
            return s.last ? go(pointwise_mma_kernel<T, MODE, ACT, true, PAIR>) : go(pointwise_mma_kernel<T, MODE, ACT, false, PAIR>);
        };
        auto run = [&](auto pair) { return bf16 ? of_type(__nv_bfloat16(), pair) : of_type(__half(), pair); };
        if constexpr (MODE != SLOPE)
            if (plan.per_sm == 2) return run(std::integral_constant<int, 1>());
        return run(std::integral_constant<int, 2>());
    });
}

// TMA wants rows that start on 16 bytes; the epilogue's vectors too.
bool rows_aligned(const PointwiseShape &s)
{
    if (s.io_kind == BC_IO_F32 || s.Ci % 8 || s.Ci < 8) return false;
    return s.last ? s.Co % 8 == 0 && s.Co >= 8 : s.P % 8 == 0;
}

}  // namespace

// ---- the products with pixels in the rows; false: not for these kernels
bool pointwise_mma_suits(const PointwiseShape &s, bool input)
{
    Plan plan;
    return rows_aligned(s) && plan_product(s, input ? s.Co : s.Ci, input ? s.Ci : s.Co, input ? INPUT : SLOPE, &plan);
}
bool pointwise_mma_aligned(const void *a, const void *b, const void *c, const void *d, const void *e)
{
    return aligned16(a) && aligned16(b) && aligned16(c) && aligned16(d) && aligned16(e);
}
int pointwise_mma_sums_rows(const PointwiseShape &s)
{
    Plan plan;
    return plan_product(s, s.Ci, s.Co, SLOPE, &plan) ? (int)plan.walkers : 0;
}
int launch_pointwise_mma_forward(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual, void *out,
                                 cudaStream_t stream)
{
    Plan plan;
    plan_product(s, s.Ci, s.Co, FORWARD, &plan);
    MmaProduct q{};
    q.bias = bias;
    q.residual = residual;
    q.out = out;
    q.K = s.Ci;
    q.Cn = s.Co;
    return launch_mma<FORWARD>(s, plan, q, x, nullptr, weight, stream);
}
int launch_pointwise_mma_slope(const PointwiseShape &s, const void *x, const void *weight, const void *bias, const void *residual,
                               const void *grad, void *dz, void *rest, float *sums, cudaStream_t stream)
{
    Plan plan;
    plan_product(s, s.Ci, s.Co, SLOPE, &plan);
    MmaProduct q{};
    q.bias = bias;
    q.residual = residual;
    q.grad = grad;
    q.out = dz;
    q.rest = rest;
    q.sums = sums;
    q.K = s.Ci;
    q.Cn = s.Co;
    return launch_mma<SLOPE>(s, plan, q, x, nullptr, weight, stream);
}
int launch_pointwise_mma_input(const PointwiseShape &s, const void *dz, const void *rest, const void *weight, void *grad_input,
                               cudaStream_t stream)
{
    Plan plan;
    plan_product(s, s.Co, s.Ci, INPUT, &plan);
    MmaProduct q{};
    q.out = grad_input;
    q.K = s.Co;
    q.Cn = s.Ci;
    return launch_mma<INPUT>(s, plan, q, dz, rest, weight, stream);
}

// ---- grad_weight: rows of pointwise_partial_stride() floats, to be added
namespace {
struct WeightPlan {
    int tiles_o, tiles_i, bn, stages, columns, splits;
    int64_t slices, per;
    uint32_t smem;
};
bool plan_weight(const PointwiseShape &s, int parts, WeightPlan *plan)
{
    if (!rows_aligned(s)) return false;
    const int64_t P = s.last ? s.N * s.P : s.P, samples = s.last ? 1 : s.N;
    if (P > INT32_MAX - 256 || P * std::max(s.Ci, s.Co) >= (int64_t)1 << 38) return false;
    WeightPlan r{};
    r.tiles_o = (int)ceil_div(s.Co, 128);
    r.tiles_i = (int)ceil_div(s.Ci, 256);
    r.bn = (int)ceil_div(ceil_div(s.Ci, r.tiles_i), 16) * 16;
    r.tiles_i = (int)ceil_div(s.Ci, r.bn);
    r.columns = 32;
    while (r.columns < r.bn) r.columns *= 2;
    for (r.stages = kMostStages; r.stages > 2; --r.stages) {
        r.smem = WeightLayout{r.bn, r.stages, parts, s.last}.bytes();
        if (r.smem <= 200 << 10) break;
    }
    r.slices = ceil_div(P, 64);
    const int64_t all = r.slices * samples, tiles = (int64_t)r.tiles_o * r.tiles_i;
    r.per = slices_of_split(all, tiles, kSumSlices<__half> * kMostSums<__half>);
    r.splits = (int)ceil_div(all, r.per);
    if (r.splits * tiles > INT32_MAX) return false;
    *plan = r;
    return true;
}
}  // namespace

int pointwise_mma_weight_splits(const PointwiseShape &s)
{
    WeightPlan plan;
    return plan_weight(s, 1, &plan) ? plan.splits : 0;      // (as many in two parts)
}
int launch_pointwise_mma_weight(const PointwiseShape &s, const void *dz, const void *rest, const void *x, float *partial, bool sums,
                                cudaStream_t stream)
{
    WeightPlan plan;
    plan_weight(s, rest ? 2 : 1, &plan);
    const bool bf16 = s.io_kind == BC_IO_BF16;
    WeightMma q{};
    q.partial = partial;
    q.per = plan.per;
    q.slices = plan.slices;
    q.samples = s.last ? 1 : s.N;
    q.Ci = s.Ci;
    q.Co = s.Co;
    q.tiles_i = plan.tiles_i;
    q.bn = plan.bn;
    q.rows = std::min(128, (int)ceil_div(s.Co, 8) * 8);
    q.stages = plan.stages;
    q.columns = plan.columns;
    q.sums = sums;
    q.instruction = mma_instruction(bf16, s.last, s.last, plan.bn);
    const int64_t P = s.last ? s.N * s.P : s.P;
    auto map = [&](CUtensorMap *to, const void *from, int C, uint32_t rows) {
        const uint64_t last_sizes[2] = {(uint64_t)C, (uint64_t)P}, last_strides[1] = {(uint64_t)C};
        const uint64_t sizes[3] = {(uint64_t)P, (uint64_t)C, (uint64_t)s.N}, strides[2] = {(uint64_t)P, (uint64_t)P * C};
        const uint32_t last_box[2] = {64, 64}, box[3] = {64, rows, 1};
        return s.last ? make_map(to, from, bf16, 2, last_sizes, last_strides, last_box) : make_map(to, from, bf16, 3, sizes, strides, box);
    };
    q.sums_at = sum_columns(plan.per > kSumSlices<__half>, plan.columns, plan.bn);
    if (const int e = map(&q.dz, dz, s.Co, q.rows)) return e;
    if (rest)
        if (const int e = map(&q.dz_rest, rest, s.Co, q.rows)) return e;
    if (const int e = map(&q.x, x, s.Ci, plan.bn)) return e;
    auto go = [&](auto kernel) {
        if (const int e = raise_smem_limit((const void *)kernel, 200 << 10)) return e;
        const LaunchScope scope(KID_POINTWISE_WEIGHT_MMA, stream);
        launch_overlapped(kernel, (unsigned)(plan.splits * plan.tiles_o * plan.tiles_i), kWeightThreads, plan.smem, stream, q);
        return check_launch("pointwise_weight_mma_kernel");
    };
    auto of = [&](auto t, auto parts) {
        using T = decltype(t);
        return s.last ? go(pointwise_weight_mma_kernel<T, true, decltype(parts)::value>) : go(pointwise_weight_mma_kernel<T, false, decltype(parts)::value>);
    };
    auto of_parts = [&](auto parts) { return bf16 ? of(__nv_bfloat16(), parts) : of(__half(), parts); };
    return rest ? of_parts(std::integral_constant<int, 2>()) : of_parts(std::integral_constant<int, 1>());
}

int read_wait_timeouts_mma(int *count) { return read_wait_timeouts_here(count); }

}  // namespace bc
