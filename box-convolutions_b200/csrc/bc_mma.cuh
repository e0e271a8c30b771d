// tcgen05 products of 16-bit operands: shared-memory descriptors, issue, completion; tensor maps.
//
// Operands lie in shared memory as TMA's 128-byte swizzle leaves them.  K-major (k runs along memory): rows of 64 k, 8 rows of
// 128 bytes a swizzle atom.  MN-major (the other index runs along memory): blocks of 64 m or n, a row of 128 bytes for each k.
#pragma once
#include <cuda.h>

#include "bc_layers.cuh"
#include "bc_tile_io.cuh"
#include "bc_tmem.cuh"

namespace bc {

namespace {

constexpr uint32_t kBlockBytes = 64 * 128;      // an MN-major block of 64 k

// 14 bits each: start, leading and stride byte offsets in units of 16; version 1; 128-byte swizzle.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t leading, uint32_t stride)
{
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// K-major: 16 k are 32 bytes on within the atoms' rows.
__device__ __forceinline__ uint64_t k_major(uint32_t addr, int k) { return operand(addr + 2 * k, 16, 1024); }
// MN-major: blocks `block` bytes apart; 8 k are an atom of 1024 bytes.
__device__ __forceinline__ uint64_t mn_major(uint32_t addr, int k, uint32_t block) { return operand(addr + 128 * k, block, 1024); }

// The same operand `bytes` further on.  (The issuing thread is alone on its scheduler slot: what it computes for every
// instruction, the tensor cores wait for.)
__device__ __forceinline__ uint64_t further(uint64_t operand, uint32_t bytes) { return operand + (bytes >> 4); }

// 16-bit operands of one type, float accumulators, M 128.
__host__ __device__ inline uint32_t mma_instruction(bool bf16, bool a_mn, bool b_mn, int n)
{
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 |
           (uint32_t)(128 >> 4) << 24;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add) : "memory");
}
// The same of operands in two words, the address in the lower one.
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t instruction, bool add)
{
    asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %6, 0;\n mov.b64 x, {%1, %2};\n mov.b64 y, {%3, %4};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, p;\n}"
                 ::"r"(d), "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(instruction), "r"((uint32_t)add) : "memory");
}
// Arrives once everything issued so far by this thread is done (and has been read).
__device__ __forceinline__ void mma_commit(uint32_t mbar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(mbar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t mbar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mbar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t mbar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mbar) : "memory"); }
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t mbar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(mbar) : "memory");
}
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t mbar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(mbar) : "memory");
}
__device__ __forceinline__ void map_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// The tensor memory of such sums: one or two sets of accumulators of `columns` (a power of two), two where there is room, and
// behind them `width` columns of totals.
struct SumColumns {
    int sets, all;
};
inline SumColumns sum_columns(bool several, int columns, int width)
{
    if (!several) return {1, columns};
    const int sets = 2 * columns + width <= 512 ? 2 : 1;
    int all = 32;
    while (all < sets * columns + width) all *= 2;
    return {sets, all};
}

// 16 accumulators of each of the warp's lanes.
__device__ __forceinline__ void accumulators16(uint32_t at, float (&v)[16])
{
    float4 q[4];
    tmem_load16(at, q);
    tmem_wait_load(q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[4 * i] = q[i].x;
        v[4 * i + 1] = q[i].y;
        v[4 * i + 2] = q[i].z;
        v[4 * i + 3] = q[i].w;
    }
}

__device__ __forceinline__ void store16(uint32_t at, const float (&v)[16])
{
#pragma unroll
    for (int i = 0; i < 16; i += 8)
        tmem_store8(at + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), make_float4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]));
}
__device__ __forceinline__ void add16(uint32_t at, float (&v)[16])
{
    float u[16];
    accumulators16(at, u);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += u[j];
}

// Halves the values of the two lanes that `mask` tells apart: the one without the bit goes on with the lower half of both's sums.
template <int N>
__device__ __forceinline__ void fold(float (&v)[N], int lane, int mask, int half)
{
#pragma unroll
    for (int j = 0; j < N / 2; ++j)
        if (j < half) {
            const bool high = lane & mask;
            const float keep = high ? v[j + half] : v[j], send = high ? v[j] : v[j + half];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, send, mask);
        }
}

// Slices of 64 pixels that an accumulator of grad_weight takes before its sum goes on to another part of tensor memory.  An
// accumulator rounds towards zero with every addition (two an instruction of 16 pixels, as measured: 28340 instructions lost 2.8e-3
// of a sum of one sign), which adds up, so a sum is of 128 additions for float tensors and 512 for 16-bit ones: they lose 2^-17
// and 2^-15 of a sum that grows evenly, whatever the number of pixels.  What follows is rounded to nearest: kMostSums of them in
// a row of partial sums, and the rows in double.  Kernels, one accumulator throughout and so: (64,128->128,64,128) f32 291 us
// and 289, channels last 504 and 516; (1,16->16,2048,2048) f32 432 and 513; (16,128->32,64,128) f32 43.5 and 47.6.
template <typename T>
constexpr int kSumSlices = sizeof(T) == 4 ? 16 : 64;
template <typename T>
constexpr int kMostSums = sizeof(T) == 4 ? 16 : 64;
// Slices of a CTA, `most` or less: a CTA an SM with four at least, else as few rounds of them as will do.
inline int64_t slices_of_split(int64_t all, int64_t tiles, int64_t most)
{
    const int64_t walkers = std::max<int64_t>(1, 148 / tiles), per = std::max<int64_t>(std::min<int64_t>(4, all), (all + walkers - 1) / walkers);
    const int64_t rounds = (per + most - 1) / most;
    return rounds > 1 ? (all + walkers * rounds - 1) / (walkers * rounds) : per;
}

// A wait whose expiry ends all further ones of the thread: a lost arrival is counted (bc_wait_timeouts), and nothing hangs.
// Threads learn of a loss each for itself, so one that works alone may leave its loop on it, and a warp as a whole whose loop
// has no other warps' barriers; whoever shares those goes round to the loop's end, where further waits return at once and
// values mean nothing.
struct Waiter {
    bool lost = false;
    __device__ __forceinline__ bool operator()(uint32_t mbar, uint32_t parity)
    {
        if (lost) return false;
        if (mbar_wait(mbar, parity)) return true;
        atomicAdd(&g_wait_timeouts, 1);
        lost = true;
        return false;
    }
};
// Before a CTA that has lost an arrival leaves: time for its copies and products in flight, far more than any takes.
__device__ __forceinline__ void let_copies_land()
{
    for (const long long t0 = clock64(); clock64() - t0 < 20000000LL;) __nanosleep(1000);
}

}  // namespace

// Tensor map of 16-bit values, 128-byte swizzle, zeros outside: `rank` sizes and boxes, innermost first, strides in values of
// the second dimension on.
inline int make_map(CUtensorMap *map, const void *base, bool bf16, int rank, const uint64_t *sizes, const uint64_t *strides,
                    const uint32_t *box)
{
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                               CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return (Encode)f;
    }();
    if (!encode) return cuda_failed(cudaErrorNotSupported, "cuTensorMapEncodeTiled");
    cuuint64_t bytes[4] = {};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    for (int i = 0; i + 1 < rank; ++i) bytes[i] = 2 * strides[i];
    auto call = [&] {
        return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void *>(base), sizes, bytes,
                      box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = call();
    if (r != CUDA_SUCCESS) {
        // A thread whose first call into CUDA this is (autograd's, say) has a device but no context yet, which the driver's
        // function asks for and the runtime's provide.
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess) e = cudaSetDevice(device);
        if (e != cudaSuccess) return cuda_failed(e, "cuTensorMapEncodeTiled");
        r = call();
    }
    return r == CUDA_SUCCESS ? BC_OK : cuda_failed(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
}

}  // namespace bc
