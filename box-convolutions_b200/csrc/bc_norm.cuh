// Group normalisation on vectors of 16 bytes: what group_norm_last.cu and group_norm_planes.cu share.
//
// A unit is what has statistics in common (a group's planes; channels last, some groups of a sample), cut into slices,
// one a CTA.  A slice is read twice, once for its sums and once for the results, and is short enough for the second
// reading to come from the SM's L1 cache or from L2: memory is read once.  Between the two the unit's CTAs exchange their
// sums: up to 8 CTAs as a cluster through distributed shared memory, in one launch; more (few samples of many pixels) through
// a workspace, in two.
#pragma once
#include "bc_cluster.cuh"
#include "bc_layers.cuh"

namespace bc {

// Which part a launch does: both readings (a cluster), the sums, the results.
enum { NORM_WHOLE, NORM_SUMS, NORM_RESULTS };

// Count, mean and variance: two of them make the third's without cancellation wherever the mean lies.  (The variance and not
// the sum of squares, which may be no float where the variance is one.)
struct Moments {
    float n, mean, var;
};
__device__ __forceinline__ Moments merged(const Moments &a, const Moments &b)
{
    // (nothing on either side leaves the other as it is: its mean's square, which has no part in this, may be no float)
    if (a.n == 0.f) return b;
    if (b.n == 0.f) return a;
    const float n = a.n + b.n, d = b.mean - a.mean, share = __fdividef(b.n, n);
    return {n, fmaf(d, share, a.mean), fmaf(share, fmaf(d * d, 1.f - share, b.var - a.var), a.var)};
}
__device__ __forceinline__ Moments warp_merged(Moments v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Moments w{__shfl_down_sync(0xffffffffu, v.n, o), __shfl_down_sync(0xffffffffu, v.mean, o),
                        __shfl_down_sync(0xffffffffu, v.var, o)};
        v = merged(v, w);
    }
    return v;      // lane 0's
}

__device__ __forceinline__ float cluster_load(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// ---- plans: how many CTAs share a unit
constexpr int kNormCluster = 8;
// Bytes of a slice that are worth a CTA, and CTAs that fill the GPU (two an SM).
constexpr int64_t kNormSlice = 64 << 10;
constexpr int kNormFill = 296;

struct NormRows {       // channels last
    int threads, active;       // of a CTA; of those with work
    int width, slabs;          // channels of a unit, units of a sample
    int k, per;                // CTAs of a unit, pixels of each
};
bool plan_rows(const NormShape &s, NormRows *plan);
size_t rows_sums_bytes(const NormShape &s, const NormRows &plan, bool backward);

struct NormPlanes {
    int threads;
    int chunk, chunks;         // values of a piece, pieces of a plane
    int k, per;                // CTAs of a unit, pieces of each
};
void plan_planes(const NormShape &s, NormPlanes *plan);
size_t planes_sums_bytes(const NormShape &s, const NormPlanes &plan, bool backward);

// The results of the launches; backward: `sums` receives `*rows` rows of C pairs, S1 and S2 of each channel, to be added.
int launch_norm_rows_forward(const NormShape &s, const NormRows &plan, const void *x, const void *weight, const void *bias, void *out,
                             float *stats, void *ws, cudaStream_t stream);
int launch_norm_rows_backward(const NormShape &s, const NormRows &plan, const void *x, const void *weight, const void *bias,
                              const float *stats, const void *grad, void *grad_input, float *sums, cudaStream_t stream);
int launch_norm_planes_forward(const NormShape &s, const NormPlanes &plan, const void *x, const void *weight, const void *bias, void *out,
                               float *stats, void *ws, cudaStream_t stream);
int launch_norm_planes_backward(const NormShape &s, const NormPlanes &plan, const void *x, const void *weight, const void *bias,
                                const float *stats, const void *grad, void *grad_input, float *sums, cudaStream_t stream);

inline int64_t norm_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace bc
