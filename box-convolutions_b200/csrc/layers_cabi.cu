// The extern "C" surface of the layers around a box convolution: argument checks and dispatch, as in cabi.cu.
#include "bc_layers.cuh"

using namespace bc;

namespace {

bool kind_ok(int io_kind) { return io_kind == BC_IO_F32 || io_kind == BC_IO_F16 || io_kind == BC_IO_BF16; }
bool act_ok(int act) { return act >= BC_ACT_NONE && act <= BC_ACT_GELU; }

// Sizes whose products stay below 2^62: every offset is a 64-bit one.
bool sizes_ok(int N, int C, int64_t pixels)
{
    if (N < 0 || C < 0 || pixels < 0 || pixels > INT32_MAX) return false;
    const __int128 total = (__int128)N * (C ? C : 1) * pixels;
    return total < ((__int128)1 << 60);
}

int check(const NormShape &s)
{
    if (!sizes_ok(s.N, s.C, s.P) || s.G < 1 || s.C % s.G) return BC_ERR_BAD_SHAPE;
    return kind_ok(s.io_kind) && act_ok(s.act) ? BC_OK : BC_ERR_UNSUPPORTED;
}

int check(const PointwiseShape &s)
{
    if (!sizes_ok(s.N, s.Ci, s.P) || !sizes_ok(s.N, s.Co, s.P)) return BC_ERR_BAD_SHAPE;
    return kind_ok(s.io_kind) && act_ok(s.act) ? BC_OK : BC_ERR_UNSUPPORTED;
}

// With one pixel a sample the two layouts are the same memory, and rows of channels the longer runs.
bool rows(int channels_last, int64_t pixels) { return channels_last || pixels == 1; }

int zeros(void *p, size_t bytes, cudaStream_t stream)
{
    if (!bytes) return BC_OK;
    const cudaError_t e = cudaMemsetAsync(p, 0, bytes, stream);
    return e == cudaSuccess ? BC_OK : cuda_failed(e, "cudaMemsetAsync");
}

}  // namespace

extern "C" {

int bc_pointwise_forward(const void *input, const void *weight, const void *bias, const void *residual, void *out, int io_kind,
                         int N, int in_planes, int out_planes, int64_t pixels, int channels_last, int activation, bc_stream_t stream)
{
    const PointwiseShape s{N, in_planes, out_planes, pixels, rows(channels_last, pixels), io_kind, activation};
    if (const int e = check(s)) return e;
    if (!N || !out_planes || !pixels) return BC_OK;
    if (!out || (in_planes && (!input || !weight))) return BC_ERR_NULL_POINTER;
    return launch_pointwise_forward(s, input, weight, bias, residual, out, stream);
}

size_t bc_pointwise_backward_workspace(int io_kind, int N, int in_planes, int out_planes, int64_t pixels, int channels_last,
                                       int activation, int need_mask)
{
    const PointwiseShape s{N, in_planes, out_planes, pixels, rows(channels_last, pixels), io_kind, activation};
    if (check(s) || !N || !out_planes || !pixels) return 0;
    return pointwise_workspace(s, need_mask);
}

int bc_pointwise_backward(const void *input, const void *weight, const void *bias, const void *residual, const void *grad_output,
                          int io_kind, int N, int in_planes, int out_planes, int64_t pixels, int channels_last, int activation,
                          int need_mask, void *grad_input, void *grad_weight, void *grad_bias, void *grad_residual,
                          void *workspace, size_t workspace_bytes, bc_stream_t stream)
{
    const PointwiseShape s{N, in_planes, out_planes, pixels, rows(channels_last, pixels), io_kind, activation};
    if (const int e = check(s)) return e;
    need_mask &= BC_NEED_PW_INPUT | BC_NEED_PW_WEIGHT | BC_NEED_PW_BIAS | (activation == BC_ACT_NONE ? 0 : BC_NEED_PW_RESIDUAL);
    // (gradients without a value)
    if (!N || !pixels || !in_planes) need_mask &= ~BC_NEED_PW_INPUT;
    if (!in_planes || !out_planes) need_mask &= ~BC_NEED_PW_WEIGHT;
    if (!out_planes) need_mask &= ~BC_NEED_PW_BIAS;
    if (!N || !pixels || !out_planes) need_mask &= ~BC_NEED_PW_RESIDUAL;
    if (((need_mask & BC_NEED_PW_INPUT) && !grad_input) || ((need_mask & BC_NEED_PW_WEIGHT) && !grad_weight) ||
        ((need_mask & BC_NEED_PW_BIAS) && !grad_bias) || ((need_mask & BC_NEED_PW_RESIDUAL) && !grad_residual))
        return BC_ERR_NULL_POINTER;
    if (!need_mask) return BC_OK;
    const size_t size = io_size(io_kind);
    if (!N || !pixels || !out_planes) {      // sums over nothing
        int e = BC_OK;
        if (need_mask & BC_NEED_PW_INPUT) e = zeros(grad_input, size * N * in_planes * pixels, stream);
        if (!e && (need_mask & BC_NEED_PW_WEIGHT)) e = zeros(grad_weight, size * out_planes * in_planes, stream);
        if (!e && (need_mask & BC_NEED_PW_BIAS)) e = zeros(grad_bias, size * out_planes, stream);
        return e;
    }
    if (!grad_output || (in_planes && (!input || !weight))) return BC_ERR_NULL_POINTER;
    const size_t need = pointwise_workspace(s, need_mask);
    if (need && (!workspace || workspace_bytes < need)) return BC_ERR_WORKSPACE;
    return launch_pointwise_backward(s, input, weight, bias, residual, grad_output, need_mask, grad_input, grad_weight, grad_bias,
                                     grad_residual, workspace, stream);
}

size_t bc_group_norm_forward_workspace(int io_kind, int N, int C, int64_t pixels, int groups, int channels_last)
{
    const NormShape s{N, C, groups, pixels, rows(channels_last, pixels), io_kind, BC_ACT_NONE, 0.f};
    return check(s) || !N || !C || !pixels ? 0 : group_norm_workspace(s, 0);
}

int bc_group_norm_forward(const void *input, const void *weight, const void *bias, void *out, float *stats, int io_kind, int N, int C,
                          int64_t pixels, int groups, float eps, int channels_last, int activation, void *workspace,
                          size_t workspace_bytes, bc_stream_t stream)
{
    const NormShape s{N, C, groups, pixels, rows(channels_last, pixels), io_kind, activation, eps};
    if (const int e = check(s)) return e;
    if (!N || !C || !pixels) return BC_OK;
    if (!input || !out) return BC_ERR_NULL_POINTER;
    const size_t need = group_norm_workspace(s, 0);
    if (need && (!workspace || workspace_bytes < need)) return BC_ERR_WORKSPACE;
    return launch_group_norm_forward(s, input, weight, bias, out, stats, workspace, stream);
}

size_t bc_group_norm_backward_workspace(int io_kind, int N, int C, int64_t pixels, int groups, int channels_last)
{
    const NormShape s{N, C, groups, pixels, rows(channels_last, pixels), io_kind, BC_ACT_NONE, 0.f};
    return check(s) || !N || !C || !pixels ? 0 : group_norm_workspace(s, BC_NEED_GN_INPUT | BC_NEED_GN_WEIGHT | BC_NEED_GN_BIAS);
}

int bc_group_norm_backward(const void *input, const void *weight, const void *bias, const float *stats, const void *grad_output,
                           int io_kind, int N, int C, int64_t pixels, int groups, int channels_last, int activation, int need_mask,
                           void *grad_input, void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes,
                           bc_stream_t stream)
{
    const NormShape s{N, C, groups, pixels, rows(channels_last, pixels), io_kind, activation, 0.f};
    if (const int e = check(s)) return e;
    need_mask &= BC_NEED_GN_INPUT | BC_NEED_GN_WEIGHT | BC_NEED_GN_BIAS;
    if (!C) return BC_OK;
    if (!N || !pixels) need_mask &= ~BC_NEED_GN_INPUT;
    if (((need_mask & BC_NEED_GN_INPUT) && !grad_input) || ((need_mask & BC_NEED_GN_WEIGHT) && !grad_weight) ||
        ((need_mask & BC_NEED_GN_BIAS) && !grad_bias))
        return BC_ERR_NULL_POINTER;
    if (!need_mask) return BC_OK;
    if (!N || !pixels) {
        int e = BC_OK;
        if (need_mask & BC_NEED_GN_WEIGHT) e = zeros(grad_weight, (size_t)io_size(io_kind) * C, stream);
        if (!e && (need_mask & BC_NEED_GN_BIAS)) e = zeros(grad_bias, (size_t)io_size(io_kind) * C, stream);
        return e;
    }
    if (!input || !grad_output || !stats) return BC_ERR_NULL_POINTER;
    const size_t need = group_norm_workspace(s, BC_NEED_GN_INPUT | BC_NEED_GN_WEIGHT | BC_NEED_GN_BIAS);
    if (need && (!workspace || workspace_bytes < need)) return BC_ERR_WORKSPACE;
    return launch_group_norm_backward(s, input, weight, bias, stats, grad_output, need_mask, grad_input, grad_weight, grad_bias, workspace,
                                      stream);
}

}  // extern "C"
