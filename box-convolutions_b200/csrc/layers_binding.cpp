// The layers around a box convolution (box_convolution/layers.py documents them): argument checks, allocation, autograd
// nodes.  Like the box convolution's own path in torch_binding.cpp, and for the same reason: a step of a small block is
// bound by what the host does between its kernels.
#include "binding_common.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void require_layer_tensor(const Tensor &t, const std::string &what, const Tensor &input)
{
    if (!t.is_cuda()) fail(what + " is not a CUDA tensor; this build has no CPU implementation");
    const at::ScalarType have = t.scalar_type();
    if (have != at::kFloat && !is_narrow(have)) fail(what + " must be float32, float16 or bfloat16, got " + dtype_name(have));
    if (have != input.scalar_type())
        fail(what + " is " + dtype_name(have) + " but the call's input is " + dtype_name(input.scalar_type()));
    if (t.device() != input.device()) fail(what + " and the input are on different devices");
}

// Tensors of a call are all planes or all channels last, as the input is; what has other strides is copied.
// (One plane a sample is both; its strides tell what the caller takes it for.)
bool is_last(const Tensor &input) { return input.suggest_memory_format() == at::MemoryFormat::ChannelsLast; }
at::MemoryFormat format(bool last) { return last ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous; }
Tensor dense(const Tensor &t, bool last) { return t.defined() ? t.contiguous(format(last)) : t; }
Tensor row(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
Tensor new_maps(at::IntArrayRef sizes, bool last, const Tensor &like)
{
    return Tensor(at::detail::empty_cuda(sizes, like.scalar_type(), like.device(), format(last)));
}
const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// Calls for the Python classes of layers.py, torch.autograd.Functions: a trace records them as operations, and they refuse
// tangents of forward-mode differentiation and function transforms.
template <class... Ts>
bool needs_python_class(const Ts &...tensors)
{
    using c10::impl::tls_is_dispatch_key_included;
    if (tls_is_dispatch_key_included(at::DispatchKey::Tracer) ||
        tls_is_dispatch_key_included(at::DispatchKey::FuncTorchDynamicLayerFrontMode))
        return true;
    return ((tensors.defined() && tensors._fw_grad(/*level=*/0).defined()) || ...);
}
template <class... Ts>
bool wants_gradient(const Ts &...tensors)
{
    return at::GradMode::is_enabled() && ((tensors.defined() && tensors.requires_grad()) || ...);
}

// Gradients made with create_graph: differentiating them again is an error and not a gradient without its other half.
variable_list once_differentiable(variable_list &&list, bool create_graph, const char *name)
{
    if (!create_graph) return std::move(list);
    for (Tensor &t : list)
        if (t.defined()) t = t.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(name) + ": the gradient cannot be differentiated again", (int64_t)list.size());
    return (*error)(std::move(list));
}

// An output that a trace has seen being made.
Tensor seen_by_trace(const Tensor &out)
{
    if (!out.defined() || !c10::impl::tls_is_dispatch_key_included(at::DispatchKey::Tracer)) return out;
    const Tensor seen = at::empty(out.sizes(), out.options(), out.suggest_memory_format());
    at::tracer::impl::NoTracerDispatchMode no_tracer;
    seen.copy_(out);
    return seen;
}

PyObject *wrap_list(const std::vector<Tensor> &v)
{
    THPObjectPtr list(PyList_New((Py_ssize_t)v.size()));
    if (!list) throw python_error();
    for (size_t i = 0; i < v.size(); ++i) PyList_SET_ITEM(list.get(), (Py_ssize_t)i, wrap(v[i]));
    return list.release();
}

int activation_of(int64_t act)
{
    if (act < BC_ACT_NONE || act > BC_ACT_GELU) fail("box_convolution: unknown activation");
    return (int)act;
}

// ---- pointwise convolution -----------------------------------------------------------------------

struct Mixing {
    int N, Ci, Co, act;
    int64_t P;
    bool last;
    std::array<int64_t, 4> out_sizes;
};

Mixing check_pointwise(const Tensor &input, const Tensor &weight, const Tensor &bias, const Tensor &residual, int64_t act)
{
    require_layer_tensor(input, "pointwise_conv2d: input", input);
    if (input.dim() != 4) fail("pointwise_conv2d: input must have 4 dimensions");
    require_layer_tensor(weight, "pointwise_conv2d: weight", input);
    if (!(weight.dim() == 2 || (weight.dim() == 4 && weight.size(2) == 1 && weight.size(3) == 1)) || weight.size(1) != input.size(1))
        fail("pointwise_conv2d: weight must be (out_planes, " + std::to_string(input.size(1)) + ") or (out_planes, " +
             std::to_string(input.size(1)) + ", 1, 1)");
    Mixing s{to_int(input.size(0)), to_int(input.size(1)), to_int(weight.size(0)), activation_of(act), input.size(2) * input.size(3),
             is_last(input), {input.size(0), weight.size(0), input.size(2), input.size(3)}};
    to_int(s.P);
    if (bias.defined()) {
        require_layer_tensor(bias, "pointwise_conv2d: bias", input);
        if (bias.dim() != 1 || bias.size(0) != s.Co) fail("pointwise_conv2d: bias must hold " + std::to_string(s.Co) + " values");
    }
    if (residual.defined()) {
        require_layer_tensor(residual, "pointwise_conv2d: residual", input);
        if (residual.sizes() != at::IntArrayRef(s.out_sizes)) fail("pointwise_conv2d: residual must have the output's shape");
    }
    return s;
}

// x, weight, bias, residual: dense
Tensor run_pointwise(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &residual, const Mixing &s)
{
    Tensor out = new_maps(s.out_sizes, s.last, x);
    check_status(bc_pointwise_forward(ptr(x), ptr(weight), ptr(bias), ptr(residual), out.data_ptr(), io_kind(x.scalar_type()), s.N, s.Ci,
                                      s.Co, s.P, s.last, s.act, current_stream(x)),
                 "pointwise_conv2d");
    return out;
}

std::vector<Tensor> run_pointwise_backward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &residual,
                                           const Tensor &grad_output, const Mixing &s, int mask)
{
    std::vector<Tensor> g(4);
    if (!mask) return g;
    require_layer_tensor(grad_output, "pointwise_conv2d: grad_output", x);
    if (grad_output.sizes() != at::IntArrayRef(s.out_sizes)) fail("pointwise_conv2d: grad_output must have the output's shape");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor grad = dense(grad_output, s.last), w = row(weight), b = row(bias), r = dense(residual, s.last);
    if (mask & BC_NEED_PW_INPUT) g[0] = new_maps(x.sizes(), s.last, x);
    if (mask & BC_NEED_PW_WEIGHT) g[1] = new_tensor(weight.sizes(), x.scalar_type(), x);
    if (mask & BC_NEED_PW_BIAS) g[2] = new_tensor({s.Co}, x.scalar_type(), x);
    if (mask & BC_NEED_PW_RESIDUAL) g[3] = s.act == BC_ACT_NONE ? grad : new_maps(s.out_sizes, s.last, x);
    const int kind = io_kind(x.scalar_type());
    const size_t bytes = bc_pointwise_backward_workspace(kind, s.N, s.Ci, s.Co, s.P, s.last, s.act, mask);
    Tensor ws;
    if (bytes) ws = new_workspace(bytes, x);
    check_status(bc_pointwise_backward(ptr(x), ptr(w), ptr(b), ptr(r), ptr(grad), kind, s.N, s.Ci, s.Co, s.P, s.last, s.act, mask, out_ptr(g[0]),
                                       out_ptr(g[1]), out_ptr(g[2]), out_ptr(g[3]), out_ptr(ws), bytes, current_stream(x)),
                 "pointwise_conv2d backward");
    return g;
}

struct PointwiseConvBackward : torch::autograd::Node {
    SavedVariable x, weight, bias, residual;      // (bias and residual: where an activation's slope asks for them)
    Mixing shape;
    std::mutex mutex;

    variable_list apply(variable_list &&grads) override
    {
        int mask = 0;
        for (int i = 0; i < 4; ++i)
            if (task_should_compute_output(i)) mask |= 1 << i;
        const bool create_graph = at::GradMode::is_enabled();
        variable_list list(4);
        if (!mask || !grads[0].defined()) return list;
        {
            const at::NoGradGuard no_grad;
            Tensor in, w, b, r;
            {
                std::lock_guard<std::mutex> lock(mutex);
                in = x.unpack();
                w = weight.unpack();
                b = bias.unpack();
                r = residual.unpack();
            }
            std::vector<Tensor> g = run_pointwise_backward(in, w, b, r, grads[0], shape, mask);
            for (int i = 0; i < 4; ++i) list[i] = std::move(g[i]);
        }
        return once_differentiable(std::move(list), create_graph, "pointwise_conv2d");
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex);
        x.reset_data();
        weight.reset_data();
        bias.reset_data();
        residual.reset_data();
    }
    std::string name() const override { return "PointwiseConvFunctionBackward"; }
};

Tensor pointwise(const Tensor &input, const Tensor &weight, const Tensor &bias, const Tensor &residual, int64_t act)
{
    const Mixing s = check_pointwise(input, weight, bias, residual, act);
    const c10::cuda::CUDAGuard guard(input.device());
    const bool wanted = wants_gradient(input, weight, bias, residual);
    Tensor x, out;
    {
        const at::NoGradGuard no_grad;
        x = dense(input, s.last);
        out = run_pointwise(x, row(weight), row(bias), dense(residual, s.last), s);
    }
    if (!wanted) return out;
    auto node = std::shared_ptr<PointwiseConvBackward>(new PointwiseConvBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(input, weight, bias, residual));
    node->x = SavedVariable(x, false);
    node->weight = SavedVariable(weight, false);
    if (s.act != BC_ACT_NONE) {
        if (bias.defined()) node->bias = SavedVariable(bias, false);
        if (residual.defined()) node->residual = SavedVariable(residual, false);
    }
    node->shape = s;
    torch::autograd::set_history(out, node);
    return out;
}

// ---- group normalisation --------------------------------------------------------------------------

struct Norm {
    int N, C, G, act;
    int64_t P;
    double eps;
    bool last;
};

Norm check_norm(const Tensor &input, const Tensor &weight, const Tensor &bias, int64_t groups, double eps, int64_t act)
{
    require_layer_tensor(input, "group_norm: input", input);
    if (input.dim() != 4) fail("group_norm: input must have 4 dimensions");
    if (groups < 1 || input.size(1) < 1 || input.size(1) % groups)
        fail("group_norm: " + std::to_string(input.size(1)) + " planes do not make " + std::to_string(groups) + " groups");
    for (const auto &[t, name] : {std::pair<const Tensor &, const char *>(weight, "weight"), {bias, "bias"}}) {
        if (!t.defined()) continue;
        require_layer_tensor(t, std::string("group_norm: ") + name, input);
        if (t.dim() != 1 || t.size(0) != input.size(1))
            fail(std::string("group_norm: ") + name + " must hold " + std::to_string(input.size(1)) + " values");
    }
    const Norm s{to_int(input.size(0)), to_int(input.size(1)), to_int(groups), activation_of(act), input.size(2) * input.size(3), eps,
                 is_last(input)};
    to_int(s.P);
    return s;
}

Tensor run_norm(const Tensor &x, const Tensor &weight, const Tensor &bias, const Norm &s, Tensor *stats)
{
    Tensor out = new_maps(x.sizes(), s.last, x), ws;
    if (stats) *stats = new_tensor({s.N, s.G, 2}, at::kFloat, x);
    const int kind = io_kind(x.scalar_type());
    const size_t bytes = bc_group_norm_forward_workspace(kind, s.N, s.C, s.P, s.G, s.last);
    if (bytes) ws = new_workspace(bytes, x);
    check_status(bc_group_norm_forward(ptr(x), ptr(weight), ptr(bias), out.data_ptr(), stats ? stats->data_ptr<float>() : nullptr, kind, s.N,
                                       s.C, s.P, s.G, (float)s.eps, s.last, s.act, out_ptr(ws), bytes, current_stream(x)),
                 "group_norm");
    return out;
}

std::vector<Tensor> run_norm_backward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &stats,
                                      const Tensor &grad_output, const Norm &s, int mask)
{
    std::vector<Tensor> g(3);
    if (!mask) return g;
    require_layer_tensor(grad_output, "group_norm: grad_output", x);
    if (grad_output.sizes() != x.sizes()) fail("group_norm: grad_output must have the output's shape");
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor grad = dense(grad_output, s.last), w = row(weight), b = row(bias);
    if (mask & BC_NEED_GN_INPUT) g[0] = new_maps(x.sizes(), s.last, x);
    if (mask & BC_NEED_GN_WEIGHT) g[1] = new_tensor({s.C}, x.scalar_type(), x);
    if (mask & BC_NEED_GN_BIAS) g[2] = new_tensor({s.C}, x.scalar_type(), x);
    const int kind = io_kind(x.scalar_type());
    const size_t bytes = bc_group_norm_backward_workspace(kind, s.N, s.C, s.P, s.G, s.last);
    Tensor ws;
    if (bytes) ws = new_workspace(bytes, x);
    check_status(bc_group_norm_backward(ptr(x), ptr(w), ptr(b), stats.const_data_ptr<float>(), ptr(grad), kind, s.N, s.C, s.P, s.G, s.last, s.act,
                                        mask, out_ptr(g[0]), out_ptr(g[1]), out_ptr(g[2]), out_ptr(ws), bytes, current_stream(x)),
                 "group_norm backward");
    return g;
}

struct GroupNormBackward : torch::autograd::Node {
    SavedVariable x, weight, bias, stats;
    Norm shape;
    std::mutex mutex;

    variable_list apply(variable_list &&grads) override
    {
        int mask = 0;
        for (int i = 0; i < 3; ++i)
            if (task_should_compute_output(i)) mask |= 1 << i;
        const bool create_graph = at::GradMode::is_enabled();
        variable_list list(3);
        if (!mask || !grads[0].defined()) return list;
        {
            const at::NoGradGuard no_grad;
            Tensor in, w, b, st;
            {
                std::lock_guard<std::mutex> lock(mutex);
                in = x.unpack();
                w = weight.unpack();
                b = bias.unpack();
                st = stats.unpack();
            }
            std::vector<Tensor> g = run_norm_backward(in, w, b, st, grads[0], shape, mask);
            for (int i = 0; i < 3; ++i) list[i] = std::move(g[i]);
        }
        return once_differentiable(std::move(list), create_graph, "group_norm");
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex);
        x.reset_data();
        weight.reset_data();
        bias.reset_data();
        stats.reset_data();
    }
    std::string name() const override { return "GroupNormFunctionBackward"; }
};

Tensor group_norm(const Tensor &input, const Tensor &weight, const Tensor &bias, int64_t groups, double eps, int64_t act)
{
    const Norm s = check_norm(input, weight, bias, groups, eps, act);
    const c10::cuda::CUDAGuard guard(input.device());
    const bool wanted = wants_gradient(input, weight, bias);
    Tensor x, out, stats;
    {
        const at::NoGradGuard no_grad;
        x = dense(input, s.last);
        out = run_norm(x, row(weight), row(bias), s, wanted ? &stats : nullptr);
    }
    if (!wanted) return out;
    auto node = std::shared_ptr<GroupNormBackward>(new GroupNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(input, weight, bias));
    node->x = SavedVariable(x, false);
    node->stats = SavedVariable(stats, false);
    if (weight.defined()) node->weight = SavedVariable(weight, false);
    if (bias.defined() && s.act != BC_ACT_NONE) node->bias = SavedVariable(bias, false);
    node->shape = s;
    torch::autograd::set_history(out, node);
    return out;
}

// ---- CPython entry points

// pointwise(input, weight, bias, residual, activation) -> output or NotImplemented
PyObject *py_pointwise(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Args a(v, n, 5);
    const Tensor input = a.tensor("input"), weight = a.tensor("weight"), bias = a.optional_tensor("bias"),
                 residual = a.optional_tensor("residual");
    const int64_t act = a.integer();
    if (needs_python_class(input, weight, bias, residual)) Py_RETURN_NOTIMPLEMENTED;
    Tensor out;
    {
        py::gil_scoped_release release;
        out = pointwise(input, weight, bias, residual, act);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// The two halves of the Python class.
PyObject *py_pointwise_forward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Args a(v, n, 5);
    const Tensor input = a.tensor("input"), weight = a.tensor("weight"), bias = a.optional_tensor("bias"),
                 residual = a.optional_tensor("residual");
    const int64_t act = a.integer();
    Tensor out;
    {
        py::gil_scoped_release release;
        at::NoGradGuard no_grad;
        {
            at::tracer::impl::NoTracerDispatchMode no_tracer;
            out = pointwise(input, weight, bias, residual, act);
        }
        out = seen_by_trace(out);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// pointwise_backward(input, weight, bias, residual, grad_output, activation, need_mask) -> four gradients or None
PyObject *py_pointwise_backward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Args a(v, n, 7);
    const Tensor input = a.tensor("input"), weight = a.tensor("weight"), bias = a.optional_tensor("bias"),
                 residual = a.optional_tensor("residual"), grad = a.tensor("grad_output");
    const int64_t act = a.integer();
    const int mask = (int)a.integer() & 15;
    std::vector<Tensor> g;
    {
        py::gil_scoped_release release;
        at::NoGradGuard no_grad;
        const Mixing s = check_pointwise(input, weight, bias, residual, act);
        g = run_pointwise_backward(dense(input, s.last), weight, bias, residual, grad, s, mask);
    }
    return wrap_list(g);
    END_HANDLE_TH_ERRORS
}

// group_norm(input, weight, bias, groups, eps, activation) -> output or NotImplemented
PyObject *py_group_norm(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Args a(v, n, 6);
    const Tensor input = a.tensor("input"), weight = a.optional_tensor("weight"), bias = a.optional_tensor("bias");
    const int64_t groups = a.integer();
    const double eps = a.number();
    const int64_t act = a.integer();
    if (needs_python_class(input, weight, bias)) Py_RETURN_NOTIMPLEMENTED;
    Tensor out;
    {
        py::gil_scoped_release release;
        out = group_norm(input, weight, bias, groups, eps, act);
    }
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// The two halves of the Python class: group_norm_forward(arguments of group_norm) -> [output, statistics]
PyObject *py_group_norm_forward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Args a(v, n, 6);
    const Tensor input = a.tensor("input"), weight = a.optional_tensor("weight"), bias = a.optional_tensor("bias");
    const int64_t groups = a.integer();
    const double eps = a.number();
    const int64_t act = a.integer();
    Tensor out, stats;
    {
        py::gil_scoped_release release;
        at::NoGradGuard no_grad;
        {
            at::tracer::impl::NoTracerDispatchMode no_tracer;
            const Norm s = check_norm(input, weight, bias, groups, eps, act);
            const c10::cuda::CUDAGuard guard(input.device());
            out = run_norm(dense(input, s.last), row(weight), row(bias), s, &stats);
        }
        out = seen_by_trace(out);
    }
    return wrap_list({out, stats});
    END_HANDLE_TH_ERRORS
}

// group_norm_backward(input, weight, bias, statistics, grad_output, groups, activation, need_mask) -> three gradients or None
PyObject *py_group_norm_backward(PyObject *, PyObject *const *v, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    Args a(v, n, 8);
    const Tensor input = a.tensor("input"), weight = a.optional_tensor("weight"), bias = a.optional_tensor("bias"),
                 stats = a.tensor("statistics"), grad = a.tensor("grad_output");
    const int64_t groups = a.integer(), act = a.integer();
    const int mask = (int)a.integer() & 7;
    std::vector<Tensor> g;
    {
        py::gil_scoped_release release;
        at::NoGradGuard no_grad;
        const Norm s = check_norm(input, weight, bias, groups, 0., act);
        if (!stats.is_cuda() || stats.scalar_type() != at::kFloat || stats.device() != input.device() || !stats.is_contiguous() ||
            stats.sizes() != at::IntArrayRef({s.N, s.G, 2}))
            fail("group_norm: statistics are not those of this input");
        g = run_norm_backward(dense(input, s.last), weight, bias, stats, grad, s, mask);
    }
    return wrap_list(g);
    END_HANDLE_TH_ERRORS
}

}  // namespace

#define BC_FAST(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}
PyMethodDef layer_methods[] = {BC_FAST(pointwise), BC_FAST(pointwise_forward), BC_FAST(pointwise_backward), BC_FAST(group_norm),
                               BC_FAST(group_norm_forward), BC_FAST(group_norm_backward), {nullptr, nullptr, 0, nullptr}};
