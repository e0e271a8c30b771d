"""The layers around a box convolution.

``BoxConv2d`` filters every plane by itself.  What mixes the planes and keeps their scale stands around it, as in the
reference's ``BottleneckBoxConv`` (``examples/Cityscapes/models/ENet.py:282-304``): a 1 x 1 convolution in front of it,
normalisations with an activation, a skip connection.  Here are those two operators with their neighbours folded in, for
training and inference:

``pointwise_conv2d`` / ``PointwiseConv2d``   ``act(weight x + bias + residual)`` per pixel, in one pass over the pixels;
``group_norm`` / ``GroupNorm2d``             ``act(weight (x - mean) / sqrt(var + eps) + bias)``, statistics per sample and
group of planes, so that a step does not depend on how the batch is sharded.

Inputs are float32, float16 or bfloat16, all tensors of a call alike, ``(N, C, h, w)`` in planes (contiguous: what a box
convolution reads and writes) or channels last; outputs and gradients come in the input's layout.  Tensors of other
strides are copied first.  The fastest kernels want arrays on 16 bytes, 16-bit convolutions also rows of a multiple of 16 bytes; a
normalisation of a view that starts elsewhere (or, channels last, of channels that take more than 1024 vectors of 16 bytes to
repeat their place in one) runs value by value, many times slower.  Sums, statistics and activations are float32 whatever the type, results are rounded once (a
16-bit gradient through an activation enters its products as two values of that type, off by 2^-16 or 2^-22 of it).  Results
are the same bits from call to call.  Activations: None, "relu", "silu", "gelu" (the one with the error function).  The backward pass computes the
activation's argument again from what the forward pass was given: nothing but the inputs is kept (and two
statistics a group).  Gradients of gradients are refused.
"""
import math

import torch

from . import _torch_binding as _native

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _activation(name):
    try:
        return _ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError("box_convolution: activation must be None, 'relu', 'silu' or 'gelu', got %r" % (name,)) from None


class PointwiseConvFunction(torch.autograd.Function):
    """What ``pointwise_conv2d`` calls inside a trace, a function transform or forward-mode differentiation; ordinary calls
    get a node of the same name in C++."""

    @staticmethod
    def forward(ctx, input, weight, bias, residual, activation):
        ctx.save_for_backward(input, weight, bias, residual)
        ctx.activation = activation
        return _native.pointwise_forward(input, weight, bias, residual, activation)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        mask = sum(1 << i for i, needed in enumerate(ctx.needs_input_grad[:4]) if needed)
        return (*_native.pointwise_backward(*ctx.saved_tensors, grad_output, ctx.activation, mask), None)


class GroupNormFunction(torch.autograd.Function):
    """What ``group_norm`` calls inside a trace, a function transform or forward-mode differentiation; ordinary calls get a
    node of the same name in C++."""

    @staticmethod
    def forward(ctx, input, weight, bias, num_groups, eps, activation):
        out, stats = _native.group_norm_forward(input, weight, bias, num_groups, eps, activation)
        ctx.save_for_backward(input, weight, bias, stats)
        ctx.options = num_groups, activation
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        mask = sum(1 << i for i, needed in enumerate(ctx.needs_input_grad[:3]) if needed)
        return (*_native.group_norm_backward(*ctx.saved_tensors, grad_output, *ctx.options, mask), None, None, None)


def pointwise_conv2d(input, weight, bias=None, *, activation=None, residual=None):
    """``out[n, o, y, x] = act(sum_i weight[o, i] * input[n, i, y, x] + bias[o] + residual[n, o, y, x])``.

    weight    ``(out_planes, in_planes)``, or with two more sizes of 1 as ``nn.Conv2d`` has it;
    bias      ``out_planes`` values or None;
    residual  tensor of the output's shape or None, inside the activation as in ``fused_box_block``.
    """
    act = _activation(activation)
    out = _native.pointwise(input, weight, bias, residual, act)
    if out is NotImplemented:
        out = PointwiseConvFunction.apply(input, weight, bias, residual, act)
    return out


def group_norm(input, num_groups, weight=None, bias=None, eps=1e-5, *, activation=None):
    """``act(weight[c] * (input - mean) / sqrt(var + eps) + bias[c])``, mean and biased variance over the pixels of the
    ``C / num_groups`` adjacent planes of a sample's group.  ``weight`` and ``bias``: ``C`` values each, or None."""
    act = _activation(activation)
    out = _native.group_norm(input, weight, bias, num_groups, eps, act)
    if out is NotImplemented:
        out = GroupNormFunction.apply(input, weight, bias, num_groups, eps, act)
    return out


class PointwiseConv2d(torch.nn.Module):
    """``pointwise_conv2d`` with its parameters, which have the names, shapes and initial values of those of
    ``nn.Conv2d(in_planes, out_planes, 1)``: checkpoints load unchanged.  ``activation`` may be changed later."""

    def __init__(self, in_planes, out_planes, bias=True, activation=None):
        super().__init__()
        _activation(activation)
        self.in_planes, self.out_planes, self.activation = in_planes, out_planes, activation
        self.weight = torch.nn.Parameter(torch.empty(out_planes, in_planes, 1, 1))
        self.register_parameter("bias", torch.nn.Parameter(torch.empty(out_planes)) if bias else None)
        self.reset_parameters()

    def reset_parameters(self):
        bound = 1 / math.sqrt(max(1, self.in_planes))
        torch.nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            torch.nn.init.uniform_(self.bias, -bound, bound)

    def forward(self, input, residual=None):
        return pointwise_conv2d(input, self.weight, self.bias, activation=self.activation, residual=residual)

    def extra_repr(self):
        return "%d, %d, bias=%s, activation=%r" % (self.in_planes, self.out_planes, self.bias is not None, self.activation)


class GroupNorm2d(torch.nn.Module):
    """``group_norm`` with its parameters, which have the names, shapes and initial values of those of
    ``nn.GroupNorm(num_groups, num_planes)``: checkpoints load unchanged.  ``activation`` and ``eps`` may be changed later."""

    def __init__(self, num_groups, num_planes, eps=1e-5, affine=True, activation=None):
        super().__init__()
        _activation(activation)
        if num_groups < 1 or num_planes < 1 or num_planes % num_groups:
            raise ValueError("GroupNorm2d: %d planes do not make %d groups" % (num_planes, num_groups))
        self.num_groups, self.num_planes, self.eps, self.activation = num_groups, num_planes, eps, activation
        self.register_parameter("weight", torch.nn.Parameter(torch.ones(num_planes)) if affine else None)
        self.register_parameter("bias", torch.nn.Parameter(torch.zeros(num_planes)) if affine else None)

    def reset_parameters(self):
        if self.weight is not None:
            torch.nn.init.ones_(self.weight)
            torch.nn.init.zeros_(self.bias)

    def forward(self, input):
        return group_norm(input, self.num_groups, self.weight, self.bias, self.eps, activation=self.activation)

    def extra_repr(self):
        return "%d, %d, eps=%g, affine=%s, activation=%r" % (self.num_groups, self.num_planes, self.eps, self.weight is not None,
                                                            self.activation)
