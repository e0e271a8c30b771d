"""The layers around a box convolution, as far as they need no GPU: parameters and their initial values (checkpoints of
nn.Conv2d and nn.GroupNorm load unchanged), refusals, argument checks of the C ABI."""
import pytest
import torch

import box_convolution as bc
from box_convolution import _cabi

lib = _cabi.lib
F32, F16, BF16 = 0, 1, 2


@pytest.mark.parametrize("bias", [True, False])
def test_pointwise_parameters_are_those_of_a_convolution(bias):
    torch.manual_seed(4)
    ref = torch.nn.Conv2d(12, 7, 1, bias=bias)
    torch.manual_seed(4)
    m = bc.PointwiseConv2d(12, 7, bias=bias)
    assert list(m.state_dict()) == list(ref.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(m.state_dict().values(), ref.state_dict().values()))
    m.load_state_dict(ref.state_dict())
    assert (m.in_planes, m.out_planes, m.activation) == (12, 7, None)


@pytest.mark.parametrize("affine", [True, False])
def test_norm_parameters_are_those_of_a_group_norm(affine):
    ref = torch.nn.GroupNorm(3, 12, affine=affine)
    m = bc.GroupNorm2d(3, 12, affine=affine, activation="silu")
    assert list(m.state_dict()) == list(ref.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(m.state_dict().values(), ref.state_dict().values()))
    assert (m.num_groups, m.num_planes, m.eps, m.activation) == (3, 12, 1e-5, "silu")
    m.reset_parameters()


def test_constructors_refuse_what_cannot_be():
    with pytest.raises(ValueError, match="activation"):
        bc.PointwiseConv2d(4, 4, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        bc.GroupNorm2d(2, 4, activation=torch.relu)
    for groups, planes in ((3, 4), (0, 4), (8, 4), (2, 0)):
        with pytest.raises(ValueError, match="groups"):
            bc.GroupNorm2d(groups, planes)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 5, 5)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        bc.pointwise_conv2d(x, torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        bc.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        bc.PointwiseConv2d(4, 3)(x)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        bc.GroupNorm2d(2, 4)(x)
    with pytest.raises(ValueError, match="activation"):
        bc.pointwise_conv2d(x, torch.zeros(3, 4), activation="softplus")
    with pytest.raises(TypeError):
        bc.group_norm(x.numpy(), 2)


def test_pointwise_entry_points_check_their_arguments():
    f, b, q = lib.bc_pointwise_forward, lib.bc_pointwise_backward, lib.bc_pointwise_backward_workspace
    none = [None] * 5
    assert f(*none, F32, 0, 4, 4, 9, 0, 0, None) == 0          # nothing to do
    assert f(*none, F32, 2, 4, 0, 9, 0, 0, None) == 0
    assert f(*none, F32, 2, 4, 4, 0, 0, 0, None) == 0
    assert f(*none, F32, 2, 4, 4, 9, 0, 0, None) == -1
    assert f(*none, F32, -1, 4, 4, 9, 0, 0, None) == -2
    assert f(*none, F32, 2, 4, 4, 1 << 33, 0, 0, None) == -2
    assert f(*none, F32, 1 << 30, 1 << 10, 4, 1 << 30, 0, 0, None) == -2
    assert f(*none, 3, 2, 4, 4, 9, 0, 0, None) == -5
    assert f(*none, F32, 2, 4, 4, 9, 0, 4, None) == -5
    assert b(*none, F32, 2, 4, 4, 9, 0, 0, 0, *[None] * 5, 0, None) == 0          # no gradient asked for
    assert b(*none, F32, 2, 4, 4, 9, 0, 0, 8, *[None] * 5, 0, None) == 0          # without an activation it is grad_output
    assert b(*none, F32, 2, 4, 4, 9, 0, 0, 1, *[None] * 5, 0, None) == -1
    one = 256       # (an address that is never followed: the checks come first)
    assert b(one, one, None, None, one, F32, 2, 4, 4, 9, 0, 0, 2, None, one, None, None, None, 0, None) == -3
    assert q(F32, 2, 4, 4, 9, 0, 0, 2) > 0 and q(F32, 2, 4, 4, 9, 0, 0, 0) == 0
    assert q(F32, 0, 4, 4, 9, 0, 0, 15) == 0 and q(9, 2, 4, 4, 9, 0, 0, 15) == 0


def test_norm_entry_points_check_their_arguments():
    f, b, q = lib.bc_group_norm_forward, lib.bc_group_norm_backward, lib.bc_group_norm_backward_workspace
    none = [None] * 5
    assert f(*none, BF16, 0, 4, 9, 2, 1e-5, 0, 0, None, 0, None) == 0
    assert f(*none, BF16, 2, 0, 9, 1, 1e-5, 0, 0, None, 0, None) == 0
    assert f(*none, BF16, 2, 4, 9, 2, 1e-5, 0, 0, None, 0, None) == -1
    assert f(*none, BF16, 2, 4, 9, 3, 1e-5, 0, 0, None, 0, None) == -2
    assert f(*none, BF16, 2, 4, 9, 0, 1e-5, 0, 0, None, 0, None) == -2
    assert f(*none, BF16, 2, 4, -9, 2, 1e-5, 0, 0, None, 0, None) == -2
    assert f(*none, 7, 2, 4, 9, 2, 1e-5, 0, 0, None, 0, None) == -5
    assert f(*none, BF16, 2, 4, 9, 2, 1e-5, 0, -1, None, 0, None) == -5
    assert b(*none, F16, 2, 4, 9, 2, 0, 0, 0, None, None, None, None, 0, None) == 0
    assert b(*none, F16, 2, 4, 9, 2, 0, 0, 1, None, None, None, None, 0, None) == -1
    one = 256
    assert b(one, None, None, one, one, F16, 2, 4, 9, 2, 0, 0, 1, one, None, None, None, 0, None) == -3
    assert q(F16, 2, 4, 9, 2, 0) > 0 and q(F16, 0, 4, 9, 2, 0) == 0
