"""pointwise_conv2d and group_norm where values, sums or strides are unusual: slopes that enter products, groups far from zero,
tails of SiLU and GELU, very long sums and exact ones, layouts of gradients.  Definitions in 64 bits and tolerances as in test_gpu_layers.py."""
import math

import pytest
import torch

from test_gpu_layers import DTYPES, FN, TINY, U, act64, bc, check_norm, maps, same_layout, slope64, slope_error, within  # noqa: F401

pytestmark = pytest.mark.gpu

LAYOUTS = pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
NARROW = [torch.float16, torch.bfloat16]


# ---- products of a slope ---------------------------------------------------------------------------------

# one product a value, tiles of TMA (several slices of channels, one CTA an SM and two), rows that it does not take, weights
# that only multiply-adds hold (of grad_input; of the slope)
SLOPES = [(2, 8, 1, 4, 6), (2, 1, 1, 5, 7), (2, 16, 24, 8, 16), (1, 256, 72, 8, 16), (1, 64, 200, 9, 16), (2, 17, 33, 3, 43), (1, 60, 130, 7, 9),
          (1, 40, 2500, 4, 8), (1, 41, 2500, 3, 7), (1, 4609, 24, 3, 7), (300, 24, 40, 1, 1)]


@LAYOUTS
@pytest.mark.parametrize("dtype", NARROW, ids=str)
@pytest.mark.parametrize("shape", SLOPES, ids=str)
def test_a_slope_enters_its_products_unrounded(bc, shape, dtype, last):  # noqa: F811
    """dz = grad * slope is not rounded to the tensors' type before grad_input, grad_weight and grad_bias are made of it: it
    is held in two parts of that type, the second a rounding of u of what the first leaves (u |dz|)."""
    N, Ci, Co, h, w = shape
    u, gen = U[dtype], torch.Generator(device="cuda").manual_seed(Ci + Co)
    for act in ("silu", "gelu", "relu"):
        x, r, g = maps(gen, (N, Ci, h, w), dtype, last), maps(gen, (N, Co, h, w), dtype, last), maps(gen, (N, Co, h, w), dtype, last)
        weight = (torch.randn(Co, Ci, device="cuda", generator=gen) / math.sqrt(Ci)).to(dtype)
        bias = torch.randn(Co, device="cuda", generator=gen).to(dtype)
        X, W = x.double().permute(0, 2, 3, 1).reshape(-1, Ci), weight.double()
        R, G = (t.double().permute(0, 2, 3, 1).reshape(-1, Co) for t in (r, g))
        z = X @ W.T + bias.double() + R
        dz_arg = (Ci + 2) * 2.0 ** -23 * (X.abs() @ W.abs().T + bias.double().abs() + R.abs())
        dz = G * slope64(z, act)
        near = G.abs() * slope_error(z, dz_arg, act) + 2.0 ** -23 * dz.abs()
        off = near + u * u * dz.abs() + TINY[dtype]
        # two parts in every product: twice the additions
        rows, size = X.shape[0], dz.abs() + off
        planes = lambda t: t.reshape(N, h, w, -1).permute(0, 3, 1, 2)  # noqa: E731
        for of_residual in (True, False):      # (dz is the residual's gradient as well, or nobody's)
            leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
            rr = r.detach().requires_grad_(of_residual)
            out = bc.pointwise_conv2d(*leaves, activation=act, residual=rr)
            got = torch.autograd.grad(out, leaves + [rr] * of_residual, g)
            within(got[0], planes(dz @ W), planes(off @ W.abs() + (2 * Co + 2) * 2.0 ** -23 * (size @ W.abs())), dtype, "grad_input")
            within(got[1], dz.T @ X, off.T @ X.abs() + (2 * rows + 2) * 2.0 ** -23 * (size.T @ X.abs()), dtype, "grad_weight")
            within(got[2], dz.sum(0), off.sum(0) + (2 * rows + 2) * 2.0 ** -23 * size.sum(0), dtype, "grad_bias")
            if of_residual:
                within(got[3], planes(dz), planes(near), dtype, "grad_residual")


# ---- groups far from zero --------------------------------------------------------------------------------

@LAYOUTS
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(2, 8, 2, 8, 8), (2, 8, 8, 8, 8), (1, 64, 16, 2, 2), (1, 16, 1, 1, 3), (3, 24, 3, 5, 7), (1, 32, 1, 64, 96),
                                   (1, 8, 1, 250, 251), (2, 20, 4, 16, 24), (1, 2048, 2, 1, 3)], ids=str)
def test_norm_of_groups_whose_squares_are_near_the_largest(bc, shape, dtype, last):  # noqa: F811
    """Means of 1e19 with a spread of 1e17, of either sign: mean^2 times a few values is no float, the sum of squares about the
    mean is.  Lanes, warps and CTAs without a value take part in such a group as well."""
    N, C, G, h, w = shape
    gen = torch.Generator(device="cuda").manual_seed(3)
    g = maps(gen, (N, C, h, w), dtype, last)
    for sign in (1.0, -1.0):
        x = maps(gen, (N, C, h, w), dtype, last, 1e17, sign * 1e19)
        check_norm(bc, x, G, None, None, g, "silu" if sign > 0 else None)
    # one value far off among many
    x = maps(gen, (N, C, h, w), dtype, last)
    x[0, 0, 0, 0] = 1e18
    check_norm(bc, x, G, None, None, g, None)


# ---- SiLU far below zero ---------------------------------------------------------------------------------

SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}      # steps of subnormal numbers


def close(got, ref, relative, what):
    """Within a relative error, and a step of the type's smallest numbers."""
    off, bound = (got.double() - ref).abs(), relative * ref.abs() + 1.01 * SMALLEST[got.dtype]
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d; first %r instead of %r" % (what, int(bad.sum()), bad.numel(), float(got[bad][0]), float(ref[bad][0]))


@LAYOUTS
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("count", [512, 509])
def test_silu_keeps_its_tails(bc, dtype, last, count):  # noqa: F811
    """z from -104 to 104, relative errors of value and slope: sigmoid(z) is a normal number down to -87.3 and z sigmoid(z) to
    -91.8.  float: half a step of its own, 2^-24, in each of the dozen operations, 2^-22 in the power of two: 2^-20.  16-bit: u,
    that, and an exponent z log2(e) of at most 151 that is rounded to half of 2^-16, times log(2): 2^-17."""
    z = torch.linspace(-104, 104, count, device="cuda").to(dtype)
    ref, slope = act64(z.double(), "silu"), slope64(z.double(), "silu")
    # what is there of a slope near its zero (-1.278): the error of its argument, none, and of its terms
    parts = torch.sigmoid(z.double()) * (1 + z.double().abs() * torch.sigmoid(-z.double()))
    tol = FN + (U[dtype] + 2.0 ** -17 if dtype != torch.float32 else 0)
    # z as a residual, and its slope as the residual's gradient
    shape = (1, 8, count, 1) if not last else (1, 8, 1, count)
    r = z.view(shape[2:]).expand(shape).contiguous(memory_format=torch.channels_last if last else torch.contiguous_format).requires_grad_()
    x, w = torch.zeros(1, 8, *shape[2:], device="cuda", dtype=dtype), torch.zeros(8, 8, device="cuda", dtype=dtype)
    out = bc.pointwise_conv2d(x.contiguous(memory_format=torch.channels_last) if last else x, w, activation="silu", residual=r)
    close(out[0].flatten(1), ref.expand(8, -1), tol, "pointwise")
    grad = torch.autograd.grad(out, r, torch.ones_like(out))[0]
    assert ((grad[0].flatten(1).double() - slope).abs() <= tol * parts + 1.01 * SMALLEST[dtype]).all()
    # z as a normalisation's bias, and its slope as the gradient of that
    x = torch.randn(1, count, 1, 1, device="cuda").to(dtype)
    for gx in (x, x.expand(1, count, 1, 9).contiguous(memory_format=torch.channels_last if last else torch.contiguous_format)):
        b = z.clone().requires_grad_()
        out = bc.group_norm(gx, 1, torch.zeros_like(z), b, activation="silu")
        close(out[0].flatten(1), ref[:, None].expand(-1, gx.shape[3]), tol, "group_norm")
        g = torch.zeros_like(out)
        g[..., 0] = 1
        grad = torch.autograd.grad(out, b, g)[0]
        assert ((grad.double() - slope).abs() <= tol * parts + 1.01 * SMALLEST[dtype]).all()


# ---- GELU far below zero ---------------------------------------------------------------------------------

@LAYOUTS
@pytest.mark.parametrize("dtype", NARROW, ids=str)
@pytest.mark.parametrize("count", [512, 509])
def test_gelu_of_16_bits_keeps_its_tails(bc, dtype, last, count):  # noqa: F811
    """z from -13 to 13, where z times the normal distribution function is a normal number of bfloat16, relative errors of value and
    slope: u, 2^-13 of the function, and an argument z^2 / 2 of the exponential that is rounded to half a step, which moves it by up
    to z^2 2^-24 relatively, twice that with a dozen other steps."""
    z = torch.linspace(-13, 13, count, device="cuda").to(dtype)
    Z = z.double()
    P, density = 0.5 * torch.erfc(-Z / math.sqrt(2)), torch.exp(-0.5 * Z * Z) / math.sqrt(2 * math.pi)
    ref, slope, parts = Z * P, P + Z * density, P + Z.abs() * density
    tol = 2.0 ** -23 * (Z * Z + 16) + U[dtype] + 2.0 ** -13
    shape = (1, 8, count, 1) if not last else (1, 8, 1, count)
    layout = torch.channels_last if last else torch.contiguous_format
    r = z.view(shape[2:]).expand(shape).contiguous(memory_format=layout).requires_grad_()
    x, w = torch.zeros(1, 8, *shape[2:], device="cuda", dtype=dtype).contiguous(memory_format=layout), torch.zeros(8, 8, device="cuda", dtype=dtype)
    out = bc.pointwise_conv2d(x, w, activation="gelu", residual=r)
    close(out[0].flatten(1), ref.expand(8, -1), tol, "pointwise")
    grad = torch.autograd.grad(out, r, torch.ones_like(out))[0]
    assert ((grad[0].flatten(1).double() - slope).abs() <= tol * parts + 1.01 * SMALLEST[dtype]).all()
    x = torch.randn(1, count, 1, 1, device="cuda").to(dtype)
    for gx in (x, x.expand(1, count, 1, 9).contiguous(memory_format=layout)):
        b = z.clone().requires_grad_()
        out = bc.group_norm(gx, 1, torch.zeros_like(z), b, activation="gelu")
        close(out[0].flatten(1), ref[:, None].expand(-1, gx.shape[3]), tol[:, None], "group_norm")
        g = torch.zeros_like(out)
        g[..., 0] = 1
        grad = torch.autograd.grad(out, b, g)[0]
        assert ((grad.double() - slope).abs() <= tol * parts + 1.01 * SMALLEST[dtype]).all()


# ---- exact sums over many pixels -------------------------------------------------------------------------

@LAYOUTS
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 24, 40, 311, 328), (2, 25, 37, 311, 331), (1, 264, 136, 161, 168), (3, 130, 20, 101, 171)], ids=str)
def test_sums_of_whole_numbers_are_exact(bc, shape, act, dtype, last):  # noqa: F811
    """Small whole numbers, whose sums are exact in any order: a slice of pixels that is lost or taken twice shows, with some
    twenty slices and more for every partial sum (rings go round several times)."""
    N, Ci, Co, h, w = shape
    gen = torch.Generator(device="cuda").manual_seed(Ci)

    def whole(size, most):
        t = torch.randint(-most, most + 1, size, device="cuda", generator=gen).to(dtype)
        return t.contiguous(memory_format=torch.channels_last if last else torch.contiguous_format) if len(size) == 4 else t

    x, g = whole((N, Ci, h, w), 2).requires_grad_(), whole((N, Co, h, w), 2)
    weight, bias = whole((Co, Ci), 1).requires_grad_(), (whole((Co,), 3) + 0.5).requires_grad_()
    out = bc.pointwise_conv2d(x, weight, bias, activation=act)
    got = torch.autograd.grad(out, (x, weight, bias), g)
    X, G = (t.detach().double().permute(0, 2, 3, 1).reshape(-1, t.shape[1]) for t in (x, g))
    z = X @ weight.detach().double().T + bias.detach().double()
    dz = G * (z > 0) if act else G
    planes = lambda t: t.reshape(N, h, w, -1).permute(0, 3, 1, 2)  # noqa: E731
    for name, a, b in (("out", out, planes(act64(z, act))), ("grad_input", got[0], planes(dz @ weight.detach().double())),
                       ("grad_weight", got[1], dz.T @ X), ("grad_bias", got[2], dz.sum(0))):
        assert torch.equal(a, b.to(dtype)), name


# ---- long sums of one sign -------------------------------------------------------------------------------

@LAYOUTS
@pytest.mark.parametrize("shape, dtype", [((1, 16, 16, 2048, 2048), torch.float32), ((1, 1, 1, 8192, 8192), torch.float32), ((1, 3, 2, 4001, 4003), torch.float32),
                                          ((1, 8, 8, 8192, 4096), torch.float16), ((1, 3, 5, 4096, 4099), torch.float16), ((1, 8, 8, 4096, 4096), torch.bfloat16)], ids=str)
def test_sums_of_millions_of_one_sign(bc, shape, dtype, last):  # noqa: F811
    """An accumulator's additions round towards zero, so what they lose of a sum of one sign adds up: it must not grow with the
    pixels.  n additions that are each off by less than a step of a sum that grows evenly lose less than n / 2 steps of 2^-23.  A
    sum in an accumulator is of 128 additions at most (16-bit tensors 512): 2^-17 (2^-15).  16 (64) of those make a row, rounded
    to nearest, half a step: 2^-21 (2^-19), and the rows are added in double.  grad_bias: 256 (512) additions, 8 (64) of or in
    those, up to 64 threads' in order, rounded to nearest: less than 2^-16 (2^-14)."""
    N, Ci, Co, h, w = shape
    gen = torch.Generator(device="cuda").manual_seed(1)
    layout = torch.channels_last if last else torch.contiguous_format
    x = torch.empty(N, Ci, h, w, device="cuda", dtype=dtype, memory_format=layout).uniform_(0.5, 1.5, generator=gen)
    g = torch.empty(N, Co, h, w, device="cuda", dtype=dtype, memory_format=layout).uniform_(0.5, 1.5, generator=gen)
    weight, bias = torch.zeros(Co, Ci, device="cuda", dtype=dtype).requires_grad_(), torch.zeros(Co, device="cuda", dtype=dtype).requires_grad_()
    # (16-bit: an eighth of a small power of two, so that sums of 2^25 are in float16's range)
    scale = 2.0 ** -12 if dtype == torch.float16 else 1.0
    g = g * scale
    out = bc.pointwise_conv2d(x, weight, bias)
    gw, gb = torch.autograd.grad(out, (weight, bias), g)
    W, B = torch.zeros(Co, Ci, device="cuda").double(), torch.zeros(Co, device="cuda").double()
    for rows in range(0, h, 256):
        X, G = x[0, :, rows:rows + 256].double().flatten(1), g[0, :, rows:rows + 256].double().flatten(1)
        W += G @ X.T
        B += G.sum(1)
    once = 0 if dtype == torch.float32 else U[dtype]
    tol = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -14 + 2.0 ** -18
    assert float(((gw.double() - W).abs() / W).max()) <= once + tol
    assert float(((gb.double() - B).abs() / B).max()) <= once + tol


# ---- layouts ---------------------------------------------------------------------------------------------

@LAYOUTS
@pytest.mark.parametrize("act", [None, "silu"])
def test_every_gradient_has_the_inputs_layout(bc, act, last):  # noqa: F811
    x, r = (maps(torch.Generator(device="cuda").manual_seed(s), (2, c, 6, 10), torch.float32, last).requires_grad_() for s, c in ((1, 24), (2, 40)))
    w = torch.randn(40, 24, device="cuda")
    other = torch.contiguous_format if last else torch.channels_last
    for g in (torch.randn(2, 40, 6, 10, device="cuda").contiguous(memory_format=other), torch.randn(1, 40, 1, 1, device="cuda").expand(2, 40, 6, 10),
              torch.randn(2, 40, 10, 6, device="cuda").transpose(2, 3)):
        for leaves in ((x, r), (r,)):
            got = torch.autograd.grad(bc.pointwise_conv2d(x, w, activation=act, residual=r), leaves, g)
            assert all(same_layout(t, last) for t in got)
            if act is None:
                assert torch.equal(got[-1], g)


def test_no_wait_has_expired():
    from box_convolution import _cabi
    assert _cabi.wait_timeouts() == 0
