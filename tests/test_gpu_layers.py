"""pointwise_conv2d and group_norm on the GPU against their definitions in 64 bits, gradients by differentiation of the
definition.

Tolerances go by element and are derived, not fitted.  u is half a step of the tensors' type (the rounding of a result), E
bounds what 32-bit arithmetic adds.  A sum of K products has an error of at most K 2^-23 times the sum of their
magnitudes, were every addition rounded by a whole step; products of 16-bit values are exact.  The functions of an
activation have relative errors of some steps: 2^-20.  An argument that is off by dz moves an activation by at most 1.13 dz
(the steepest slopes of SiLU and GELU are 1.10 and 1.13) and its slope by at most dz (their steepest are 0.5 and 0.8), or, a
ReLU's, by 1 where the argument is within dz of zero.  A 16-bit dz = grad * slope is rounded once before it enters the
products: u |dz|.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}     # half a step of the smallest numbers
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
FN = 2.0 ** -20


@pytest.fixture(scope="module")
def bc():
    import box_convolution
    assert torch.cuda.is_available()
    return box_convolution


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    return z


def slope64(z, act):
    z = z.detach().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, act).sum(), z)[0].detach()


def slope_error(z, dz, act):
    """How far a slope is off whose argument is off by dz."""
    if act is None:
        return torch.zeros_like(z)
    return (z.abs() <= dz).double() if act == "relu" else dz + FN


def maps(gen, shape, dtype, last, scale=1.0, offset=0.0):
    t = (torch.randn(*shape, device="cuda", generator=gen) * scale + offset).to(dtype)
    return t.contiguous(memory_format=torch.channels_last if last else torch.contiguous_format)


def within(got, ref, error, dtype, what):
    assert got.dtype == dtype and got.shape == ref.shape, what
    off = (got.double() - ref).abs()
    bound = U[dtype] * ref.abs() + error * (1 + U[dtype]) + TINY[dtype]
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values; worst is %.3g times its bound" % (
        what, int(bad.sum()), bad.numel(), float((off / bound.clamp_min(1e-300)).nan_to_num(1e9).max()))


def same_layout(t, last):
    return t.is_contiguous(memory_format=torch.channels_last if last else torch.contiguous_format)


# ---- pointwise -------------------------------------------------------------------------------------------

def check_pointwise(bc, x, w, b, r, g, act, train=True):
    """One call and its gradients against the definition."""
    dtype, u = x.dtype, U[x.dtype]
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, r)]
    x, w, b, r = leaves
    out = bc.pointwise_conv2d(x, w, b, activation=act, residual=r)
    X, W = x.detach().double().permute(0, 2, 3, 1), w.detach().double().reshape(w.shape[0], w.shape[1])
    z, size = X @ W.T, X.abs() @ W.T.abs()
    if b is not None:
        z, size = z + b.detach().double(), size + b.detach().double().abs()
    if r is not None:
        R = r.detach().double().permute(0, 2, 3, 1)
        z, size = z + R, size + R.abs()
    Ci, Co = x.shape[1], w.shape[0]
    dz_arg = (Ci + 2) * 2.0 ** -23 * size
    planes = lambda t: t.permute(0, 3, 1, 2)  # noqa: E731
    ref = act64(z, act)
    within(out, planes(ref), planes(1.13 * dz_arg + FN * ref.abs() + (FN * z.abs() if act == "gelu" else 0)), dtype, "out")
    if not train:
        return out
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], g)
    G = g.double().permute(0, 2, 3, 1)
    dz = G * slope64(z, act)
    off = G.abs() * slope_error(z, dz_arg, act)
    if act is not None:
        off = off + u * dz.abs() + TINY[dtype]
    rows = X.numel() // max(1, Ci) if Ci else z.numel() // max(1, Co)
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    got = dict(zip([n for n, t in zip("xwbr", leaves) if t is not None], grads))
    within(got["x"], planes(dz @ W), planes(off @ W.abs() + (Co + 2) * 2.0 ** -23 * ((dz.abs() + off) @ W.abs())), dtype, "grad_input")
    many = (rows + 2) * 2.0 ** -23
    A, OFF = flat(dz.abs() + off).T, flat(off).T
    within(got["w"], (flat(dz).T @ flat(X)).reshape(w.shape), (OFF @ flat(X).abs() + many * (A @ flat(X).abs())).reshape(w.shape), dtype, "grad_weight")
    if b is not None:
        within(got["b"], flat(dz).sum(0), OFF.sum(1) + many * A.sum(1), dtype, "grad_bias")
    if r is not None:
        within(got["r"], planes(dz), planes(off), dtype, "grad_residual")
    return out, got


# (N, Ci, Co, h, w): one of everything, sizes around tiles (16, 32, 64, 128 channels; 128 pixels), odd ones, single pixels
POINTWISE = [
    (1, 1, 1, 1, 1), (2, 3, 5, 1, 1), (300, 24, 40, 1, 1), (1, 16, 16, 1, 128), (2, 17, 33, 3, 43), (3, 64, 16, 9, 15),
    (2, 32, 128, 16, 24), (1, 128, 32, 40, 50), (2, 60, 20, 31, 37), (2, 65, 129, 11, 13), (1, 256, 256, 16, 16),
    (5, 8, 72, 7, 7), (1, 1, 64, 20, 20), (1, 64, 1, 20, 20), (2, 320, 24, 8, 16), (1, 40, 264, 10, 26), (1, 512, 320, 8, 24),
    # more tiles than CTAs, aligned and not; more input channels than shared memory holds the weights of
    (3, 72, 40, 136, 152), (2, 37, 19, 151, 203), (1, 4609, 24, 3, 7), (1, 2304, 40, 4, 10),
]


@pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", POINTWISE, ids=str)
def test_pointwise(bc, shape, dtype, last):
    N, Ci, Co, h, w = shape
    gen = torch.Generator(device="cuda").manual_seed(N * Ci + Co)
    for k, act in enumerate((None, "relu", "silu", "gelu")):
        x, g = maps(gen, (N, Ci, h, w), dtype, last), maps(gen, (N, Co, h, w), dtype, last)
        weight = (torch.randn(Co, Ci, 1, 1, device="cuda", generator=gen) / math.sqrt(Ci)).to(dtype)
        bias = torch.randn(Co, device="cuda", generator=gen).to(dtype) if k != 1 else None
        residual = maps(gen, (N, Co, h, w), dtype, last) if k % 2 else None
        out, got = check_pointwise(bc, x, weight, bias, residual, g, act)
        # (a single plane is laid out alike either way, and its strides say planes)
        assert same_layout(out, last and Ci > 1) and same_layout(got["x"], last)
        assert got["w"].is_contiguous()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_pointwise_subsets_of_gradients_have_the_bits_of_all(bc, dtype):
    gen = torch.Generator(device="cuda").manual_seed(9)
    for act, last in ((None, False), ("silu", True), ("gelu", False)):
        t = [maps(gen, (2, 24, 9, 40), dtype, last), (0.3 * torch.randn(40, 24, device="cuda", generator=gen)).to(dtype),
             torch.randn(40, device="cuda", generator=gen).to(dtype), maps(gen, (2, 40, 9, 40), dtype, last)]
        g = maps(gen, (2, 40, 9, 40), dtype, last)

        def grads(which):
            leaves = [v.detach().requires_grad_(i in which) for i, v in enumerate(t)]
            out = bc.pointwise_conv2d(*leaves[:3], activation=act, residual=leaves[3])
            return dict(zip(which, torch.autograd.grad(out, [leaves[i] for i in which], g)))

        everything = grads((0, 1, 2, 3))
        for which in ((0,), (1,), (2,), (3,), (0, 1), (1, 2), (0, 3), (2, 3)):
            for i, v in grads(which).items():
                assert torch.equal(v, everything[i]), (act, which, i)


def test_pointwise_without_pixels_planes_or_samples(bc):
    for N, Ci, Co, h, w in ((0, 4, 3, 5, 5), (2, 4, 3, 0, 5), (2, 0, 3, 4, 5), (2, 4, 0, 4, 5)):
        x = torch.randn(N, Ci, h, w, device="cuda").requires_grad_()
        weight = torch.randn(Co, Ci, device="cuda").requires_grad_()
        bias = torch.randn(Co, device="cuda").requires_grad_()
        out = bc.pointwise_conv2d(x, weight, bias, activation="silu")
        assert out.shape == (N, Co, h, w)
        ref = act64(bias.detach().double(), "silu").view(1, -1, 1, 1).expand_as(out)
        if not Ci:
            within(out, ref, FN * ref.abs(), torch.float32, "out")
        gx, gw, gb = torch.autograd.grad(out, (x, weight, bias), torch.ones_like(out))
        assert gx.shape == x.shape and gw.shape == weight.shape and gb.shape == bias.shape
        assert not gx.any() and not gw.any()
        if not N or not h:
            assert not gb.any()


# ---- group normalisation ---------------------------------------------------------------------------------

def check_norm(bc, x, G, w, b, g, act, eps=1e-5, train=True):
    dtype, (N, C, h, wd) = x.dtype, x.shape
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    out = bc.group_norm(leaves[0], G, leaves[1], leaves[2], eps, activation=act)
    X = x.double().reshape(N, G, -1)
    mean, var = X.mean(2, keepdim=True), X.var(2, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    unit = (X - mean) * rstd
    # 32 half steps of 32 bits for the statistics and each further step: of the values around the mean, whose differences
    # keep the values' own errors, and of the spread
    e_unit = FN * 2 * (rstd * (X.abs() + mean.abs() + X.abs().mean(2, keepdim=True)) + unit.abs())
    per = lambda t: t.detach().double().view(1, C, 1) if t is not None else None  # noqa: E731
    back = lambda t: t.reshape(N, C, -1)  # noqa: E731
    full = lambda t: t.reshape(N, C, h, wd)  # noqa: E731
    W, B = per(w) if w is not None else torch.ones(1, C, 1, device=x.device).double(), per(b) if b is not None else 0.0
    z = back(unit) * W + B
    dz_arg = back(e_unit) * W.abs() + FN * (back(unit).abs() * W.abs() + (B.abs() if b is not None else 0))
    ref = act64(z, act)
    within(out, full(ref), full(1.13 * dz_arg + FN * (ref.abs() + z.abs())), dtype, "out")
    if not train:
        return out
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], g)
    Gr = g.double().reshape(N, C, -1)
    dz = Gr * slope64(z, act)
    off = Gr.abs() * slope_error(z, dz_arg, act) + FN * dz.abs()
    grouped = lambda t: t.reshape(N, G, -1)  # noqa: E731
    d, do = grouped(dz * W), grouped(off * W.abs())
    avg = lambda t: t.mean(2, keepdim=True)  # noqa: E731
    dx = rstd * (d - avg(d) - unit * avg(d * unit))
    e_dx = rstd * (do + avg(do) + unit.abs() * avg(do * unit.abs()) + e_unit * avg((d * unit).abs()) + unit.abs() * avg(d.abs() * e_unit)
                   + 2 * FN * (d.abs() + avg(d.abs()) + unit.abs() * avg((d * unit).abs())))
    got = dict(zip([n for n, t in zip("xwb", leaves) if t is not None], grads))
    within(got["x"], full(dx), full(e_dx), dtype, "grad_input")
    if w is not None:
        within(got["w"], (dz * back(unit)).sum((0, 2)),
               (off * back(unit).abs() + dz.abs() * back(e_unit) + 2 * FN * (dz * back(unit)).abs()).sum((0, 2)), dtype, "grad_weight")
    if b is not None:
        within(got["b"], dz.sum((0, 2)), (off + 2 * FN * dz.abs()).sum((0, 2)), dtype, "grad_bias")
    return out, got


# (N, C, G, h, w): one value a group, a channel a group, all in one, groups that cut vectors, odd sides, many pixels
NORM = [
    (1, 1, 1, 1, 1), (2, 6, 6, 1, 1), (3, 8, 2, 1, 1), (2, 32, 8, 32, 32), (1, 24, 1, 9, 11), (2, 60, 20, 31, 37), (2, 20, 4, 16, 24),
    (4, 128, 32, 16, 32), (1, 64, 16, 96, 128), (2, 7, 7, 13, 17), (1, 3, 1, 200, 301), (3, 96, 3, 5, 5), (64, 16, 4, 8, 8),
    (1, 512, 32, 7, 9), (1, 1030, 10, 6, 7), (2, 1035, 5, 5, 6), (3, 6144, 6144, 3, 3), (2, 1023, 1, 5, 4), (1, 8, 8, 128, 256), (2, 48, 6, 64, 64), (1, 2048, 32, 4, 5), (1, 8, 1, 250, 251),
]


@pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", NORM, ids=str)
def test_norm(bc, shape, dtype, last):
    N, C, G, h, w = shape
    gen = torch.Generator(device="cuda").manual_seed(C + G * h)
    for k, act in enumerate((None, "relu", "silu", "gelu")):
        x, g = maps(gen, (N, C, h, w), dtype, last, 1.5, 0.5), maps(gen, (N, C, h, w), dtype, last)
        weight = (1 + 0.3 * torch.randn(C, device="cuda", generator=gen)).to(dtype) if k != 1 else None
        bias = torch.randn(C, device="cuda", generator=gen).to(dtype) if k != 3 else None
        out, got = check_norm(bc, x, G, weight, bias, g, act, eps=1e-5 if k else 1e-3)
        assert same_layout(out, last) and same_layout(got["x"], last)


@pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(2, 32, 8, 40, 64), (1, 24, 2, 128, 160), (2, 20, 4, 33, 35)], ids=str)
def test_norm_of_values_far_from_zero(bc, shape, dtype, last):
    """A mean a thousand times the spread, and one value a million times it: sums of squares would lose the variance."""
    N, C, G, h, w = shape
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = maps(gen, (N, C, h, w), dtype, last)
    x = maps(gen, (N, C, h, w), dtype, last, 1.0 if dtype == torch.float32 else 16.0, 1000.0)
    check_norm(bc, x, G, None, None, g, "silu")
    x = maps(gen, (N, C, h, w), dtype, last)
    x[0, 0, 0, 0] = 1e6
    check_norm(bc, x, G, None, None, g, None)


@pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
@pytest.mark.parametrize("shape", [(2, 16, 4, 16, 16), (2, 24, 3, 65, 77)], ids=str)
def test_norm_of_equal_values(bc, shape, last):
    N, C, G, h, w = shape
    x = maps(torch.Generator(device="cuda").manual_seed(1), shape[:2] + shape[3:], torch.float32, last, 0.0, 3.25).requires_grad_()
    out = bc.group_norm(x, G, eps=1e-5)
    assert not out.any()
    assert not torch.autograd.grad(out, x, torch.ones_like(out))[0].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_norm_subsets_of_gradients_have_the_bits_of_all(bc, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for act, last in ((None, False), ("silu", True), ("gelu", False)):
        t = [maps(gen, (3, 24, 20, 24), dtype, last), torch.rand(24, device="cuda", generator=gen).to(dtype),
             torch.randn(24, device="cuda", generator=gen).to(dtype)]
        g = maps(gen, (3, 24, 20, 24), dtype, last)

        def grads(which):
            leaves = [v.detach().requires_grad_(i in which) for i, v in enumerate(t)]
            out = bc.group_norm(leaves[0], 6, *leaves[1:], activation=act)
            return dict(zip(which, torch.autograd.grad(out, [leaves[i] for i in which], g)))

        everything = grads((0, 1, 2))
        for which in ((0,), (1,), (2,), (0, 1), (1, 2)):
            for i, v in grads(which).items():
                assert torch.equal(v, everything[i]), (act, which, i)


def test_norm_without_pixels_or_samples(bc):
    for N, h in ((0, 5), (2, 0)):
        x = torch.randn(N, 8, h, 5, device="cuda").requires_grad_()
        w, b = (torch.randn(8, device="cuda").requires_grad_() for _ in range(2))
        out = bc.group_norm(x, 2, w, b, activation="gelu")
        assert out.shape == x.shape
        gx, gw, gb = torch.autograd.grad(out, (x, w, b), torch.ones_like(out))
        assert gx.shape == x.shape and not gw.any() and not gb.any()


# ---- both ------------------------------------------------------------------------------------------------

def _calls(bc):
    """Both layers on (N, 24, h, w), as f(x, *params) with their parameters."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    return [("pointwise", lambda x, w, b: bc.pointwise_conv2d(x, w, b, activation="silu"), [0.2 * r(40, 24), r(40)]),
            ("norm", lambda x, w, b: bc.group_norm(x, 6, w, b, activation="silu"), [1 + 0.2 * r(24), r(24)])]


def _step(f, x, params, g):
    leaves = [t.detach().requires_grad_() for t in (x, *params)]
    out = f(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, g[:, :out.shape[1]].contiguous())]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_other_strides(bc, dtype):
    """Slices, transposes, expanded and shifted tensors give what their copies give; a row off a vector's alignment too."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    big = torch.randn(3, 50, 21, 34, device="cuda", generator=gen).to(dtype)
    views = [big[:, :24], big[:, 1:25], big[:, ::2][:, :24], big[..., 1:], big.transpose(2, 3), big[:, :24].transpose(0, 2)[:3].transpose(0, 2),
             big[:1].expand(3, -1, -1, -1), big.contiguous(memory_format=torch.channels_last)[:, 3:27]]
    flat = torch.randn(2 * 24 * 20 * 16 + 1, device="cuda", generator=gen).to(dtype)[1:]
    views += [flat.view(2, 24, 20, 16), flat.view(2, 20, 16, 24).permute(0, 3, 1, 2)]
    for name, f, params in _calls(bc):
        params = [p.to(dtype) for p in params]
        shifted = [torch.cat([p.flatten()[:1], p.flatten()])[1:].view(p.shape) for p in params]
        for i, v in enumerate(views):
            v = v[:, :24]
            g = torch.randn(v.shape[0], 40, *v.shape[2:], device="cuda", generator=gen).to(dtype)
            a = _step(f, v, params, g)
            last = not v.is_contiguous() and v.is_contiguous(memory_format=torch.channels_last)
            copy = v.clone(memory_format=torch.channels_last if last else torch.contiguous_format)
            b = _step(f, copy, shifted, g)
            for k, (p, q) in enumerate(zip(a, b)):      # (a different alignment may take another order of sums)
                tol = 3e-5 if dtype == torch.float32 else 4 * U[dtype]
                assert p.shape == q.shape and (p.double() - q.double()).norm() <= tol * q.double().norm(), (name, i, k)


def test_gradients_of_other_strides(bc):
    for name, f, params in _calls(bc):
        x = torch.randn(2, 24, 12, 20, device="cuda")
        out = f(x, *params)
        for g in (torch.randn_like(out).contiguous(memory_format=torch.channels_last), torch.randn(1, 1, 1, 1, device="cuda").expand_as(out),
                  torch.randn(*out.shape[:2], 20, 12, device="cuda").transpose(2, 3)):
            leaves = [t.detach().requires_grad_() for t in (x, *params)]
            a = torch.autograd.grad(f(*leaves), leaves, g)
            b = torch.autograd.grad(f(*leaves), leaves, g.contiguous())
            assert all(torch.equal(p, q) for p, q in zip(a, b)), name


def test_residual_in_another_layout_and_two_dimensional_weight(bc):
    x, r = torch.randn(2, 24, 6, 10, device="cuda"), torch.randn(2, 40, 6, 10, device="cuda")
    w = torch.randn(40, 24, device="cuda")
    a = bc.pointwise_conv2d(x, w, residual=r.contiguous(memory_format=torch.channels_last))
    assert torch.equal(a, bc.pointwise_conv2d(x, w.view(40, 24, 1, 1), residual=r)) and a.is_contiguous()
    assert torch.equal(a, bc.pointwise_conv2d(x, w.t().contiguous().t(), residual=r))


def test_refusals(bc):
    x, w, b = torch.randn(2, 4, 5, 6, device="cuda"), torch.randn(3, 4, device="cuda"), torch.randn(3, device="cuda")
    cases = [
        (lambda: bc.pointwise_conv2d(x[0], w), "4 dimensions"),
        (lambda: bc.pointwise_conv2d(x, w[:, :3]), "weight must be"),
        (lambda: bc.pointwise_conv2d(x, torch.randn(3, 4, 3, 3, device="cuda")), "weight must be"),
        (lambda: bc.pointwise_conv2d(x, w, b[:2]), "bias must hold"),
        (lambda: bc.pointwise_conv2d(x, w, residual=x), "residual must have"),
        (lambda: bc.pointwise_conv2d(x, w.half()), "weight is torch.float16"),
        (lambda: bc.pointwise_conv2d(x.double(), w.double()), "float32, float16 or bfloat16"),
        (lambda: bc.pointwise_conv2d(x, w.cpu()), "no CPU implementation"),
        (lambda: bc.pointwise_conv2d(x.long(), w), "float32, float16 or bfloat16"),
        (lambda: bc.group_norm(x[0], 2), "4 dimensions"),
        (lambda: bc.group_norm(x, 3), "do not make 3 groups"),
        (lambda: bc.group_norm(x, 0), "do not make 0 groups"),
        (lambda: bc.group_norm(x, -2), "groups"),
        (lambda: bc.group_norm(torch.randn(2, 0, 5, 6, device="cuda"), 1), "groups"),
        (lambda: bc.group_norm(x, 2, b), "weight must hold"),
        (lambda: bc.group_norm(x, 2, None, b), "bias must hold"),
        (lambda: bc.group_norm(x, 2, torch.randn(4, device="cuda").bfloat16()), "weight is torch.bfloat16"),
        (lambda: bc.group_norm(x.double(), 2), "float32, float16 or bfloat16"),
    ]
    for i, (call, text) in enumerate(cases):
        with pytest.raises(RuntimeError, match=text):
            call()
            pytest.fail("case %d was not refused" % i)


def test_not_a_number_stays_where_it_belongs(bc):
    """NaN and infinity reach what depends on them and nothing else."""
    for dtype in DTYPES:
        for last in (False, True):
            x = maps(torch.Generator(device="cuda").manual_seed(1), (3, 24, 9, 24), dtype, last)
            w = torch.randn(40, 24, device="cuda").to(dtype)
            for act in ("relu", "silu", "gelu"):
                clean = bc.pointwise_conv2d(x, w, activation=act)
                for bad in (float("nan"), float("inf"), -float("inf")):
                    y = x.clone()
                    y[1, 3, 4, 5] = bad
                    out = bc.pointwise_conv2d(y, w, activation=act)
                    touched = torch.zeros_like(out, dtype=torch.bool)
                    touched[1, :, 4, 5] = True
                    # (16-bit SiLU: a value's neighbour is in its 22nd bit, which can move the rounding by one step, 2 u)
                    off = (out[~touched].double() - clean[~touched].double()).abs()
                    one = 2 * U[dtype] * clean[~touched].double().abs() + 2 * TINY[dtype] if act == "silu" and dtype != torch.float32 else 0
                    assert (off <= one).all()
                    if bad != bad:
                        assert out[touched].isnan().all()
                    else:
                        want = act64(bad * torch.sign(w[:, 3]).double(), act)
                        assert torch.equal(out[touched].double().nan_to_num(-1, posinf=1), want.nan_to_num(-1, posinf=1))
            clean = bc.group_norm(x, 6)
            for bad in (float("nan"), float("inf")):
                y = x.clone()
                y[1, 5, 4, 5] = bad
                out = bc.group_norm(y, 6, activation="relu" if bad != bad else None)
                assert out[1, 4:8].isnan().any()
                if bad != bad:
                    assert out[1, 4:8].isnan().all()
                else:
                    rest = torch.ones_like(out, dtype=torch.bool)
                    rest[1, 4:8] = False
                    assert torch.equal(out[rest], clean[rest])


def test_same_bits_from_call_to_call_and_on_another_stream(bc):
    for dtype in DTYPES:
        for last in (False, True):
            x = maps(torch.Generator(device="cuda").manual_seed(8), (4, 24, 40, 48), dtype, last)
            g = maps(torch.Generator(device="cuda").manual_seed(9), (4, 40, 40, 48), dtype, last)
            for name, f, params in _calls(bc):
                params = [p.to(dtype) for p in params]
                first = _step(f, x, params, g)
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    second = _step(f, x, params, g)
                torch.cuda.current_stream().wait_stream(side)
                third = _step(f, x, params, g)
                assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, second, third)), name


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_two_captured_steps_replayed_at_once(bc, dtype):
    """Graphs of whole steps, gradients included, on two streams: each has workspaces of its own and computes on new data."""
    for name, f, params in _calls(bc):
        graphs = []
        params = [p.to(dtype) for p in params]
        for k in range(2):
            x, g = torch.randn(2, 24, 40, 48, device="cuda").to(dtype), torch.randn(2, 40, 40, 48, device="cuda").to(dtype)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                _step(f, x, params, g)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = _step(f, x, params, g)
            graphs.append((graph, x, g, out, torch.cuda.Stream()))
        for turn in range(3):
            wanted = []
            for graph, x, g, out, s in graphs:
                x.normal_()
                g.normal_()
                wanted.append(_step(f, x, params, g))
            torch.cuda.synchronize()
            for graph, x, g, out, s in graphs:
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for (graph, x, g, out, s), want in zip(graphs, wanted):
                assert all(torch.equal(a, b) for a, b in zip(out, want)), (name, turn)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_first_call_of_a_thread(bc, dtype):
    """A thread that has not called into CUDA before, with memory at hand that needs no call either."""
    import threading
    x, g = torch.randn(2, 24, 16, 16, device="cuda").to(dtype), torch.randn(2, 40, 16, 16, device="cuda").to(dtype)
    for name, f, params in _calls(bc):
        params = [p.to(dtype) for p in params]
        for what in (lambda: [f(x, *params)], lambda: _step(f, x, params, g)):
            want, got = what(), []

            def work():
                got.extend(what())
                torch.cuda.synchronize()

            del want[1:]
            t = threading.Thread(target=work)
            t.start()
            t.join()
            assert got and torch.equal(got[0], want[0]), name


def test_what_autograd_asks_for(bc):
    import torch.autograd.forward_ad as fwad
    for name, f, params in _calls(bc):
        x = torch.randn(2, 24, 12, 20, device="cuda")
        leaves = [t.detach().requires_grad_() for t in (x, *params)]
        out = f(*leaves)
        assert out.grad_fn.name() == {"pointwise": "PointwiseConvFunctionBackward", "norm": "GroupNormFunctionBackward"}[name]
        g = torch.autograd.grad(out.sum(), leaves[0], create_graph=True)[0]
        with pytest.raises(RuntimeError, match="differentiated"):
            torch.autograd.grad(g.sum(), leaves[0])
        out = f(*leaves)
        with torch.no_grad():
            leaves[1].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaves)
        out = f(*leaves)
        torch.autograd.grad(out.sum(), leaves)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(out.sum(), leaves)
        with torch.no_grad():
            assert not f(*leaves).requires_grad
        assert not f(x, *params).requires_grad
        with pytest.raises(RuntimeError):
            with fwad.dual_level():
                f(fwad.make_dual(x, torch.ones_like(x)), *params)
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda t: f(t, *params))(x[None])
        with torch.inference_mode():
            assert torch.equal(f(x, *params), f(x, *params))


def test_trace_and_the_python_classes(bc):
    for name, f, params in _calls(bc):
        x = torch.randn(2, 24, 12, 20, device="cuda")
        traced = torch.jit.trace(lambda t: f(t, *params), x, check_trace=False)
        for other in (x, torch.randn_like(x)):
            assert torch.equal(traced(other), f(other, *params))
        leaves = [t.detach().requires_grad_() for t in (x, *params)]
        if name == "pointwise":
            out = bc.PointwiseConvFunction.apply(*leaves, None, 2)
        else:
            out = bc.GroupNormFunction.apply(*leaves, 6, 1e-5, 2)
        g = torch.randn_like(out)
        a = [out, *torch.autograd.grad(out, leaves, g)]
        out = f(*leaves)
        assert all(torch.equal(p, q) for p, q in zip(a, [out, *torch.autograd.grad(out, leaves, g)])), name


@pytest.mark.parametrize("w", [1024, 1023])
@pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
def test_offsets_past_32_bits(bc, last, w):
    """More than 2^31 values; samples at both ends against calls on them alone."""
    N, C, h = 68, 64 if last is False or w == 1024 else 65, 512
    x = torch.empty(N, C, h, w, device="cuda", dtype=torch.bfloat16,
                    memory_format=torch.channels_last if last else torch.contiguous_format)
    for n in range(N):
        x[n].normal_(n % 3, 1 + n % 2)
    ends = torch.tensor([0, 33, N - 1], device="cuda")
    few = x[ends].contiguous(memory_format=torch.channels_last if last else torch.contiguous_format)
    weight = torch.randn(8, C, device="cuda").bfloat16()
    assert torch.equal(bc.pointwise_conv2d(x, weight)[ends], bc.pointwise_conv2d(few, weight))
    out = bc.group_norm(x, 16 if C % 16 == 0 else 13)
    small = bc.group_norm(few, 16 if C % 16 == 0 else 13)
    assert (out[ends].double() - small.double()).abs().max() <= 2 ** -7 * small.double().abs().max()
    del out
    x.requires_grad_()
    g = torch.randn(1, C, 1, 1, device="cuda").bfloat16().expand(N, C, h, w)
    G = 16 if C % 16 == 0 else 13
    gx = torch.autograd.grad(bc.group_norm(x, G), x, g)[0][ends]
    few.requires_grad_()
    gf = torch.autograd.grad(bc.group_norm(few, G), few, g[:3])[0]
    assert (gx.double() - gf.double()).abs().max() <= 2 ** -7 * gf.double().abs().max()


@pytest.mark.parametrize("last", [False, True], ids=["planes", "last"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_the_layers_of_a_block_together(bc, dtype, last):
    """1 x 1 convolution, normalisation, box convolution, normalisation, 1 x 1 convolution with the skip connection: forward
    and every gradient against the same chain in 64 bits (the box convolution's own 64-bit form in it)."""
    torch.manual_seed(0)
    C, F, h, w = 8, 4, 33, 40

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.reduce, self.norm1 = bc.PointwiseConv2d(C * F, C, bias=False), bc.GroupNorm2d(2, C, activation="silu")
            self.box, self.norm2 = bc.BoxConv2d(C, F, h, w), bc.GroupNorm2d(8, C * F, activation="gelu")
            self.expand = bc.PointwiseConv2d(C * F, C * F, activation="silu")

        def forward(self, x):
            return self.expand(self.norm2(self.box(self.norm1(self.reduce(x)))), residual=x)

    m = Block().cuda().to(dtype)
    x = torch.randn(2, C * F, h, w, device="cuda").to(dtype)
    x = x.contiguous(memory_format=torch.channels_last if last else torch.contiguous_format).requires_grad_()
    out = m(x)
    g = torch.randn_like(out)
    params = dict(m.named_parameters())
    got = dict(zip(["x", *params], torch.autograd.grad(out, [x, *params.values()], g)))

    q = {k: v.detach().double().requires_grad_() for k, v in params.items()}
    X = x.detach().double().requires_grad_()
    box = bc.BoxConv2d(C, F, h, w).cuda().double().eval()
    t = torch.einsum("oi,nihw->nohw", q["reduce.weight"][:, :, 0, 0], X)
    t = act64(torch.nn.functional.group_norm(t, 2, q["norm1.weight"], q["norm1.bias"]), "silu")
    t = bc.BoxConvolutionFunction.apply(t, q["box.x_min"], q["box.x_max"], q["box.y_min"], q["box.y_max"], box.reparametrization_h,
                                        box.reparametrization_w, True, True)
    t = act64(torch.nn.functional.group_norm(t, 8, q["norm2.weight"], q["norm2.bias"]), "gelu")
    t = torch.einsum("oi,nihw->nohw", q["expand.weight"][:, :, 0, 0], t) + q["expand.bias"].view(1, -1, 1, 1) + X
    ref = act64(t, "silu")
    want = dict(zip(["x", *q], torch.autograd.grad(ref, [X, *q.values()], g.double())))
    # five tensors in a row are rounded on the way there and as many back, each by u of its size on top of what came before:
    # 2-norms off by a dozen u, times what normalisations of small spreads magnify (2); float32: the box convolution's
    # tolerances, 1e-4 and 1e-3 for the box parameters
    tol = 1e-4 if dtype == torch.float32 else 24 * U[dtype]
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(out, ref) < tol
    for k in want:
        assert rel(got[k], want[k]) < (10 * tol if k.startswith("box") else tol), k


def test_no_wait_has_expired():
    from box_convolution import _cabi
    assert _cabi.wait_timeouts() == 0
