"""The operators around a box convolution as cases that can be timed: the pointwise (1 x 1) convolution that
mixes its channels, with bias, skip connection and activation in one pass, and group normalisation with an
activation; both on planes (N, C, h, w) and channels last, forward alone and with their gradients.

    pointwise   out = act(W x + b + residual)          per pixel, W (out_planes, in_planes)
    norm        out = act(weight * (x - mean) / sqrt(var + eps) + bias)      mean, var over a group's planes

`own` false: plain form, elementary operations in 32 bits, rounded once.  `own` true: the package's functions.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def pointwise(name, train, N, cin, cout, h, w, dtype, act="none", residual=False, last=False):
    c = {"op": "pointwise", "train": train, "N": N, "cin": cin, "cout": cout, "h": h, "w": w, "dtype": dtype,
         "act": act, "residual": residual, "last": last}
    return dict(c, name=name) if name else c


def norm(name, train, N, C, groups, h, w, dtype, act="none", affine=True, last=False):
    c = {"op": "norm", "train": train, "N": N, "C": C, "groups": groups, "h": h, "w": w, "dtype": dtype,
         "act": act, "affine": affine, "last": last}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a head on globally pooled features: eight pixels in all, nothing but latency
        pointwise("pointwise_pooled", False, 8, 128, 32, 1, 1, "float32", "relu"),
        # in front of the box convolution of one frame's block at 1/8 of 512 x 1024
        pointwise("pointwise_frame", False, 1, 128, 32, 64, 128, "float32", "relu"),
        # the same place in training, a normalisation behind it, so without activation
        pointwise("pointwise_train_bf16", True, 16, 128, 32, 64, 128, "bfloat16"),
        # back to the block's width behind a box convolution with a skip connection, channels last, inference of a batch
        pointwise("pointwise_expand_f16", False, 32, 32, 128, 64, 128, "float16", "relu", residual=True, last=True),
        # training in float32, the package's default type
        pointwise("pointwise_train_f32", True, 16, 128, 32, 64, 128, "float32", "silu"),
        # a wide mixing layer on a large batch, channels last: everything at once
        pointwise("pointwise_wide_bf16", True, 64, 256, 256, 64, 128, "bfloat16", "gelu", residual=True, last=True),
        # feature maps whose sides and channels are no multiple of anything
        pointwise("pointwise_odd_f16", True, 6, 60, 20, 93, 157, "float16", "silu", residual=True),
        # one small crop
        norm("norm_crop", False, 1, 32, 8, 32, 32, "float32", "relu"),
        # behind a box convolution's block at 1/8 of a frame, ordinary batch, channels last
        norm("norm_train_bf16", True, 16, 128, 32, 64, 128, "bfloat16", "silu", last=True),
        # 256 samples of planes in front of a box convolution
        norm("norm_batch256_f32", True, 256, 32, 8, 64, 128, "float32", "silu"),
        # one frame at 1/4 of 1024 x 2048, channels last: few statistics over many pixels
        norm("norm_frame_f32", False, 1, 64, 16, 256, 512, "float32", "relu", last=True),
        # odd sides, channels that are no multiple of a vector
        norm("norm_odd_f16", True, 6, 60, 20, 93, 157, "float16", "gelu", last=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, hi):
    c = _log_int(rng, 1, hi)
    return c if c < 8 or rng.random() < 0.4 else c // 8 * 8


def draw(rng):
    """Sizes over their logarithm: single pixels to planes of a quarter frame, one channel to 512 (normalised: 1024)."""
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    train, last = rng.random() < 0.6, rng.random() < 0.5
    # (a ReLU's gradient jumps where 32-bit sums differ in sign: forward only)
    act = rng.choice(["none", "silu", "gelu"] if train else ["none", "relu", "relu", "silu", "gelu"])
    N, h, w = _log_int(rng, 1, 64), _log_int(rng, 1, 512), _log_int(rng, 1, 512)
    if rng.random() < 0.5:
        cin, cout, residual = _channels(rng, 512), _channels(rng, 512), rng.random() < 0.4
        while N * h * w * (cin + cout) > 1 << 27 or N * h * w * cin * cout > 1 << 34:
            N, h = max(1, N // 2), (h if N > 1 else h // 2)
        return pointwise(None, train, N, cin, cout, h, w, dtype, act, residual, last)
    groups = _log_int(rng, 1, 32)
    C, affine = groups * _log_int(rng, 1, 32), rng.random() < 0.8
    h = max(h, -(-32 // (w * (C // groups))))       # (statistics of a handful of values leave gradients of nothing but rounding)
    while N * h * w * C > 1 << 27:
        N, h = max(1, N // 2), (h if N > 1 else h // 2)
    return norm(None, train, N, C, groups, h, w, dtype, act, affine, last)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    layout = torch.channels_last if case["last"] else torch.contiguous_format

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def maps(t):
        return t.to(dtype).contiguous(memory_format=layout)

    N, h, w = case["N"], case["h"], case["w"]
    state = {"case": case}
    if case["op"] == "pointwise":
        cin, cout = case["cin"], case["cout"]
        state["x"] = maps(randn(N, cin, h, w))
        state["weight"] = (randn(cout, cin, 1, 1) / math.sqrt(cin)).to(dtype)
        state["bias"] = (0.1 * randn(cout)).to(dtype)
        state["residual"] = maps(randn(N, cout, h, w)) if case["residual"] else None
        out = (N, cout, h, w)
    else:
        C = case["C"]
        # channels of their own offsets and spreads, as layers give them
        state["x"] = maps(randn(N, C, h, w) * (0.5 + randn(1, C, 1, 1).abs()) + randn(1, C, 1, 1))
        state["weight"] = (1 + 0.2 * randn(C)).to(dtype) if case["affine"] else None
        state["bias"] = (0.2 * randn(C)).to(dtype) if case["affine"] else None
        out = (N, C, h, w)
    if case["train"]:
        state["grad"] = maps(randn(*out))
        state["leaves"] = [t.requires_grad_() for t in (state["x"], state["weight"], state["bias"], state.get("residual"))
                           if t is not None]
    return state


# ---- plain forms -----------------------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _plain_pointwise(state):
    case, dtype = state["case"], state["x"].dtype
    N, h, w = case["N"], case["h"], case["w"]
    x = state["x"].detach().float().reshape(N, case["cin"], h * w)
    weight = state["weight"].detach().float().reshape(case["cout"], case["cin"])
    z = torch.matmul(weight, x) + state["bias"].detach().float()[:, None]
    if state["residual"] is not None:
        z = z + state["residual"].detach().float().reshape(z.shape)
    out = _act(z, case["act"]).to(dtype).reshape(N, case["cout"], h, w)
    if not case["train"]:
        return out
    dz = state["grad"].float().reshape(z.shape) * _act_slope(z, case["act"])
    grads = [torch.matmul(weight.t(), dz).reshape(state["x"].shape), torch.matmul(dz, x.transpose(1, 2)).sum(0).reshape(state["weight"].shape),
             dz.sum((0, 2))]
    if state["residual"] is not None:
        grads.append(dz.reshape(out.shape))
    return [out] + [g.to(dtype) for g in grads]


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    N, C, G = case["N"], case["C"], case["groups"]
    x = state["x"].detach().float().reshape(N, G, -1)
    d = x - x.mean(2, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(2, keepdim=True) + EPS)
    xhat = (d * rstd).reshape(N, C, -1)
    affine = case["affine"]
    weight = state["weight"].detach().float()[:, None] if affine else 1.0
    z = xhat * weight + (state["bias"].detach().float()[:, None] if affine else 0.0)
    out = _act(z, case["act"]).to(dtype).reshape(state["x"].shape)
    if not case["train"]:
        return out
    dz = state["grad"].float().reshape(z.shape) * _act_slope(z, case["act"])
    dxhat, unit = (dz * weight).reshape(N, G, -1), xhat.reshape(N, G, -1)
    dx = rstd * (dxhat - dxhat.mean(2, keepdim=True) - unit * (dxhat * unit).mean(2, keepdim=True))
    grads = [dx.reshape(state["x"].shape)]
    if affine:
        grads += [(dz * xhat).sum((0, 2)), dz.sum((0, 2))]
    return [out] + [g.to(dtype) for g in grads]


# ---- the package's functions -----------------------------------------------------------------------------

def _package():
    path = os.path.join(os.getcwd(), "box-convolutions_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import box_convolution
    return box_convolution


def _own(state):
    bc, case = _package(), state["case"]
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "pointwise":
        out = bc.pointwise_conv2d(state["x"], state["weight"], state["bias"], activation=act, residual=state["residual"])
    else:
        out = bc.group_norm(state["x"], case["groups"], state["weight"], state["bias"], EPS, activation=act)
    if not case["train"]:
        return out
    return [out.detach(), *torch.autograd.grad(out, state["leaves"], state["grad"])]


def run(state):
    if own:
        return _own(state)
    return _plain_pointwise(state) if state["case"]["op"] == "pointwise" else _plain_norm(state)


def work(case):
    """Inputs read once, outputs written once.  Operations: a multiplication and an addition per weight and pixel, three
    times that with both gradients; about ten a value for a normalisation, thirty with its gradient."""
    size, pixels = (4 if case["dtype"] == "float32" else 2), case["N"] * case["h"] * case["w"]
    if case["op"] == "pointwise":
        cin, cout, train = case["cin"], case["cout"], case["train"]
        values = pixels * (cin + cout * (2 if case["residual"] else 1)) + cout * (cin + 1)
        return {"bytes": size * values * (2 if train else 1), "flops": 2 * pixels * cin * cout * (3 if train else 1)}
    values = pixels * case["C"]
    return {"bytes": size * values * (4 if case["train"] else 2), "flops": values * (30 if case["train"] else 10)}


# ---- the definitions in 64 bits, gradients by differentiation of the definition --------------------------

def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: state[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias", "residual")
            if state.get(k) is not None}
    if case["op"] == "pointwise":
        rows = wide["x"].permute(0, 2, 3, 1) @ wide["weight"][:, :, 0, 0].T + wide["bias"]
        z = rows.permute(0, 3, 1, 2)
        z = z + wide["residual"] if "residual" in wide else z
    else:
        grouped = wide["x"].unflatten(1, (case["groups"], -1))
        var, mean = torch.var_mean(grouped, (2, 3, 4), keepdim=True, correction=0)
        z = ((grouped - mean) * torch.rsqrt(var + EPS)).flatten(1, 2)
        if case["affine"]:
            z = z * wide["weight"].view(-1, 1, 1) + wide["bias"].view(-1, 1, 1)
    if case["act"] == "relu":
        z = z.clamp_min(0)
    elif case["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif case["act"] == "gelu":
        z = z * torch.special.ndtr(z)
    if not case["train"]:
        return z
    names = [k for k in ("x", "weight", "bias", "residual") if k in wide]
    return [z.detach(), *torch.autograd.grad(z, [wide[k] for k in names], state["grad"].double())]
