"""64-bit restatement (torch, CPU) of the 8-bit activation checkpoints, the activations, the group norm and the checkpointed layers:
include/dbev_hip.h (dbev_act8_*, dbev_gn_act_*) states the definitions.  The reference has no such operators: nn.GroupNorm, F.silu / F.gelu
and nn.Linear are its plain counterparts, to which these reduce without a checkpoint."""
import math

import torch

BLOCK = 32


def quantise(x, fmt):
    """x [rows, C] (any float type) -> codes uint8 [rows, C], scale bytes uint8 [rows, ceil(C / 32)], one block at a time in Python numbers
    where it matters (math.frexp is exact)"""
    rows, C = x.shape
    nb = -(-C // BLOCK)
    codes = torch.zeros((rows, C), dtype=torch.uint8)
    scales = torch.zeros((rows, nb), dtype=torch.uint8)
    xd = x.detach().cpu().double()
    for r in range(rows):
        for b in range(nb):
            v = xd[r, b * BLOCK:(b + 1) * BLOCK]
            if not bool(torch.isfinite(v).all()):
                scales[r, b] = 255
                continue
            a = float(v.abs().max())
            e = math.frexp(a)[1] - 1 if a > 0 else -10 ** 6
            if fmt == "int8":
                k = max(e - 6, -127)
                q = torch.clamp(torch.round(v / 2.0 ** k), -127, 127).to(torch.int8).view(torch.uint8)
            else:
                k = max(e - 8, -127)
                if a > 448.0 * 2.0 ** k:
                    k += 1
                q = (v / 2.0 ** k).float().to(torch.float8_e4m3fn).view(torch.uint8)     # exact in fp32, then one rounding
            scales[r, b] = k + 127
            codes[r, b * BLOCK:(b + 1) * BLOCK] = q
    return codes, scales


def values(codes, scales, fmt):
    """f64 values of codes / scales"""
    rows, C = codes.shape
    c = codes.view(torch.int8).double() if fmt == "int8" else codes.view(torch.float8_e4m3fn).double()
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127)
    s[scales == 255] = float("nan")
    return c * s.repeat_interleave(BLOCK, 1)[:, :C]


def restored(x, fmt):
    """x [rows, C] -> x^ f64 (x itself without a format); vectorised, agrees with `values(*quantise(x, fmt))` (tests/test_host_act8.py)"""
    x = x.detach().double()
    if fmt is None:
        return x
    rows, C = x.shape
    t = torch.nn.functional.pad(x, (0, -C % BLOCK)).view(rows, -1, BLOCK)
    a = t.abs().amax(2, keepdim=True)
    e = torch.where(a > 0, torch.frexp(a)[1].double() - 1, torch.full_like(a, -1000.0))
    if fmt == "int8":
        u = torch.exp2((e - 6).clamp(min=-127))
        q = torch.clamp(torch.round(t / u), -127, 127)
    else:
        u = torch.exp2((e - 8).clamp(min=-127))
        u = torch.where(a > 448 * u, 2 * u, u)
        q = (t / u).float().to(torch.float8_e4m3fn).double()
    out = torch.where(torch.isfinite(a), q * u, torch.full_like(t, float("nan")))
    return out.view(rows, -1)[:, :C].contiguous()


def act(z, name):
    """(act(z), act'(z)) in f64"""
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), torch.where(z > 0, torch.ones_like(z), torch.where(z == z, torch.zeros_like(z), z))
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        p = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


class ActFn(torch.autograd.Function):
    """activation of f64 rows whose gradient is taken at the checkpoint"""

    @staticmethod
    def forward(ctx, x, name, fmt):
        ctx.save_for_backward(restored(x, fmt))
        ctx.name = name
        return act(x, name)[0]

    @staticmethod
    def backward(ctx, g):
        return g * act(ctx.saved_tensors[0], ctx.name)[1], None, None


class LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, fmt):
        ctx.save_for_backward(restored(x, fmt), w)
        return x @ w.t() + (0 if b is None else b)

    @staticmethod
    def backward(ctx, g):
        xr, w = ctx.saved_tensors
        return g @ w, g.t() @ xr, g.sum(0) if ctx.needs_input_grad[2] else None, None


def group_norm(x, G, weight, bias, eps, name, fmt=None, gy=None):
    """x [N, S, C] f64 -> y, or with gy (y, dx, dgamma, dbeta, z) by the formulas (z: the activation's argument in the backward)"""
    N, S, C = x.shape
    w = x.new_ones(C) if weight is None else weight
    b = x.new_zeros(C) if bias is None else bias
    t = x.view(N, S, G, C // G)
    mean = t.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((t - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    z = ((t - mean) * rstd).view(N, S, C) * w + b
    y = act(z, name)[0]
    if gy is None:
        return y
    if fmt is not None:
        t = restored(x.reshape(N * S, C), fmt).view(N, S, G, C // G)
    xh = ((t - mean) * rstd).view(N, S, C)
    z = xh * w + b
    g = gy * act(z, name)[1]
    db, dg = g.sum((0, 1)), (g * xh).sum((0, 1))
    gw = (g * w).view(N, S, G, C // G)
    xg = xh.view(N, S, G, C // G)
    dx = rstd * (gw - gw.mean((1, 3), keepdim=True) - xg * (gw * xg).mean((1, 3), keepdim=True))
    return y, dx.reshape(N, S, C), dg, db, z


class GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, G, weight, bias, eps, name, fmt):
        ctx.save_for_backward(x, weight, bias)
        ctx.cfg = (G, eps, name, fmt)
        return group_norm(x, G, weight, bias, eps, name)

    @staticmethod
    def backward(ctx, gy):
        x, w, b = ctx.saved_tensors
        G, eps, name, fmt = ctx.cfg
        _, dx, dg, db, _ = group_norm(x, G, w, b, eps, name, fmt, gy)
        return dx, None, dg, db, None, None, None
