"""8-bit activation checkpoints on the GPU (csrc/act8.hip, csrc/act8_wgrad.hip, distill_bev_amd/act8.py) against oracle/act8.py (64 bits).

Codes, scale bytes and restored values are compared for equality: scales are powers of two, the code is the only rounding.  Tolerances of
computed values, u = 2^-24 (half a step of fp32), and half a step of the output type on top (`_half`):
  silu      exp2's argument is rounded (|z| u), exp2, 1 +, reciprocal and product a few u each: |dy| <= (1.5 |z| + 8) u |y|
  silu'     f = s (1 + z (1 - s)); a relative error e = (1.5 |z| + 8) u of s moves f by s e (1 + |z|)
  gelu      Q = 1 - Phi(|z|) to (z^2 + 16) u relative (fit 3.2e-8, fp32 Horner 5 u, argument z^2 / 2 rounded twice); Phi = 1 - Q or Q
  gelu'     f = Phi + z phi, phi to (z^2 + 6) u
  (sigmoid, Q and phi below 2^-126 are flushed to zero by the hardware's exp2 and reciprocal: |z| 2^-126 of the result, (1 + |z|) 2^-126 of
  the derivative)
  weight gradient   products exact, fp32 sums of n terms in chains and a tree: independent roundings grow like sqrt(n):
                    |dg| <= (8 + 4 sqrt(3 M)) u sum |gy| |x^|"""
import math

import pytest
import torch
import torch.nn as nn

from oracle import act8 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _half(ref, dtype):
    """half a step of `dtype` at |ref| (and below its normal range)"""
    f = torch.finfo(dtype)
    return (f.eps / 2) * ref.abs().clamp(min=f.tiny)


def _data(rows, C, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g) * torch.exp(1.5 * torch.randn(rows, 1, generator=g))
    return x.to(dtype)


def _within(got, ref, lim, what=""):
    """|got - ref| <= lim everywhere; says where not"""
    d = (got.detach().cpu().double() - ref).abs()
    bad = ~(d <= lim)
    if bool(bad.any()):
        i = int((d / lim).nan_to_num(posinf=1e30, nan=1e30).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()}, worst at {i}: {float(got.reshape(-1)[i])} against {float(ref.reshape(-1)[i])}, "
                             f"off by {float(d.reshape(-1)[i]):.3e}, limit {float(lim.reshape(-1)[i]):.3e}")


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (7, 64), (4, 200), (129, 80), (64, 256), (50, 59), (9, 1030), (2, 4097), (600, 10)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", SHAPES)
def test_pack_and_unpack_equal_the_definition(rows, C, dtype, fmt):
    from distill_bev_amd import act8 as A
    x = _data(rows, C, dtype, rows * 7 + C)
    ck = A.pack(x.to(DEV), fmt, -1)
    codes, scales = O.quantise(x, fmt)
    assert torch.equal(ck.scales.cpu(), scales) and torch.equal(ck.codes.cpu(), codes)
    ref = O.values(codes, scales, fmt)
    out = A.unpack(ck)
    assert out.dtype == dtype and out.shape == x.shape and torch.equal(out.cpu(), ref.to(dtype))
    assert torch.equal(A.unpack(ck, torch.float32).cpu().double(), ref)
    for other in DTYPES:
        assert torch.equal(A.unpack(ck, other).cpu(), ref.float().to(other))
    assert ck.nbytes == rows * C + rows * -(-C // 32)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_special_values(fmt):
    from distill_bev_amd import act8 as A
    fmax = torch.finfo(torch.float32).max
    x = torch.zeros(16, 64)
    x[1] = -0.0
    x[2, :32] = torch.linspace(-127.5, 127.5, 32)                      # ties and the clamp
    x[2, 32:] = torch.arange(32) + 0.5
    x[3, 5] = float("inf")
    x[4, 40] = float("-inf")
    x[5, 63] = float("nan")
    x[6] = fmax * torch.linspace(-1, 1, 64)
    x[7] = 1e-45 * torch.arange(64)                                     # subnormals
    x[8] = 2.0 ** -126 * torch.linspace(-1, 1, 64)
    x[9] = 1.75 * torch.linspace(-1, 1, 64)                             # 448 / 256: the largest that does not move the exponent
    x[10] = torch.nextafter(torch.tensor(1.75), torch.tensor(2.0)) * torch.linspace(-1, 1, 64)
    x[11] = 2.0 ** torch.arange(-32, 32)
    x[12, 0], x[12, 1:] = 1e4, 1e-3
    x[13] = 2.0 ** -120 * torch.linspace(-1, 1, 64)
    x[14] = (1 + 2.0 ** -4) * 2.0 ** torch.arange(-40, 24)              # ties of e4m3
    x[15] = torch.randn(64, generator=torch.Generator().manual_seed(1))
    ck = A.pack(x.to(DEV), fmt)
    codes, scales = O.quantise(x, fmt)
    assert torch.equal(ck.scales.cpu(), scales) and torch.equal(ck.codes.cpu().int() * (scales.repeat_interleave(32, 1) != 255),
                                                                codes.int() * (scales.repeat_interleave(32, 1) != 255))
    # (the value is rounded to fp32: the e4m3 neighbour of fp32's largest number is 2^128, an infinity there)
    out, ref = A.unpack(ck).cpu().double(), O.values(codes, scales, fmt).float().double()
    assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(out.nan_to_num(), ref.nan_to_num())
    assert bool(torch.isnan(out[3, :32]).all()) and bool((out[3, 32:] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_strides_and_alignment(dtype, fmt):
    from distill_bev_amd import act8 as A
    big = _data(60, 300, dtype, 3).to(DEV)
    views = {"columns": big[:, 3:131], "even columns": big[:, 2:98], "odd width": big[:, 1:60], "every second row": big[::2, :64],
             "transposed": big.t(), "expanded": big[:1].expand(7, 300), "three dimensions": big.view(6, 10, 300)[:, 1:9, 16:80],
             "one row": big[5:6, 7:77], "offset storage": big.view(-1)[5:5 + 64 * 9].view(9, 64)}
    for name, v in views.items():
        ck = A.pack(v, fmt, -1)
        ref = O.restored(v.cpu().reshape(-1, v.shape[-1]), fmt).view(v.shape)
        assert torch.equal(A.unpack(ck, torch.float32).cpu().double(), ref), name
    m = _data(2 * 5 * 7, 40, dtype, 4).to(DEV).view(2, 5, 7, 40).permute(0, 3, 1, 2)         # channels-last map
    ck = A.pack(m, fmt)
    out = A.unpack(ck)
    assert ck.dim == 1 and out.shape == m.shape and out.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(out.cpu().double(), O.restored(m.cpu().permute(0, 2, 3, 1).reshape(-1, 40), fmt).to(dtype).double().view(2, 5, 7, 40).permute(0, 3, 1, 2))
    assert A.pack(m.contiguous(), fmt).dim == 3
    for shape in ((0, 32), (4, 0), (2, 0, 5)):
        e = A.unpack(A.pack(torch.empty(shape, dtype=dtype, device=DEV), fmt, -1))
        assert e.shape == shape


def _act_bounds(z, act):
    a = z.abs()
    if act == "silu":
        s = torch.sigmoid(z)
        e = (1.5 * a + 8) * U
        return e * (z * s).abs(), s * e * (1 + a)
    if act == "gelu":
        q = 0.5 * torch.special.erfc(a / math.sqrt(2))
        phi = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        dq = q * (z * z + 16) * U + (z > 0) * 2 * U
        return a * dq + 2 * U * O.act(z, act)[0].abs(), dq + a * phi * (z * z + 6) * U + 2 * U
    return torch.zeros_like(z), torch.zeros_like(z)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", [(1, 1), (5, 33), (40, 64), (17, 200), (300, 59)])
def test_activation_forward_and_backward(rows, C, dtype, act, fmt):
    from distill_bev_amd import act8 as A
    x = _data(rows, C, dtype, C)
    gy = _data(rows, C, dtype, C + 1)
    leaf = x.to(DEV).requires_grad_(True)
    y = A.activation(leaf, act, fmt, -1)
    dx, = torch.autograd.grad(y, (leaf,), gy.to(DEV))
    assert y.dtype == dtype and dx.dtype == dtype and y.shape == x.shape
    z = x.double()
    zr = O.restored(x, fmt)
    ref, dref = O.act(z, act)[0], gy.double() * O.act(zr, act)[1]
    by, bd = _act_bounds(z, act)[0], gy.double().abs() * (_act_bounds(zr, act)[1] + 2 * U * O.act(zr, act)[1].abs())
    flush, gflush = z.abs() * 2.0 ** -126, gy.double().abs() * (1 + zr.abs()) * 2.0 ** -126
    _within(y, ref, 3 * by + flush + _half(ref, dtype), f"{act} forward")
    _within(dx, dref, 3 * bd + gflush + _half(dref, dtype), f"{act} backward")
    with torch.no_grad():
        assert torch.equal(A.activation(leaf, act, fmt, -1), y)          # without a gradient: the same values


def test_activation_tails_and_non_finite_values():
    from distill_bev_amd import act8 as A
    x = torch.cat([torch.linspace(-40, 40, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3e38, -3e38, float("inf"), float("nan")])]).view(1, -1)
    for act in ("silu", "gelu", "relu"):
        y = A.activation(x.to(DEV), act)
        ref = O.act(x.double(), act)[0]
        fin = torch.isfinite(ref)
        _within(y.cpu()[fin], ref[fin], (_act_bounds(x.double(), act)[0] * 3 + x.double().abs() * 2.0 ** -126 + _half(ref, torch.float32))[fin], act)
        # at +infinity the formulas' own limit (the library's CPU gelu gives a NaN there, so it is no reference)
        assert torch.equal(torch.isnan(y.cpu()), torch.isnan(ref)) and torch.equal(torch.isinf(y.cpu()), torch.isinf(ref.float()))


def test_activation_layouts_and_gradient_forms():
    from distill_bev_amd import act8 as A
    base = _data(2 * 6 * 5, 70, torch.float32, 5).to(DEV)
    m = base[:, :40].reshape(2, 6, 5, 40).permute(0, 3, 1, 2).requires_grad_(True)     # channels-last map
    y = A.activation(m, "silu", "int8")
    assert y.is_contiguous(memory_format=torch.channels_last)
    g, = torch.autograd.grad(y.sum(), (m,))                              # an expanded gradient
    zr = O.restored(m.detach().cpu().permute(0, 2, 3, 1).reshape(-1, 40), "int8")
    assert torch.allclose(g.cpu().permute(0, 2, 3, 1).reshape(-1, 40).double(), O.act(zr, "silu")[1], atol=2e-6, rtol=0)
    leaf = base.clone().requires_grad_(True)
    y = A.activation(leaf[:, 3:50], "gelu", "e4m3")                      # a strided input inside a graph
    g, = torch.autograd.grad(y, (leaf,), base[:, 10:57])                 # a strided gradient
    zr = O.restored(base[:, 3:50].cpu(), "e4m3")
    ref = torch.zeros(60, 70, dtype=torch.float64)
    ref[:, 3:50] = base[:, 10:57].cpu().double() * O.act(zr, "gelu")[1]
    assert torch.allclose(g.cpu().double(), ref, atol=1e-5, rtol=1e-6)
    e = torch.empty((0, 32), device=DEV, requires_grad=True)
    A.activation(e, "gelu").sum().backward()
    assert e.grad.shape == (0, 32)
    leaf = base.clone().requires_grad_(True)
    y = A.activation(leaf, "gelu", "int8")
    with torch.no_grad():
        leaf.mul_(2.0)                                                   # the checkpoint is kept, not the tensor: nothing to detect
    y.sum().backward()
    assert torch.allclose(leaf.grad.cpu().double(), O.act(O.restored(base.cpu(), "int8"), "gelu")[1], atol=2e-6, rtol=0)


WG = [(1, 1, 1), (1, 64, 64), (5, 3, 5), (31, 64, 63), (32, 65, 64), (33, 129, 127), (127, 128, 128), (129, 256, 10), (1000, 300, 200), (700, 512, 130),
      (4100, 96, 256), (2050, 257, 66), (900, 10, 256)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,Ci,Co", WG)
def test_weight_gradient(M, Ci, Co, dtype, fmt):
    from distill_bev_amd import act8 as A
    x, gy = _data(M, Ci, dtype, M + Ci), _data(M, Co, dtype, M + Co + 1)
    ck = A.pack(x.to(DEV), fmt, -1)
    gw, gb = A.weight_gradient(ck, gy.to(DEV), bias=True)
    xr, g = O.restored(x, fmt), gy.double()
    ref, refb = g.t() @ xr, g.sum(0)
    c = (8 + 4 * math.sqrt(3 * M)) * U
    bw, bb = c * (g.abs().t() @ xr.abs()), c * g.abs().sum(0)
    assert gw.dtype == dtype and gw.shape == (Co, Ci) and gb.shape == (Co,)
    _within(gw, ref, bw * (1 + c) + _half(ref, dtype) * (1 + c), "weight gradient")
    _within(gb, refb, bb * (1 + c) + _half(refb, dtype), "bias gradient")
    assert torch.equal(A.weight_gradient(ck, gy.to(DEV)), gw)            # fixed order, with and without the bias


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,Ci,Co", [(64, 96, 33), (517, 130, 65), (2000, 64, 200)])
def test_weight_gradient_of_whole_numbers_is_exact(M, Ci, Co, dtype):
    """whole numbers up to 127 are their own checkpoint when a block holds a 64..127; sums below 2^24 (2^8 for bf16, 2^11 for fp16 outputs
    are rounded once): every index and every share has to be right"""
    from distill_bev_amd import act8 as A
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-9, 10, (M, Ci), generator=g).float()
    x[:, ::32] = 100
    gy = torch.randint(-8, 9, (M, Co), generator=g).float()
    gw, gb = A.weight_gradient(A.pack(x.to(DEV, dtype), "int8", -1), gy.to(DEV, dtype), bias=True)
    assert torch.equal(gw.cpu(), (gy.double().t() @ x.double()).to(dtype)) and torch.equal(gb.cpu(), gy.double().sum(0).to(dtype))


def test_weight_gradient_keeps_every_bit_of_an_fp32_gradient():
    from distill_bev_amd import act8 as A
    M, C = 128, 64
    x = torch.zeros(M, C)
    x[torch.arange(C) * 2, torch.arange(C)] = 1.0                         # one row per channel
    gy = _data(M, 40, torch.float32, 9)
    gw = A.weight_gradient(A.pack(x.to(DEV), "int8", -1), gy.to(DEV))
    assert torch.equal(gw.cpu(), gy[::2].t())
    gy16 = gy.half()
    assert torch.equal(A.weight_gradient(A.pack(x.to(DEV).half(), "e4m3", -1), gy16.to(DEV)).cpu(), gy16[::2].t())


def test_weight_gradient_non_finite_empty_and_layouts():
    from distill_bev_amd import act8 as A
    M, Ci, Co = 200, 70, 40
    x, gy = _data(M, Ci, torch.float32, 1).abs() + 0.5, _data(M, Co, torch.float32, 2)
    x[7, 40] = float("nan")                                               # channels 32..63 of the checkpoint's row 7
    gy[11, 3], gy[12, 5], gy[13, 6], gy[14, 8] = float("inf"), float("-inf"), float("nan"), 3.4e38
    gw, gb = A.weight_gradient(A.pack(x.to(DEV), "int8", -1), gy.to(DEV), bias=True)
    gw, gb = gw.cpu(), gb.cpu()
    assert bool(torch.isnan(gw[:, 32:64]).all())
    rest = [c for c in range(Ci) if not 32 <= c < 64]
    assert bool((gw[3][rest] == float("inf")).all()) and bool((gw[5][rest] == float("-inf")).all()) and bool(torch.isnan(gw[6][rest]).all())
    ok = [r for r in range(Co) if r not in (3, 5, 6, 8)]
    assert bool(torch.isfinite(gw[ok][:, rest]).all())
    assert gb[3] == float("inf") and gb[5] == float("-inf") and bool(torch.isnan(gb[6])) and bool(torch.isfinite(gb[8]))
    gw, gb = A.weight_gradient(A.pack(torch.empty((0, 48), device=DEV), "int8", -1), torch.empty((0, 20), device=DEV), bias=True)
    assert torch.equal(gw, torch.zeros_like(gw)) and torch.equal(gb, torch.zeros_like(gb))
    x, gy = _data(60, 48, torch.float32, 3).to(DEV), _data(60, 90, torch.float32, 4).to(DEV)
    a = A.weight_gradient(A.pack(x, "int8", -1), gy[:, 11:50])            # a strided gradient
    assert torch.equal(a, A.weight_gradient(A.pack(x, "int8", -1), gy[:, 11:50].contiguous()))
    m = x.view(3, 4, 5, 48).permute(0, 3, 1, 2)
    gm = gy[:, 11:50].reshape(3, 4, 5, 39).permute(0, 3, 1, 2)
    assert torch.equal(A.weight_gradient(A.pack(m, "int8", 1), gm), a)    # the same rows as a map
    with pytest.raises(ValueError):
        A.weight_gradient(A.pack(x, "int8", -1), gy[:59])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("shape,Co", [((7, 33), 20), ((3, 50, 64), 128), ((4096, 64), 128), ((60000, 128), 128)])
def test_linear_layer(shape, Co, fmt):
    """forward and data gradient are the layer's ordinary products; weight and bias gradient those of the checkpoint.  (The last size takes
    the bf16x6 products.)"""
    from distill_bev_amd import act8 as A
    torch.manual_seed(0)
    x = torch.randn(*shape)
    mod = nn.Linear(shape[-1], Co)
    xl = x.to(DEV).requires_grad_(True)
    w, b = mod.weight.detach().to(DEV).requires_grad_(True), mod.bias.detach().to(DEV).requires_grad_(True)
    gy = torch.randn(*shape[:-1], Co)
    y = A.linear(xl, w, b, fmt)
    gx, gw, gb = torch.autograd.grad(y, (xl, w, b), gy.to(DEV))
    x2, g2 = x.reshape(-1, shape[-1]).double(), gy.reshape(-1, Co).double()
    wd = mod.weight.detach().double()
    rel = lambda a, r: float((a.detach().cpu().double() - r).norm() / r.norm())    # noqa: E731
    assert rel(y.reshape(-1, Co), x2 @ wd.t() + mod.bias.detach().double()) < 2e-6
    assert rel(gx.reshape(-1, shape[-1]), g2 @ wd) < 2e-6
    assert rel(gw, g2.t() @ O.restored(x2, fmt)) < 2e-6 and rel(gb, g2.sum(0)) < 2e-6
    frozen = A.linear(xl, w.detach(), b, fmt)                             # only the bias and the input want gradients
    gx2, gb2 = torch.autograd.grad(frozen, (xl, b), gy.to(DEV))
    assert torch.equal(frozen, y) and torch.equal(gx2, gx) and rel(gb2, g2.sum(0)) < 2e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_conv1x1_layer(dtype):
    from distill_bev_amd import act8 as A
    torch.manual_seed(1)
    x = torch.randn(3, 40, 9, 7).to(dtype)
    w, b = (torch.randn(24, 40, 1, 1) * 0.2).to(dtype), torch.randn(24).to(dtype)
    gy = torch.randn(3, 24, 9, 7).to(dtype)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = A.conv1x1(*leaves, "int8")
    gx, gw, gb = torch.autograd.grad(y, leaves, gy.to(DEV))
    rows = lambda t: t.double().permute(0, 2, 3, 1).reshape(-1, t.shape[1])     # noqa: E731
    tol = 3 * torch.finfo(dtype).eps + 2e-6
    rel = lambda a, r: float((a.detach().cpu().double() - r).norm() / r.norm())    # noqa: E731
    assert y.is_contiguous(memory_format=torch.channels_last)
    assert rel(rows(y.detach().cpu()), rows(x) @ w.double().view(24, 40).t() + b.double()) < tol
    assert rel(rows(gx.cpu()), rows(gy) @ w.double().view(24, 40)) < tol and gx.shape == x.shape
    assert gw.shape == w.shape and rel(gw.view(24, 40), rows(gy).t() @ O.restored(rows(x).to(dtype), "int8")) < tol
    assert rel(gb, rows(gy).sum(0)) < tol
    with pytest.raises(ValueError):
        A.conv1x1(leaves[0], torch.randn(4, 40, 3, 3, device=DEV, dtype=dtype))
    from distill_bev_amd import _lib as L
    with pytest.raises(L.DbevHipError):
        A.conv1x1(leaves[0], leaves[1].double())


def test_feed_forward_block_as_a_model_uses_it():
    """use_act8 on a Linear -> GELU -> Linear block with a skip connection: forward equals the stock modules', gradients equal the oracle's
    (which takes the same checkpoints), memory kept between forward and backward falls"""
    from distill_bev_amd import act8 as A

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.net = nn.Sequential(nn.Linear(64, 192), nn.GELU(), nn.Linear(192, 64))

        def forward(self, x):
            return x + self.net(x)

    torch.manual_seed(3)
    stock, mod = Block(), Block()
    mod.load_state_dict(stock.state_dict())
    stock, mod = stock.to(DEV), mod.to(DEV)
    assert A.use_act8(mod, "int8") == 3 and list(mod.state_dict()) == list(stock.state_dict())
    x = torch.randn(2, 500, 64)
    xa, gy = x.to(DEV).requires_grad_(True), torch.randn(2, 500, 64)
    y = mod(xa)
    assert torch.allclose(y, stock(x.to(DEV)), atol=2e-5)
    y.backward(gy.to(DEV))
    xd = x.double().reshape(-1, 64).requires_grad_(True)
    p = [t.detach().cpu().double().requires_grad_(True) for t in stock.parameters()]
    h = O.LinearFn.apply(xd, p[0], p[1], "int8")
    out = xd + O.LinearFn.apply(O.ActFn.apply(h, "gelu", "int8"), p[2], p[3], "int8")
    out.backward(gy.double().reshape(-1, 64))
    # A hidden value within its fp32 error e of a code border may take the neighbouring code: a share 2 e / step of the values, each off by
    # one step, moves a gradient by sqrt(2 e / step) * step = sqrt(2 e step) of its norm.  In units of the spread e <= 1e-6 (64 to 192
    # products and the activation) and step <= 1 / 32 (a largest value of 2 to 4 spreads / 64): 2.5e-4.
    rel = lambda a, r: float((a.detach().cpu().double().reshape(r.shape) - r).norm() / r.norm())      # noqa: E731
    assert rel(xa.grad, xd.grad) < 2.5e-4
    for q, r in zip(mod.parameters(), p):
        assert rel(q.grad, r.grad) < 2.5e-4

    def kept(m):
        held = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append((t.untyped_storage().data_ptr(), t.untyped_storage().nbytes())) or t, lambda t: t):
            m(x.to(DEV).requires_grad_(True))
        own = {q.untyped_storage().data_ptr() for q in m.parameters()}
        return sum({a: b for a, b in held if a not in own}.values())

    assert kept(mod) < 0.3 * kept(stock)
    mod.eval()
    with torch.no_grad():
        assert torch.allclose(mod(x.to(DEV)), stock(x.to(DEV)), atol=2e-5)


def test_ineligible_device_tensors_take_the_stock_modules_and_are_counted():
    from distill_bev_amd import _lib as L
    from distill_bev_amd import act8 as A
    import warnings
    m = nn.Sequential(nn.Linear(8, 4), nn.SiLU()).to(DEV).double()
    A.use_act8(m)
    L.fallback_reset()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        m(torch.randn(3, 8, device=DEV, dtype=torch.float64)).sum().backward()
    assert L.fallback_counts()["act8"] == 2
    L.fallback_reset()


def test_other_streams_and_graph_replays():
    """on a stream of its own, and captured: forward, backward and weight gradient replayed on new inputs with eager work between"""
    from distill_bev_amd import act8 as A
    torch.manual_seed(4)
    xs = [torch.randn(300, 256, device=DEV) for _ in range(4)]             # (256 channels: the largest tile, more than 64 KB of LDS)
    gs = [torch.randn(300, 256, device=DEV) for _ in range(4)]

    def step(x, g):
        leaf = x.detach().requires_grad_(True)
        y = A.activation(leaf, "gelu", "int8")
        dx, = torch.autograd.grad(y, (leaf,), g)
        gw, gb = A.weight_gradient(A.pack(x, "e4m3", -1), g, bias=True)
        return y.detach(), dx, gw, gb

    eager = [step(x, g) for x, g in zip(xs, gs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = step(xs[1], gs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(out, eager[1]))
    sx, sg = xs[0].clone(), gs[0].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(sx, sg)
    for i in (1, 2, 3, 0, 2):
        sx.copy_(xs[i])
        sg.copy_(gs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager[i]))
        again = step(xs[3 - i], gs[3 - i])
        assert all(torch.equal(a, b) for a, b in zip(again, eager[3 - i]))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_more_than_two_to_the_31_values(fmt):
    """offsets beyond 32 bits: the last rows of a tensor of 2^31 + 2^20 values equal those of a call on them alone"""
    from distill_bev_amd import act8 as A
    rows, C = (1 << 25) + (1 << 14) + 3, 64
    x = torch.empty((rows, C), dtype=torch.bfloat16, device=DEV)
    x[:-1000].fill_(0.5)
    x[-1000:] = _data(1000, C, torch.bfloat16, 1).to(DEV)
    ck, tail = A.pack(x, fmt, -1), A.pack(x[-1000:], fmt, -1)
    assert torch.equal(ck.codes[-1000:], tail.codes) and torch.equal(ck.scales[-1000:], tail.scales)
    out = A.unpack(ck)
    assert torch.equal(out[-1000:], A.unpack(tail)) and bool((out[:1000] == 0.5).all())
    del out, ck
    leaf = x.requires_grad_(True)
    y = A.activation(leaf, "silu", fmt, -1)
    gy = torch.ones((1, 1), dtype=torch.bfloat16, device=DEV).expand(rows, C).contiguous()
    dx, = torch.autograd.grad(y, (leaf,), gy)
    small = x[-1000:].detach().requires_grad_(True)
    ys = A.activation(small, "silu", fmt, -1)
    assert torch.equal(y[-1000:], ys) and torch.equal(dx[-1000:], torch.autograd.grad(ys, (small,), gy[-1000:])[0])
    # the reduction over as many rows: ones against ones and the tail's own sums
    ck = A.pack(x.detach(), fmt, -1)
    g = torch.zeros((rows, 8), dtype=torch.bfloat16, device=DEV)
    g[-1000:, :] = 1.0
    gw, gb = A.weight_gradient(ck, g, bias=True)
    ref = A.unpack(tail, torch.float32).double().sum(0)
    assert float((gw.double() - ref).abs().max()) <= float(ref.abs().max()) * 2.0 ** -8 and bool((gb == 1000).all())


@pytest.mark.parametrize("M,Ci,Co", [(40, 8, 70001), (40, 70004, 6), (70, 66000, 3)])
def test_weight_gradient_of_wide_layers(M, Ci, Co):
    """rows of more than 2^16 values; whole numbers, so that every product and sum is exact"""
    from distill_bev_amd import act8 as A
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-60, 61, (M, Ci), generator=g).float()
    x[:, ::32] = 64.0                                                      # every block's largest value: 2^k = 1
    gy = torch.randint(-9, 10, (M, Co), generator=g).float()
    gw, gb = A.weight_gradient(A.pack(x.to(DEV), "int8", -1), gy.to(DEV), bias=True)
    assert torch.equal(gw.cpu(), gy.t() @ x) and torch.equal(gb.cpu(), gy.sum(0))


@pytest.mark.parametrize("n", [(1 << 24) + 33, (1 << 24) + 64])
def test_one_very_long_row(n):
    """a flat tensor: the same blocks as its values in rows of 32 (odd length: single values a lane, more than 2^16 column ranges)"""
    from distill_bev_amd import act8 as A
    x = torch.randn(n, device=DEV, generator=torch.Generator(DEV).manual_seed(6))
    ck, m = A.pack(x, "int8"), n // 32 * 32
    rows = A.pack(x[:m].view(-1, 32), "int8", -1)
    assert ck.rows == 1 and ck.C == n
    assert torch.equal(ck.codes[0, :m], rows.codes.reshape(-1)) and torch.equal(ck.scales[0, :m // 32], rows.scales.reshape(-1))
    back = A.unpack(ck)
    assert torch.equal(back[:m], A.unpack(rows).reshape(-1))
    if n > m:
        tail = A.unpack(A.pack(x[m:].view(1, -1), "int8", -1)).reshape(-1)
        assert torch.equal(back[m:], tail)
    leaf = x.requires_grad_(True)
    y = A.activation(leaf, "silu", "int8")
    gy = torch.ones(n, device=DEV)
    dx, = torch.autograd.grad(y, (leaf,), gy)
    part = x[:m].detach().view(-1, 32).requires_grad_(True)
    yp = A.activation(part, "silu", "int8", -1)
    assert torch.equal(y[:m], yp.reshape(-1)) and torch.equal(dx[:m], torch.autograd.grad(yp, (part,), gy[:m].view(-1, 32))[0].reshape(-1))


def test_layers_without_gradients_keep_nothing_and_refuse_autocast():
    from distill_bev_amd import _lib as L
    from distill_bev_amd import act8 as A
    torch.manual_seed(7)
    lin, conv = nn.Linear(64, 24).to(DEV), nn.Conv2d(64, 24, 1).to(DEV)
    x, m = torch.randn(50, 64, device=DEV), torch.randn(2, 64, 5, 5, device=DEV).contiguous(memory_format=torch.channels_last)
    packs = []
    pack, A.pack = A.pack, lambda *a: packs.append(a) or pack(*a)
    try:
        with torch.no_grad():
            y, z = A.linear(x, lin.weight, lin.bias), A.conv1x1(m, conv.weight, conv.bias)
        assert not packs and not y.requires_grad and not z.requires_grad
        assert torch.equal(y, A.linear(x, lin.weight, lin.bias)) and torch.equal(z, A.conv1x1(m, conv.weight, conv.bias)) and len(packs) == 2
    finally:
        A.pack = pack
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with pytest.raises(L.DbevHipError):
            A.linear(x, lin.weight, lin.bias)
        with pytest.raises(L.DbevHipError):
            A.conv1x1(m, conv.weight, conv.bias)
    wide = torch.empty((1, 8), device=DEV).expand((1 << 20) + 1, 8).requires_grad_(True)
    with pytest.raises(L.DbevHipError):                                    # before the product, not in the backward pass
        A.linear(x[:, :8], wide)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tensors_beyond_the_caches_equal_their_parts(dtype, fmt):
    """above 192 MB the accesses are other instructions: the same bits as for the two halves, which stay below"""
    from distill_bev_amd import act8 as A
    C = 512
    rows = (208 << 20) // (C * torch.finfo(dtype).bits // 8)
    x = torch.randn((rows, C), device=DEV, generator=torch.Generator(DEV).manual_seed(8)).to(dtype)
    gy = torch.randn((rows, C), device=DEV, generator=torch.Generator(DEV).manual_seed(9)).to(dtype)

    def run(x, gy):
        ck = A.pack(x, fmt, -1)
        leaf = x.requires_grad_(True)
        y = A.activation(leaf, "gelu", fmt, -1)
        return ck.codes, ck.scales, A.unpack(ck), y.detach(), torch.autograd.grad(y, (leaf,), gy)[0]

    whole, h = run(x.clone(), gy), rows // 2
    parts = [run(x[:h].clone(), gy[:h]), run(x[h:].clone(), gy[h:])]
    for i, t in enumerate(whole):
        assert torch.equal(t[:h], parts[0][i]) and torch.equal(t[h:], parts[1][i]), i


def test_silu_of_positive_bf16_values_is_correctly_rounded():
    """y = z (1 - q), q = sigmoid(-z).  q is off by (1.5 z + 8) U of itself (exp2's argument, exp2, 1 +, reciprocal, product), which is q / (1 - q)
    times that of y; 1 - q is rounded by half a step of [1/2, 1), 2^-25; the product by half a step of fp32, U / mantissa of y.  A tie of bf16
    is an fp32 value, so wherever the exact y is further than these from the nearest tie the result is the exact one's.  That
    leaves out 2^-7 alone (there y = z / 2 + z^2 / 4 to 2e-8, a tie); the closest of the others is 5.9375, 9.5e-8 from one"""
    from distill_bev_amd import act8 as A
    x = torch.arange(0x0080, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)               # every positive normal value
    z = x.double()
    q = torch.sigmoid(-z)
    y = z * (1 - q)
    m = torch.frexp(y)[0] * 256
    tie = (m - torch.floor(m) - 0.5).abs() / m
    sure = tie > q / (1 - q) * (1.5 * z + 8) * U + 0.5 * U / (1 - q) + U / (m / 128)
    assert bool(sure[x == 5.9375]) and int((~sure).sum()) == 1
    got = A.activation(x.to(DEV), "silu").cpu()
    assert torch.equal(got[sure], y.to(torch.bfloat16)[sure])


def _kept_bytes(run, own):
    """bytes of the tensors that `run` saves for its backward pass, storages counted once, those of `own` left out"""
    held = {}

    def save(t):
        held[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
        keep.append(t)                                                     # (no address is used twice)
        return t

    keep = []
    with torch.autograd.graph.saved_tensors_hooks(save, lambda t: t):
        out = run()
    skip = {q.untyped_storage().data_ptr() for q in own}
    return out, sum(b for a, b in held.items() if a not in skip)


@pytest.mark.parametrize("inplanes,planes,n,h,w", [(256, 64, 4, 120, 120), (96, 32, 4, 280, 281)])
def test_bottleneck_keeps_its_one_by_one_inputs_in_8_bits(inplanes, planes, n, h, w):
    """nets.Bottleneck runs its 1x1 convolutions without their modules' forward, with the norm's statistics from the product's epilogue (bf16x6
    in the first case, the fp32 GEMM in the second): both inputs are kept as checkpoints, the output is the same bits, and a layer's weight
    gradient is the checkpoint's"""
    from distill_bev_amd import act8 as A
    from distill_bev_amd import bn_act as BA
    from distill_bev_amd import gemm_bf6 as G
    from distill_bev_amd import nets
    from distill_bev_amd.train_step import to_channels_last
    x = torch.randn(n, inplanes, h, w, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(memory_format=torch.channels_last)
    gy = torch.randn(n, 4 * planes, h, w, device=DEV, generator=torch.Generator(DEV).manual_seed(2)).to(memory_format=torch.channels_last)

    def one(fmt):
        torch.manual_seed(3)
        ds = None if inplanes == 4 * planes else nn.Sequential(nn.Conv2d(inplanes, 4 * planes, 1, bias=False), nn.BatchNorm2d(4 * planes))
        m = nets.Bottleneck(inplanes, planes, downsample=ds).to(DEV).train()
        to_channels_last(m, fmt)
        leaf = x.clone().requires_grad_(True)
        y, kept = _kept_bytes(lambda: m(leaf), list(m.parameters()) + list(m.buffers()))
        y.backward(gy)
        return m, y.detach(), kept, leaf.grad, {k: q.grad for k, q in m.named_parameters()}

    mod, y, kept, gx, grads = one(None)
    m8, y8, kept8, gx8, grads8 = one("int8")
    assert m8.act8_modules == (2 if inplanes == 4 * planes else 3) and torch.equal(y, y8)
    M, inputs = n * h * w, {(256, 64): 256 + 64, (96, 32): 96 + 32}[(inplanes, planes)]     # (conv1 and the downsample share one fp32 input)
    codes = inputs + (0 if inplanes == 4 * planes else 96)
    assert kept - kept8 >= M * (4 * inputs - 33 / 32 * codes) - (1 << 16), (kept, kept8)
    # relative error of a kept value 2^-7 of its block's largest (3 spreads or less): a hundredth at random signs
    for k in grads:
        assert float((grads[k] - grads8[k]).norm()) < 0.03 * float(grads[k].norm()), k
    assert float((gx - gx8).norm()) < 1e-5 * float(gx.norm())              # the data gradients do not see the checkpoint
    conv, bn = m8.conv1, getattr(m8, m8.norm1_name)
    kernel = "bf6" if G.eligible(x, conv.weight) else "f32"
    assert kernel == ("bf6" if inplanes == 256 else "f32") and (kernel == "bf6" or BA.conv1x1_bn_ready(conv, bn, x)) and A.keeps(conv, x)
    gz = gy[:, :planes].contiguous(memory_format=torch.channels_last)
    leaf = x.clone().requires_grad_(True)
    z, rows = nets._conv1x1_stats(conv, bn, leaf)
    a = torch.autograd.grad(z, (leaf, conv.weight), gz)
    conv.act8_format = None                                                 # the same layer without a checkpoint
    z0, rows0 = nets._conv1x1_stats(conv, bn, leaf)
    b = torch.autograd.grad(z0, (leaf, conv.weight), gz)
    assert torch.equal(z, z0) and torch.equal(rows, rows0) and not rows.requires_grad
    assert float((a[0] - b[0]).norm()) <= 1e-6 * float(b[0].norm())
    assert torch.equal(a[1].view(planes, inplanes), A.weight_gradient(A.pack(x, "int8", 1), gz))
    with torch.no_grad():
        assert torch.equal(nets._conv1x1_stats(conv, bn, x)[0], z)
    m8.eval()
    with torch.no_grad():
        assert torch.equal(m8(x), mod.eval()(x))


@pytest.mark.parametrize("n,h,w", [(2, 9, 11), (4, 120, 120)])
def test_biased_one_by_one_layers_of_an_accelerated_model(n, h, w):
    """BiasSumConv2d alone and in front of a BatchNorm that cancels its bias, in sizes of the library's product and of the bf16x6 GEMM's: the input
    is kept in 8 bits, the forward pass is that of the layer without a checkpoint"""
    from distill_bev_amd import act8 as A
    from distill_bev_amd import colsum
    from distill_bev_amd.detectors import ThreeLayer
    from distill_bev_amd.train_step import to_channels_last
    x = torch.randn(n, 64, h, w, device=DEV, generator=torch.Generator(DEV).manual_seed(4)).to(memory_format=torch.channels_last)
    gy = torch.randn(n, 64, h, w, device=DEV, generator=torch.Generator(DEV).manual_seed(5)).to(memory_format=torch.channels_last)

    def one(build, fmt):
        torch.manual_seed(6)
        m = build().to(DEV).train()
        to_channels_last(m, fmt)
        leaf = x.clone().requires_grad_(True)
        y, kept = _kept_bytes(lambda: m(leaf), list(m.parameters()) + list(m.buffers()))
        y.backward(gy)
        return m, y.detach(), kept, leaf.grad, {k: q.grad for k, q in m.named_parameters()}

    for build, layers in ((lambda: nn.Sequential(nn.Conv2d(64, 64, 1)), 1), (lambda: ThreeLayer(64, 64, 64, kernel_size=1, stride=1), 3)):
        mod, y, kept, gx, grads = one(build, None)
        m8, y8, kept8, gx8, grads8 = one(build, "e4m3")
        convs = [m for m in m8.modules() if isinstance(m, nn.Conv2d)]
        assert m8.act8_modules == 0 and m8.act8_bias_convs == layers == len(convs) and all(type(m) is colsum.BiasSumConv2d for m in convs)
        assert torch.allclose(y8, y, rtol=0, atol=2e-6 * float(y.abs().max()))                # (the bias is added in another place)
        assert kept - kept8 >= layers * n * h * w * 64 * (4 - 33 / 32) - (1 << 12), (kept, kept8)
        assert float((gx - gx8).norm()) < 1e-5 * float(gx.norm())
        for k in grads:                          # e4m3: at most 2^-4 of each value, random signs
            if layers == 1 or not k.startswith("conv") or not k.endswith("bias"):
                assert float((grads[k] - grads8[k]).norm()) < 0.05 * float(grads[k].norm()), k
        if layers == 1:
            gw, gb = A.weight_gradient(A.pack(x, "e4m3", 1), gy, bias=True)
            assert torch.equal(grads8["0.weight"].view(64, 64), gw) and torch.equal(grads8["0.bias"], gb)
    assert A.use_act8(m8, "e4m3") == 0
