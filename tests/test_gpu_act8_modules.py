"""GPU: the modules of act8.py and gn_act.py where the kernels do not take a call -- they compute what the stock modules compute -- and what the
functions refuse."""
import warnings

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _stock(mod, *args):
    """mod's result, the ledger's counts of it"""
    from distill_bev_amd import _lib as L
    L.fallback_reset()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        out = mod(*args)
    counts = L.fallback_counts()
    L.fallback_reset()
    return out, counts


def test_modules_beyond_the_limits_take_the_stock_operators():
    from distill_bev_amd import act8 as A
    from distill_bev_amd import gn_act as GN
    gn = GN.GroupNormAct(4, 1 << 17, act="silu", checkpoint="int8").to(DEV)
    x = torch.randn(2, 1 << 17, device=DEV)
    y, n = _stock(gn, x)
    assert n["gn_act"] == 1 and torch.allclose(y, F.silu(F.group_norm(x, 4)), atol=1e-5)
    lin = nn.Linear(8, (1 << 20) + 1).to(DEV)
    ref = lin(torch.ones(3, 8, device=DEV))
    A.use_act8(lin)
    assert type(lin) is A.Act8Linear
    y, n = _stock(lin, torch.ones(3, 8, device=DEV))
    assert n["act8"] == 1 and torch.allclose(y, ref, atol=1e-5)
    conv = nn.Conv2d(8, (1 << 20) + 1, 1).to(DEV)
    A.use_act8(conv)
    y, n = _stock(conv, torch.ones(1, 8, 2, 2, device=DEV))
    assert n["act8"] == 1 and y.shape == (1, (1 << 20) + 1, 2, 2)


def _net():
    from distill_bev_amd import act8 as A
    from distill_bev_amd import gn_act as GN
    torch.manual_seed(1)
    stock = nn.Sequential(nn.Conv2d(16, 32, 1), nn.GroupNorm(4, 32), nn.SiLU(), nn.Flatten(2), nn.GELU(), nn.Linear(35, 24))
    mod = nn.Sequential(nn.Conv2d(16, 32, 1), nn.GroupNorm(4, 32), nn.SiLU(), nn.Flatten(2), nn.GELU(), nn.Linear(35, 24))
    mod.load_state_dict(stock.state_dict())
    stock, mod = stock.to(DEV), mod.to(DEV).to(memory_format=torch.channels_last)
    assert GN.fuse_gn_act_modules(mod, "int8") == 1 and A.use_act8(mod, "int8") == 3
    x = torch.randn(2, 16, 5, 7, device=DEV).to(memory_format=torch.channels_last)
    return stock, mod, x


def test_forward_mode_derivatives_pass_through_the_modules_and_are_refused_by_the_functions():
    import torch.autograd.forward_ad as fw
    from distill_bev_amd import _lib as L
    from distill_bev_amd import act8 as A
    from distill_bev_amd import gn_act as GN
    stock, mod, x = _net()
    for m in (stock, mod):
        m.requires_grad_(False)                                            # a frozen network: nothing requires grad
    t = torch.randn_like(x)
    with fw.dual_level():
        ref = fw.unpack_dual(stock(fw.make_dual(x, t)))
        (out, n) = _stock(mod, fw.make_dual(x, t))
        out = fw.unpack_dual(out)
        assert out.tangent is not None and torch.allclose(out.primal, ref.primal, atol=1e-5) and torch.allclose(out.tangent, ref.tangent, atol=1e-5)
        assert n["gn_act"] == 1
        d = fw.make_dual(x, t)
        rows = fw.make_dual(torch.randn(6, 32, device=DEV), torch.randn(6, 32, device=DEV))
        with pytest.raises(NotImplementedError):
            GN.group_norm_act(d, 4)
        for call in (lambda: A.activation(rows), lambda: A.linear(rows, torch.randn(8, 32, device=DEV)),
                     lambda: A.conv1x1(d, torch.randn(8, 16, 1, 1, device=DEV))):
            with pytest.raises(NotImplementedError):
                call()
        with pytest.raises(L.DbevHipError):
            A.pack(rows)
        plain, lw = torch.randn(6, 32, device=DEV), torch.randn(8, 32, device=DEV, requires_grad=True)
        a = A.linear(plain, lw)                                            # (nothing here is a dual tensor)
        assert torch.autograd.grad(a.sum(), (lw,))[0].shape == lw.shape and A.unpack(A.pack(plain)).shape == plain.shape
    jvp = torch.func.jvp(lambda v: _stock(mod, v)[0], (x,), (t,))
    assert torch.allclose(jvp[1], ref.tangent, atol=1e-5)
    params = dict(mod.named_parameters())
    grads = torch.func.grad(lambda p: torch.func.functional_call(mod, p, (x,)).square().sum())(params)
    want = torch.autograd.grad(stock.requires_grad_(True)(x).square().sum(), list(stock.parameters()))
    for g, w in zip(grads.values(), want):
        assert torch.allclose(g, w.view(g.shape), rtol=1e-4, atol=1e-4 * float(w.abs().max()))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: GN.group_norm_act(v, 4).sum())(x)


@pytest.mark.parametrize("grad", [False, True])
def test_modules_trace_as_the_stock_operators_and_functions_refuse(grad):
    from distill_bev_amd import _lib as L
    from distill_bev_amd import act8 as A
    from distill_bev_amd import gn_act as GN
    stock, mod, x = _net()
    for m in (stock, mod):
        m.requires_grad_(grad)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(mod, (x,))
        other = torch.randn_like(x)
        assert torch.allclose(traced(other), stock(other), atol=1e-5)
        rows = torch.randn(6, 32, device=DEV)
        w, lw = torch.randn(16, device=DEV, requires_grad=grad), torch.randn(8, 32, device=DEV, requires_grad=grad)
        cw = torch.randn(4, 16, 1, 1, device=DEV, requires_grad=grad)
        for f, a in ((lambda v: GN.group_norm_act(v, 4, w, act="silu", checkpoint="int8"), x), (lambda v: A.activation(v, "gelu"), rows),
                     (lambda v: A.linear(v, lw), rows), (lambda v: A.conv1x1(v, cw), x), (lambda v: A.unpack(A.pack(v)), rows)):
            f(a)
            with pytest.raises(L.DbevHipError, match="trace"):
                torch.jit.trace(f, (a,), check_trace=False)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("layout", [torch.channels_last, torch.contiguous_format])
def test_second_derivatives_without_a_checkpoint(act, layout):
    """a gradient penalty through group_norm_act equals the stock operators' in 64 bits (fp32 sums of 60 to 480 terms: 1e-5 of the norm); from a
    checkpoint there is none"""
    from distill_bev_amd import gn_act as GN
    torch.manual_seed(2)
    x, w, b, gy = torch.randn(2, 16, 5, 6), 1 + 0.2 * torch.randn(16), 0.2 * torch.randn(16), torch.randn(2, 16, 5, 6)
    stock = {"none": lambda t: t, "silu": F.silu, "gelu": F.gelu}[act]

    def penalty(f, leaves, g):
        first = torch.autograd.grad(f(*leaves), leaves, g, create_graph=True)
        second = torch.autograd.grad(sum(t.square().sum() for t in first), leaves, allow_unused=True)
        return [torch.zeros_like(t) if s is None else s for t, s in zip(leaves, second)]      # (the bias has none without an activation)

    ref = penalty(lambda x, w, b: stock(F.group_norm(x, 4, w, b)), [t.double().requires_grad_(True) for t in (x, w, b)], gy.double())
    leaves = [x.to(DEV).to(memory_format=layout).requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    got = penalty(lambda x, w, b: GN.group_norm_act(x, 4, w, b, act=act), leaves, gy.to(DEV))
    for a, r in zip(got, ref):
        assert float((a.cpu().double() - r).norm()) <= 1e-5 * float(r.norm())
    mod = GN.GroupNormAct(4, 16, act=act).to(DEV)
    torch.autograd.grad(torch.autograd.grad(mod(leaves[0]).square().sum(), (leaves[0],), create_graph=True)[0].square().sum(), (leaves[0],))
    with pytest.raises(RuntimeError):
        penalty(lambda x, w, b: GN.group_norm_act(x, 4, w, b, act=act, checkpoint="int8"), leaves, gy.to(DEV))


def test_modules_give_the_layout_that_they_were_given():
    """channels-last maps stay channels-last; a dense tensor of another layout comes out contiguous, by the stock operator unless a checkpoint is kept"""
    from distill_bev_amd import _lib as L
    from distill_bev_amd import gn_act as GN
    torch.manual_seed(3)
    for shape, fmt in (((2, 16, 7), None), ((2, 16, 5, 6), None), ((2, 16, 3, 4, 5), None), ((2, 16), None),
                       ((2, 16, 5, 6), torch.channels_last), ((2, 16, 3, 4, 5), torch.channels_last_3d)):
        x = torch.randn(shape, device=DEV)
        x = (x if fmt is None else x.contiguous(memory_format=fmt)).requires_grad_(True)
        gy = torch.randn(shape, device=DEV)
        dense = fmt is None and len(shape) > 2
        for ck in (None, "int8"):
            mod = GN.GroupNormAct(4, 16, act="silu", checkpoint=ck).to(DEV)
            y, n = _stock(mod, x)
            ref = F.silu(F.group_norm(x, 4, mod.weight, mod.bias))
            assert torch.allclose(y, ref, atol=1e-5) and n["gn_act"] == int(dense and ck is None)
            assert y.is_contiguous() if fmt is None else y.is_contiguous(memory_format=fmt)
            if fmt is None:
                y.view(-1)
            with torch.no_grad():
                y, n = _stock(mod, x)                                      # nothing to keep
                assert torch.allclose(y, ref, atol=1e-5) and n["gn_act"] == int(dense)
            a, = torch.autograd.grad(mod(x), (x,), gy)
            b, = torch.autograd.grad(ref, (x,), gy)
            # a checkpoint's values are off by 2^-7 of their block's largest at most (some 3 spreads)
            assert float((a - b).norm()) < (1e-5 if ck is None else 0.03) * float(b.norm())
    L.fallback_reset()
    t = torch.randn(2, 9, 16, device=DEV).transpose(1, 2)                  # neither: contiguous, as the stock operator's
    assert GN.GroupNormAct(4, 16).to(DEV)(t).is_contiguous() and L.fallback_counts()["gn_act"] == 1
    L.fallback_reset()
    half = GN.GroupNormAct(4, 16).to(DEV)(torch.randn(2, 16, 9, device=DEV, dtype=torch.bfloat16))         # fp32 parameters
    assert half.dtype == torch.bfloat16 and half.is_contiguous() and L.fallback_counts()["gn_act"] == 0


def test_gelu_of_every_fp16_value_is_the_neighbour_only_where_fp32_cannot_tell():
    """q = 1 - Phi(|z|) is off by (z^2 + 16) 2^-24 of itself, y = z q or z (1 - q): wherever the exact y is further from fp16's nearest tie than
    that (and 2 * 2^-24 for 1 - q and the product) the result is correctly rounded; these are all but one in 300 of the normal results"""
    import math
    from distill_bev_amd import act8 as A
    x = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x) & (x != 0)]
    z = x.double()
    q = 0.5 * torch.special.erfc(z.abs() / math.sqrt(2))
    y = torch.where(z > 0, z * (1 - q), z * q)
    ok = (y.abs() >= 2.0 ** -14) & (y.abs() < 65504)
    x, z, q, y = x[ok], z[ok], q[ok], y[ok]
    m = torch.frexp(y.abs())[0] * 2048
    tie = (m - torch.floor(m) - 0.5).abs() / m
    err = torch.where(z > 0, q / (1 - q), torch.ones_like(q)) * (z * z + 16) * 2.0 ** -24 + 2 * 2.0 ** -24
    sure = tie > err
    assert float(sure.double().mean()) > 1 - 1 / 300
    assert torch.equal(A.activation(x.to(DEV), "gelu").cpu()[sure], y.half()[sure])


def test_convolution_modules_give_the_layout_of_the_stock_ones():
    from distill_bev_amd import act8 as A
    from distill_bev_amd.colsum import BiasSumConv2d, use_bias_sum_convs
    for bias, cls in ((True, A.Act8Conv2d), (False, A.Act8Conv2d), (True, BiasSumConv2d)):
        for wfmt in (torch.contiguous_format, torch.channels_last):
            for xfmt in (torch.contiguous_format, torch.channels_last):
                torch.manual_seed(4)
                stock, mod = nn.Conv2d(16, 24, 1, bias=bias).to(DEV), nn.Conv2d(16, 24, 1, bias=bias).to(DEV)
                mod.load_state_dict(stock.state_dict())
                for m in (stock, mod):
                    m.weight.data = m.weight.data.contiguous(memory_format=wfmt)
                if cls is BiasSumConv2d:
                    assert use_bias_sum_convs(mod) == 1
                A.use_act8(mod)
                assert type(mod) is cls and mod.act8_format == "int8"
                x = torch.randn(2, 16, 5, 6, device=DEV).contiguous(memory_format=xfmt).requires_grad_(True)
                y, ref = mod(x), stock(x)
                assert torch.allclose(y, ref, atol=1e-5) and y.stride() == ref.stride(), (cls, wfmt, xfmt, y.stride(), ref.stride())
                a, b = torch.autograd.grad(y.sum(), (x,))[0], torch.autograd.grad(ref.sum(), (x,))[0]
                assert torch.allclose(a, b, atol=1e-5)
