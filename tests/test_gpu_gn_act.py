"""Group norm + activation on the GPU (csrc/gn_act.hip, distill_bev_amd/gn_act.py) against oracle/act8.py (64 bits).

Tolerances.  fp32: every output is a chain of K <= ~128 sequential fp32 roundings per thread (a chunk's rows, the row phases, a group's
channels) under fp64 merges; the shift by the chunk's first pixel multiplies the second moment's error by up to 1 + d^2, d ~ 4 spreads.
Independent roundings: sqrt(17 * 128) * 2^-24 * ~1.5 = 4e-6 of an output's size (norm over norm), ten times that for the worst element
against the larger of itself and the rms.  16-bit outputs: half a step (eps / 2) more."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from oracle import act8 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, ref, dtype, slack=1.0, skip=None):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    d = (got - ref).abs()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    rms = float(ref.norm()) / max(1, ref.numel()) ** 0.5
    lim = (4e-5 * slack + half) * torch.clamp(ref.abs(), min=rms) + 1e-30
    if skip is not None:
        d = torch.where(skip, torch.zeros_like(d), d)
    assert bool((d <= lim).all()), float((d / lim).max())
    if skip is None:
        assert float(d.norm()) <= (4e-6 * slack + half) * float(ref.norm()) + 1e-30


def _case(N, S, C, G, dtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, S, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g)) + offset * torch.randn(C, generator=g)
    return x.to(dtype), 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g), torch.randn(N, S, C, generator=g).to(dtype)


def _maps(t, H):
    N, S, C = t.shape
    return t.to(DEV).view(N, H, S // H, C).permute(0, 3, 1, 2)


def _rows(t):
    return t.detach().cpu().movedim(1, -1).reshape(t.shape[0], -1, t.shape[1])


SHAPES = [(1, 12, 1, 8, 4), (2, 1, 1, 64, 8), (3, 35, 5, 48, 16), (2, 600, 20, 80, 16), (1, 77, 7, 59, 1), (2, 90, 9, 130, 13), (1, 40, 4, 10, 5),
          (6, 176, 8, 256, 32), (2, 64, 8, 1030, 5), (1, 30, 3, 4096, 32), (40, 9, 3, 32, 32), (2, 2500, 50, 33, 3), (1, 9000, 90, 64, 32),
          (3, 21, 3, 512, 1), (2, 33, 3, 2058, 2)]


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,S,H,C,G", SHAPES)
def test_forward_and_backward(N, S, H, C, G, dtype, fmt):
    from distill_bev_amd import gn_act as GN
    for act in (("silu", "gelu") if fmt else ("none", "silu", "gelu")):
        x, w, b, gy = _case(N, S, C, G, dtype, S + C)
        leaves = [_maps(x, H).requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
        y = GN.group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, act, fmt)
        dx, dw, db = torch.autograd.grad(y, leaves, _maps(gy, H))
        ry, rdx, rdw, rdb, _ = O.group_norm(x.double(), G, w.double(), b.double(), 1e-5, act, fmt, gy.double())
        assert y.dtype == dtype and dx.dtype == dtype and y.movedim(1, -1).is_contiguous() and dw.dtype == torch.float32
        _close(_rows(y), ry, dtype)
        _close(_rows(dx), rdx, dtype, 2.0)
        scale = (gy.double().abs().sum((0, 1)) + 1).max()                 # parameter gradients are sums with cancellation
        assert float((dw.cpu().double() - rdw).abs().max() / scale) < 4e-6 and float((db.cpu().double() - rdb).abs().max() / scale) < 4e-6
        with torch.no_grad():
            assert torch.equal(GN.group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, act, fmt), y)


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_relu(dtype, fmt):
    """the gate is the sign of z: elements whose z lies within fp32 rounding of zero may go either way and are left out, one by one"""
    from distill_bev_amd import gn_act as GN
    N, S, C, G = 3, 140, 96, 8
    x, w, b, gy = _case(N, S, C, G, dtype, 5)
    leaves = [_maps(x, 10).requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    y = GN.group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, "relu", fmt)
    dx, dw, db = torch.autograd.grad(y, leaves, _maps(gy, 10))
    ry, rdx, rdw, rdb, z = O.group_norm(x.double(), G, w.double(), b.double(), 1e-5, "relu", fmt, gy.double())
    near = z.abs() < 2e-5
    assert float(near.double().mean()) < 1e-3
    _close(_rows(y), ry, dtype)
    if not bool(near.any()):
        near = None
    _close(_rows(dx), rdx, dtype, 2.0 if near is None else 50.0, near)
    if near is None:
        _close(dw, rdw, torch.float32, 4.0)
        _close(db, rdb, torch.float32, 4.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_against_differences(dtype):
    from distill_bev_amd import gn_act as GN
    N, S, C, G = 2, 50, 24, 3
    x, w, b, gy = _case(N, S, C, G, torch.float32, 7)
    x, gy = x.to(dtype), gy.to(dtype)
    leaves = [_maps(x, 5).requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    grads = torch.autograd.grad(GN.group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, "gelu"), leaves, _maps(gy, 5))
    loss = lambda x, w, b: float((O.group_norm(x, G, w, b, 1e-5, "gelu") * gy.double()).sum())        # noqa: E731
    base = [x.double(), w.double(), b.double()]
    for at, g in enumerate((_rows(grads[0]), grads[1].cpu(), grads[2].cpu())):
        d = torch.randn(base[at].shape, generator=torch.Generator().manual_seed(at)).double()
        up, down = list(base), list(base)
        up[at], down[at] = base[at] + 1e-5 * d, base[at] - 1e-5 * d
        num = (loss(*up) - loss(*down)) / 2e-5
        tol = (torch.finfo(dtype).eps / 2 if at == 0 else 2e-6) + 4e-6
        assert abs(num - float((g.double() * d).sum())) <= tol * float((g.double() * d).abs().sum()) + 1e-6


def test_large_offsets_keep_their_digits():
    """mean / spread = 1000: the input itself holds 2^-24 * 1000 = 6e-5 of a spread, nothing else may be lost"""
    from distill_bev_amd import gn_act as GN
    N, S, C, G = 2, 3000, 64, 8
    x, w, b, gy = _case(N, S, C, G, torch.float32, 8, offset=0.0)
    x = x + 1000.0
    y = GN.group_norm_act(_maps(x, 30), G, w.to(DEV), b.to(DEV))
    ref = O.group_norm(x.double(), G, w.double(), b.double(), 1e-5, "none")
    assert float((_rows(y).double() - ref).abs().max()) < 6e-5 * float(w.abs().max()) * 2.5


def test_parameters_absent_or_in_sixteen_bits_and_other_layouts():
    from distill_bev_amd import gn_act as GN
    x, w, b, gy = _case(3, 60, 32, 4, torch.float32, 9)
    ref = O.group_norm(x.double(), 4, None, None, 1e-3, "silu")
    _close(_rows(GN.group_norm_act(_maps(x, 6), 4, eps=1e-3, act="silu")), ref, torch.float32)
    nchw = _maps(x, 6).contiguous().requires_grad_(True)                   # another layout is copied, the gradient arrives
    y = GN.group_norm_act(nchw, 4, w.to(DEV).bfloat16().requires_grad_(True), None, act="gelu", checkpoint="int8")
    y.backward(_maps(gy, 6).contiguous())
    wb = w.bfloat16().double()
    ry, rdx, _, _, _ = O.group_norm(x.double(), 4, wb, None, 1e-5, "gelu", "int8", gy.double())
    _close(_rows(y), ry, torch.float32)
    _close(_rows(nchw.grad), rdx, torch.float32, 2.0)
    wl = w.to(DEV).bfloat16().requires_grad_(True)
    y = GN.group_norm_act(_maps(x, 6), 4, wl, None)
    y.backward(_maps(gy, 6))                                               # only the weight wants a gradient
    assert wl.grad.dtype == torch.bfloat16
    _, _, rdw, _, _ = O.group_norm(x.double(), 4, wb, None, 1e-5, "none", None, gy.double())
    _close(wl.grad, rdw, torch.bfloat16, 4.0)
    for shape in ((5, 32), (2, 32, 7), (2, 32, 3, 2, 4)):                  # other ranks
        t = torch.randn(shape, generator=torch.Generator().manual_seed(3))
        out = GN.group_norm_act(t.to(DEV), 4, w.to(DEV), b.to(DEV), act="relu")
        rows = t.movedim(1, -1).reshape(shape[0], -1, 32)
        r = O.group_norm(rows.double(), 4, w.double(), b.double(), 1e-5, "relu")
        assert out.shape == shape
        _close(out.movedim(1, -1).reshape(rows.shape), r, torch.float32)
    e = torch.empty((0, 32, 4, 4), device=DEV, requires_grad=True)
    wl = w.to(DEV).requires_grad_(True)
    GN.group_norm_act(e, 4, wl, None, checkpoint="int8").sum().backward()
    assert e.grad.shape == e.shape and torch.equal(wl.grad, torch.zeros_like(wl))


def test_non_finite_values_stay_in_their_group():
    from distill_bev_amd import gn_act as GN
    x, w, b, gy = _case(2, 50, 64, 8, torch.float32, 10)
    x[0, 3, 5], x[1, 7, 60] = float("inf"), float("nan")
    leaf = _maps(x, 5).requires_grad_(True)
    for fmt in (None, "int8"):
        y = GN.group_norm_act(leaf, 8, w.to(DEV), b.to(DEV), 1e-5, "none", fmt)
        dx, = torch.autograd.grad(y, (leaf,), _maps(gy, 5))
        yr = _rows(y)
        assert bool(torch.isnan(yr[0, :, :8]).all()) and bool(torch.isfinite(yr[0, :, 8:]).all())
        assert bool(torch.isnan(yr[1, :, 56:]).all()) and bool(torch.isfinite(yr[1, :, :56]).all())
        assert bool(torch.isnan(_rows(dx)[0, :, :8]).all())
        if fmt is None:
            assert bool(torch.isfinite(_rows(dx)[0, :, 8:]).all())


def test_refusals():
    from distill_bev_amd import _lib as L
    from distill_bev_amd import gn_act as GN
    x = torch.randn(2, 12, 3, 3, device=DEV)
    for G in (0, 5, -3, 24):
        with pytest.raises(ValueError):
            GN.group_norm_act(x, G)
    with pytest.raises(ValueError):
        GN.group_norm_act(x, 4, torch.ones(11, device=DEV))
    with pytest.raises(ValueError):
        GN.group_norm_act(x, 4, act="tanh")
    with pytest.raises(ValueError):
        GN.group_norm_act(x, 4, checkpoint="int4")
    with pytest.raises(ValueError):
        GN.group_norm_act(x, 4, eps=float("nan"))
    with pytest.raises(ValueError):
        GN.group_norm_act(torch.randn(1, 4, device=DEV), 4)               # one value per group: F.group_norm's own refusal
    with pytest.raises(L.DbevHipError):
        GN.group_norm_act(x.double(), 4)
    with pytest.raises(L.DbevHipError):
        GN.group_norm_act(x, 4, torch.ones(12))                            # weight on the host
    x = x.contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = GN.group_norm_act(x, 4)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError):                                      # x was kept: autograd sees the change
        y.sum().backward()


def test_same_bits_every_time_on_other_streams_and_in_replays():
    from distill_bev_amd import gn_act as GN
    data = [_case(4, 180, 96, 8, torch.float32, 20 + i) for i in range(4)]
    w, b = data[0][1].to(DEV), data[0][2].to(DEV)
    xs, gs = [_maps(d[0], 12) for d in data], [_maps(d[3], 12) for d in data]

    def step(x, g):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = GN.group_norm_act(leaves[0], 8, leaves[1], leaves[2], act="silu", checkpoint="int8")
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    eager = [step(x, g) for x, g in zip(xs, gs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for i, s in enumerate(streams):                                        # two calls at once
        with torch.cuda.stream(s):
            outs.append(step(xs[i], gs[i]))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i in range(2):
        assert all(torch.equal(a, c) for a, c in zip(outs[i], eager[i]))
    sx, sg = xs[0].clone(), gs[0].clone()
    streams[0].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[0]):
        step(sx, sg)
    torch.cuda.current_stream().wait_stream(streams[0])
    graphs, held = [], []
    for _ in range(2):                                                     # two graphs over the same static inputs
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(step(sx, sg))
        graphs.append(g)
    for i in (1, 3, 0, 2):
        sx.copy_(xs[i])
        sg.copy_(gs[i])
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held[i % 2], eager[i]))
        assert all(torch.equal(a, c) for a, c in zip(step(xs[3 - i], gs[3 - i]), eager[3 - i]))


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
def test_a_stack_as_a_model_uses_it(fmt):
    """1x1 conv -> GN -> SiLU -> 1x1 conv -> GN, rewired by fuse_gn_act_modules and use_act8: forward equals the stock modules', gradients the
    oracle's with the same checkpoints"""
    from distill_bev_amd import act8 as A
    from distill_bev_amd import gn_act as GN
    torch.manual_seed(6)
    build = lambda: nn.Sequential(nn.Conv2d(32, 64, 1), nn.GroupNorm(8, 64), nn.SiLU(), nn.Conv2d(64, 48, 1, bias=True), nn.GroupNorm(4, 48))   # noqa: E731
    stock = build()
    for m in stock:
        if isinstance(m, nn.GroupNorm):
            nn.init.normal_(m.weight, 1, 0.2), nn.init.normal_(m.bias, 0, 0.2)
    mod = build()
    mod.load_state_dict(stock.state_dict())
    stock, mod = stock.to(DEV), mod.to(DEV).to(memory_format=torch.channels_last)
    assert GN.fuse_gn_act_modules(mod, fmt) == 2
    if fmt:
        assert A.use_act8(mod, fmt) == 2
    x, gy = torch.randn(2, 32, 10, 9), torch.randn(2, 48, 10, 9)
    xa = x.to(DEV).to(memory_format=torch.channels_last).requires_grad_(True)
    y = mod(xa)
    assert torch.allclose(y, stock(x.to(DEV)), atol=5e-5)
    y.backward(gy.to(DEV))
    p = [t.detach().cpu().double().requires_grad_(True) for t in stock.parameters()]
    xd = x.double().permute(0, 2, 3, 1).reshape(-1, 32).requires_grad_(True)
    h = O.LinearFn.apply(xd, p[0].view(64, 32), p[1], fmt)
    h = O.GroupNormFn.apply(h.view(2, 90, 64), 8, p[2], p[3], 1e-5, "silu", fmt)
    h = O.LinearFn.apply(h.reshape(-1, 64), p[4].view(48, 64), p[5], fmt)
    out = O.GroupNormFn.apply(h.view(2, 90, 48), 4, p[6], p[7], 1e-5, "none", fmt)
    out.backward(gy.double().permute(0, 2, 3, 1).reshape(2, 90, 48))
    # codes next to a border may differ by one step after fp32 layers: sqrt(2 e step) of a gradient's norm (test_gpu_act8's feed-forward
    # test), step 1 / 32 (int8) or 1 / 8 (e4m3) of the spread, e <= 1e-6; without checkpoints fp32 rounding alone
    tol = {None: 1e-5, "int8": 2.5e-4, "e4m3": 5e-4}[fmt]
    rel = lambda a, r: float((a.detach().cpu().double().reshape(r.shape) - r).norm() / r.norm())      # noqa: E731
    assert rel(xa.grad.permute(0, 2, 3, 1), xd.grad.view(2, 10, 9, 32)) < tol
    for q, r in zip(mod.parameters(), p):
        if r is p[1] or r is p[5]:
            continue                          # a bias in front of a group norm: its gradient is what the norm leaves of a per-channel shift
        assert rel(q.grad, r.grad) < tol


def test_conv_module_with_group_norm_and_the_ledger():
    from distill_bev_amd import _lib as L
    from distill_bev_amd import gn_act as GN
    from distill_bev_amd.registry import ConvModule
    import warnings
    torch.manual_seed(7)
    m = ConvModule(8, 16, 3, padding=1, norm_cfg=dict(type="GN", num_groups=4)).to(DEV).to(memory_format=torch.channels_last)
    x = torch.randn(2, 8, 12, 10, device=DEV).to(memory_format=torch.channels_last)
    ref = F.relu(F.group_norm(m.conv(x), 4, m.norm.weight, m.norm.bias, m.norm.eps))
    assert GN.fuse_gn_act_modules(m) == 1
    L.fallback_reset()
    assert torch.allclose(m(x), ref, atol=1e-5) and L.fallback_counts()["gn_act"] == 0
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        GN.gn_act(x.double().repeat(1, 2, 1, 1), nn.GroupNorm(4, 16).to(DEV).double())
    assert L.fallback_counts()["gn_act"] == 1
    L.fallback_reset()


def test_more_than_two_to_the_31_values_and_misaligned_addresses():
    from distill_bev_amd import gn_act as GN
    S, C, G = (1 << 25) + 77, 64, 4                                         # one image, 2^31 values and some, in 16 bits
    x = torch.empty((1, S, C), dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for a in range(0, S, 1 << 22):
        x[:, a:a + (1 << 22)] = torch.randn((1, min(1 << 22, S - a), C), generator=g, device=DEV)
    w = torch.rand(C, device=DEV) + 0.5
    y = GN.group_norm_act(x.permute(0, 2, 1), G, w, None, 1e-5, "silu").permute(0, 2, 1)
    t = x.view(S, G, C // G)
    mean, sq = torch.zeros(G, dtype=torch.float64, device=DEV), torch.zeros(G, dtype=torch.float64, device=DEV)
    for a in range(0, S, 1 << 22):
        d = t[a:a + (1 << 22)].double()
        mean += d.sum((0, 2))
        sq += d.square().sum((0, 2))
    n = S * (C // G)
    mean, rstd = mean / n, 1 / torch.sqrt(sq / n - (mean / n) ** 2 + 1e-5)
    for sl in (slice(0, 1000), slice(S // 2, S // 2 + 1000), slice(S - 1000, S)):
        z = ((t[sl].double() - mean[:, None]) * rstd[:, None]).reshape(-1, C) * w.double()
        _close(y[0, sl], O.act(z, "silu")[0].cpu(), torch.bfloat16)
    del x, y, t
    for off in (1, 2, 3):                                                    # the same values at other addresses: the same bits
        x, w, b, gy = _case(2, 60, 64, 8, torch.float32, 77)
        flat, gflat = torch.zeros(2 * 60 * 64 + 4, device=DEV), torch.zeros(2 * 60 * 64 + 4, device=DEV)
        flat[off:off + x.numel()], gflat[off:off + x.numel()] = x.view(-1).to(DEV), gy.view(-1).to(DEV)
        at = lambda f: f[off:off + x.numel()].view(2, 6, 10, 64).permute(0, 3, 1, 2)      # noqa: E731
        leaf = at(flat).requires_grad_(True)
        y = GN.group_norm_act(leaf, 8, w.to(DEV), b.to(DEV), 1e-5, "gelu", "int8")
        dx, = torch.autograd.grad(y, (leaf,), at(gflat))
        ry, rdx, _, _, _ = O.group_norm(x.double(), 8, w.double(), b.double(), 1e-5, "gelu", "int8", gy.double())
        _close(_rows(y), ry, torch.float32)
        _close(_rows(dx), rdx, torch.float32, 2.0)
    e = torch.empty((2, 32, 0, 5), device=DEV, requires_grad=True)           # images without pixels
    wl = torch.ones(32, device=DEV, requires_grad=True)
    GN.group_norm_act(e, 4, wl, None).sum().backward()
    assert e.grad.shape == e.shape and torch.equal(wl.grad, torch.zeros_like(wl))


# ---- batches that go through the one-pass kernels (csrc/gn_one.hip): 2048 register tiles or more, an image of 2 to 512 of them ----------
ONE = [(260, 4200, 42, 64, 8), (24, 11440, 104, 256, 32), (66, 11000, 100, 80, 16), (31, 2111, 1, 1024, 512), (17, 20999, 1, 192, 3)]


def _run(x, w, b, gy, G, act, fmt):
    from distill_bev_amd import gn_act as GN
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = GN.group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, act, fmt)
    return (y.detach(), *torch.autograd.grad(y, leaves, gy))


def _big(N, S, H, C, G, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)                 # noqa: E731
    x = (r(N, S, C) * torch.exp(0.5 * r(C)) + r(C)).to(dtype)
    m = lambda t: t.view(N, H, S // H, C).permute(0, 3, 1, 2)              # noqa: E731
    return m(x), 1 + 0.3 * r(C), 0.3 * r(C), m(r(N, S, C).to(dtype))


@pytest.mark.parametrize("dtype,fmt,act", [(torch.float32, None, "silu"), (torch.float32, "int8", "gelu"), (torch.float32, "e4m3", "none"),
                                           (torch.bfloat16, None, "gelu"), (torch.bfloat16, "int8", "silu"), (torch.float16, "e4m3", "gelu")])
@pytest.mark.parametrize("N,S,H,C,G", ONE)
def test_large_batches(N, S, H, C, G, dtype, fmt, act):
    """against the oracle evaluated in 64 bits on the device; chains of sums are longer than in the small cases by the channels of a group and
    the tiles, both under sqrt: the same 4e-6, five times it for the worst of 10^7 elements"""
    x, w, b, gy = _big(N, S, H, C, G, dtype, S)
    y, dx, dw, db = _run(x, w, b, gy, G, act, fmt)
    rows = lambda t: t.movedim(1, -1).reshape(N, S, C).double()            # noqa: E731
    ry, rdx, rdw, rdb, _ = O.group_norm(rows(x), G, w.double(), b.double(), 1e-5, act, fmt, rows(gy))
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    for got, ref in ((rows(y), ry), (rows(dx), rdx)):
        d = (got - ref).abs()
        rms = ref.square().mean().sqrt()
        assert float(d.norm() / ref.norm()) < 8e-6 + half
        assert bool((d <= (2e-4 + half) * torch.maximum(ref.abs(), rms)).all())
    scale = float(rows(gy).abs().sum((0, 1)).max())
    assert float((dw.double() - rdw).abs().max()) < 4e-6 * scale and float((db.double() - rdb).abs().max()) < 4e-6 * scale


@pytest.mark.parametrize("dtype,fmt", [(torch.float32, None), (torch.float32, "int8"), (torch.bfloat16, "e4m3")])
def test_tiles_that_give_up_waiting_are_finished_with_the_same_bits(dtype, fmt):
    """a wait of no looks at all: whatever is not there at once goes the long way"""
    from distill_bev_amd import _lib as L
    x, w, b, gy = _big(24, 11440, 104, 256, 32, dtype, 1)
    ref = _run(x, w, b, gy, 32, "silu", fmt)
    old = L.call("dbev_gn_act_poll_limit", 0)
    try:
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(_run(x, w, b, gy, 32, "silu", fmt), ref))
        L.call("dbev_gn_act_poll_limit", 3)
        assert all(torch.equal(p, q) for p, q in zip(_run(x, w, b, gy, 32, "silu", fmt), ref))
    finally:
        assert L.call("dbev_gn_act_poll_limit", old) == 3
    assert L.call("dbev_gn_act_poll_limit", -1) == old
    assert all(torch.equal(p, q) for p, q in zip(_run(x, w, b, gy, 32, "silu", fmt), ref))


def test_large_batches_side_by_side_and_captured():
    """several at once on streams of their own, beside other work, and replayed from a graph: the bits of the call alone"""
    data = [_big(24, 11440, 104, 256, 32, torch.float32, 30 + i) for i in range(3)]
    alone = [_run(*d, 32, "silu", "int8") for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(2):
        outs = []
        for s, d in zip(streams, data):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(_run(*d, 32, "silu", "int8"))
        busy = torch.randn(4096, 4096, device=DEV)
        busy @ busy
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for a, o in zip(alone, outs):
            assert all(torch.equal(p, q) for p, q in zip(a, o))
    sx, w, b, sg = [t.clone(memory_format=torch.preserve_format) for t in data[0]]
    streams[0].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[0]):
        _run(sx, w, b, sg, 32, "silu", "int8")
    torch.cuda.current_stream().wait_stream(streams[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _run(sx, w, b, sg, 32, "silu", "int8")
    for i in (1, 2, 0, 1):
        for t, src in zip((sx, w, b, sg), data[i]):
            t.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, alone[i]))
        assert all(torch.equal(p, q) for p, q in zip(_run(*data[2 - i], 32, "silu", "int8"), alone[2 - i]))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_trainer_with_activation_checkpoints(fmt):
    """the Trainer's option on a small detector: the first loss is the plain Trainer's, the gradients differ by the checkpoints' rounding only
    -- relative error of a kept value at most 2^-6 (int8, of its block's largest) or 2^-4 (e4m3), independent signs: a few times 1e-2 at most
    -- and parameters move"""
    from test_host_act8 import _Toy
    from distill_bev_amd.train_step import Trainer
    x = torch.randn(4, 16, 20, 30, generator=torch.Generator().manual_seed(1)).to(DEV)

    def one(option):
        torch.manual_seed(11)
        tr = Trainer(_Toy(), dict(), DEV, channels_last=True, activation_checkpoint=option)
        loss = tr.step(dict(x=x))[0]
        return tr, float(loss), [p.grad.detach().clone() for p in tr.detector.parameters()]

    _, la, ga = one(None)
    tr, lb, gb = one(fmt)
    assert abs(la - lb) < 1e-5 * abs(la)
    for (name, _), a, b in zip(tr.detector.named_parameters(), ga, gb):
        if name != "neck.0.bias":                  # in front of a norm: what is left of a cancellation
            assert float((a - b).norm() / a.norm()) < 0.05, name
    before = [p.detach().clone() for p in tr.detector.parameters()]
    tr.step(dict(x=x))
    assert all(not torch.equal(p, q) for p, q in zip(before, tr.detector.parameters()))
    tr.close()


def test_a_chunk_that_begins_with_an_outlier():
    """The squares are taken about a chunk's first pixel; an outlier D there makes every term D^2.  n = 250 rows a chunk, chains of at most 40
    additions: the second moment is off by at most 40 * 250 * 2^-24 D^2, and the outlier itself gives it D^2: 6e-4 of the variance, 3e-4 of y - b.
    The chunk's mean is K + (sum of x - K) / n, sums of terms of size D: off by at most 40 * 2^-24 D in one of eight chunks, i.e. by 5 * 2^-24 D
    in all, where a spread is at least D / sqrt(2000): 5 * 2^-24 * 44.7 = 1.34e-5 <= 2^-16 spreads, times |w| in y"""
    from distill_bev_amd import gn_act as GN
    x, w, b, _ = _case(1, 2000, 8, 2, torch.float32, 9)
    x[0, 0] = 1e4
    y = GN.group_norm_act(_maps(x, 40), 2, w.to(DEV), b.to(DEV), 1e-5)
    ref = F.group_norm(x.double().movedim(1, 2), 2, w.double(), b.double(), 1e-5).movedim(1, 2)
    d = (_rows(y) - ref).abs()
    assert bool((d <= 2.0 ** -11 * (ref - b.double()).abs() + 2.0 ** -16 * w.double().abs() + 2.0 ** -22 * (1 + ref.abs())).all()), float(d.max())


def test_sizes_beyond_the_limits_are_refused():
    from distill_bev_amd import _lib as L
    from distill_bev_amd import gn_act as GN
    with pytest.raises(L.DbevHipError):
        GN.group_norm_act(torch.empty((1, 1 << 17), device=DEV), 4)
    with pytest.raises(L.DbevHipError):
        GN.group_norm_act(torch.empty((1, 8), device=DEV).expand((1 << 22) + 1, 8), 4)


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_large_image_in_many_chunks(dtype, fmt):
    """a batch too small to fill the chip with 128 chunks an image: 400 of them"""
    test_forward_and_backward(1, 40000, 200, 96, 12, dtype, fmt)


@pytest.mark.parametrize("dtype,H", [(torch.float32, 640), (torch.bfloat16, 900)])
def test_one_image_beyond_the_caches(dtype, H):
    """more than 192 MB in two launches a direction (no cached accesses, last chunks first), against 64 bits on the device; norm over norm as above"""
    from distill_bev_amd import gn_act as GN
    g = torch.Generator(DEV).manual_seed(11)
    x = torch.randn((1, H, H, 128), device=DEV, generator=g).to(dtype).permute(0, 3, 1, 2)
    gy = torch.randn((1, H, H, 128), device=DEV, generator=g).to(dtype).permute(0, 3, 1, 2)
    w, b = 1 + 0.3 * torch.randn(128, device=DEV, generator=g), 0.3 * torch.randn(128, device=DEV, generator=g)
    leaves = [x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    assert x.numel() * x.element_size() > 192 << 20
    y = GN.group_norm_act(leaves[0], 16, leaves[1], leaves[2], 1e-5, "silu")
    dx, dw, db = torch.autograd.grad(y, leaves, gy)
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    ref = [t.detach().double().contiguous().requires_grad_(True) for t in leaves]
    ry = F.silu(F.group_norm(ref[0], 16, ref[1], ref[2], 1e-5))
    rdx, rdw, rdb = torch.autograd.grad(ry, ref, gy.double())
    for got, want, slack in ((y, ry.detach(), 1.0), (dx, rdx, 2.0)):
        assert float((got.detach().double() - want).norm()) <= (4e-6 * slack + half) * float(want.norm())
    scale = float(gy.double().abs().sum((0, 2, 3)).max())
    assert float((dw.double() - rdw).abs().max()) < 4e-6 * scale and float((db.double() - rdb).abs().max()) < 4e-6 * scale


@pytest.mark.parametrize("fmt", [None, "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,S,H,C,G", [(3, 300, 20, 200, 25), (5, 2, 1, 200, 25), (2, 512, 16, 72, 9), (2, 513, 27, 72, 9), (2, 1024, 32, 40, 5), (1, 1025, 41, 40, 5),
                                       (70, 3, 1, 1040, 65), (2, 16, 4, 2048, 1), (2, 17, 1, 2056, 257)])
def test_small_images(N, S, H, C, G, dtype, fmt):
    """one workgroup an image and range of channels: last ranges of a few channels, pixel counts at the limit of a workgroup and one beyond it"""
    test_forward_and_backward(N, S, H, C, G, dtype, fmt)
