"""GroupNorm fused with the activation behind it, channels-last, optionally trained from an 8-bit checkpoint (csrc/gn_act.hip).

Host-side mirror of ``norm_cfg=dict(type='GN', num_groups=G)`` layers: nn.GroupNorm -> activation of the ConvModules (mmcv order
conv -> norm -> act; mmdet3d/models/necks/fpn.py:77-95, lss_fpn.py:30-60).  Unlike the BatchNorm kernels (bn_act.py) these take float32,
bfloat16 and float16, any channel count, ReLU, SiLU and GELU, and any [N, C, *] shape: one or two launches over the data a direction, nothing but
the output written and -- under autograd -- x or its checkpoint kept (act8.py: 1.03 bytes a value, written by the forward's own pass).

    group_norm_act(x, num_groups, weight, bias, eps, act="silu", checkpoint="int8")     # F.group_norm + activation
    gn_act(x, gn, act, checkpoint)                                                       # the same with a module's parameters
    GroupNormAct                                                                         # nn.GroupNorm + activation, same state-dict keys
    norm_act(x, norm, act)                                                               # act(norm(x)) of any norm module, in one operator where it can be
    fuse_gn_act_modules(model, checkpoint=None)                                          # rewires a built model

`group_norm_act` raises on what the kernels cannot take (a tensor in another layout is copied to channels-last first); the modules leave
CPU and float64 tensors, other layouts that keep no checkpoint, autocast, sizes beyond the kernels' and calls under torch.jit.trace, forward-mode
differentiation or a torch.func transform to the stock operators (device tensors are counted in the fallback ledger)."""
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import act8 as A

_STOCK = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}


def _maps(x):
    """x [N, C, *] as a tensor whose memory is dense [N, *, C] (x itself if it is), and its pixels per image"""
    N, C = x.shape[0], x.shape[1]
    n = x.numel()
    S = n // (N * C) if n else 0
    if x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last):
        return x, N, C, S
    t = x.movedim(1, -1)
    return (x if t.is_contiguous() else t.contiguous().movedim(-1, 1)), N, C, S


def _f32(t):
    return t if t is None or (t.dtype == torch.float32 and t.is_contiguous()) else t.detach().float().contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, N, C, S, G, weight, bias, eps, act, fmt, stats):
    """x dense channels-last -> y, f32 [2, N, G] of mean and rstd (None without `stats`), the checkpoint's buffer (None without `fmt`)"""
    dev = x.device
    y = torch.empty_like(x)                                   # dense: x's own strides
    st = torch.empty((2, N, G), dtype=torch.float32, device=dev) if stats else None
    buf = A._buffer(N * S, C, dev) if fmt else None
    n = N * S * C
    if n:
        nbytes = int(L.call("dbev_gn_act_workspace_bytes", N, S, C, G))
        if nbytes == 0:
            raise L.DbevHipError(f"group_norm_act: unsupported size {tuple(x.shape)}, {G} groups")
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        mean = _ptr(st)
        codes = _ptr(buf)
        L.call("dbev_gn_act_forward", x.data_ptr(), A.DTYPES[x.dtype], N, S, C, G, _ptr(weight), _ptr(bias), eps, A.ACTS[act], y.data_ptr(),
               mean, mean + 4 * N * G if stats else None, A.FORMATS[fmt] if fmt else 0, codes, codes + n if fmt else None, ws.data_ptr(), nbytes,
               L.raw_stream(dev), alg_bytes=2 * n * x.element_size() + (n if fmt else 0))
    return y, st, buf


def _gradients(ctx, gy):
    kept, weight, bias, st = ctx.saved_tensors
    G, eps, act, fmt = ctx.cfg
    dev = gy.device
    _, need_w, need_b = ctx.needs_input_grad[:3]
    with L.on(dev):
        w, b = _f32(weight), _f32(bias)
        dx = A.empty_dense(gy.shape, 1, gy.dtype, dev)
        gy, N, C, S = _maps(gy)
        n = N * S * C
        new = torch.empty if n else torch.zeros
        dwb = new((2, C), dtype=torch.float32, device=dev) if need_w or need_b else None
        if n:
            nbytes = int(L.call("dbev_gn_act_workspace_bytes", N, S, C, G))
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
            mean, k, dw = st.data_ptr(), kept.data_ptr(), _ptr(dwb)
            L.call("dbev_gn_act_backward", gy.data_ptr(), A.DTYPES[gy.dtype], None if fmt else k, A.FORMATS[fmt] if fmt else 0,
                   k if fmt else None, k + n if fmt else None, N, S, C, G, _ptr(w), _ptr(b), mean, mean + 4 * N * G, A.ACTS[act],
                   dx.data_ptr(), dw if need_w else None, dw + 4 * C if need_b else None, ws.data_ptr(), nbytes, L.raw_stream(dev),
                   alg_bytes=2 * n * gy.element_size() + (n if fmt else n * gy.element_size()))
        dw = db = None
        if need_w:
            dw = dwb[0] if weight.dtype == torch.float32 else dwb[0].to(weight.dtype)
        if need_b:
            db = dwb[1] if bias.dtype == torch.float32 else dwb[1].to(bias.dtype)
    return dx if ctx.needs_input_grad[0] else None, dw, db, None, None, None, None


class _GroupNormAct(Function):
    """x dense channels-last"""

    @staticmethod
    def forward(ctx, x, weight, bias, G, eps, act, fmt):
        with L.on(x.device):
            xd, N, C, S = _maps(x)
            y, st, buf = _forward(xd, N, C, S, G, _f32(weight), _f32(bias), eps, act, fmt, True)
        ctx.save_for_backward(buf if fmt else x, weight, bias, st)
        ctx.cfg = (G, eps, act, fmt)
        return y

    @staticmethod
    def backward(ctx, gy):
        if not torch.is_grad_enabled():
            return _gradients(ctx, gy)
        # gradients that will be differentiated again: those of the stock operators (nn.GroupNorm has second derivatives too)
        x, weight, bias, _ = ctx.saved_tensors
        G, eps, act, _ = ctx.cfg
        f32 = lambda t: None if t is None else t.float()                  # noqa: E731
        y = _STOCK[act](F.group_norm(x.float(), G, f32(weight), f32(bias), eps)).to(x.dtype)
        need = ctx.needs_input_grad[:3]
        grads = iter(torch.autograd.grad(y, [t for t, n in zip((x, weight, bias), need) if n], gy, create_graph=True))
        return (*(next(grads) if n else None for n in need), None, None, None, None)


class _GroupNormAct8(_GroupNormAct):
    """the same from a checkpoint: no second derivatives"""

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        return _gradients(ctx, gy)


def _fits(N, C, S):
    """the kernels' limits (dbev_gn_act_workspace_bytes has the same)"""
    return C <= 1 << 16 and N <= 1 << 22 and S <= 1 << 30 and S * C <= 1 << 36


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", checkpoint=None):
    """act(F.group_norm(x, num_groups, weight, bias, eps)) for a device tensor x [N, C, *], act one of act8.ACTS; the result is
    channels-last.  `checkpoint` ("int8" / "e4m3"): under autograd the 8-bit checkpoint of x is kept instead of x, and the gradients are
    those of the formula with x^ in place of x (mean and rstd stay x's own)."""
    special = A.transformed()
    if special:
        A.no_trace("group_norm_act")
    A._act(act)
    if checkpoint is not None:
        A._fmt(checkpoint)
    dev = L.require_cuda(x, weight, bias)
    A._dtype(x)
    G = int(num_groups)
    if x.dim() < 2:
        raise ValueError(f"group_norm_act: [N, C, *] expected, got {tuple(x.shape)}")
    N, C = x.shape[:2]
    if G < 1 or C == 0 or C % G:
        raise ValueError(f"group_norm_act: {C} channels in {num_groups} groups")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (C,) or t.dtype not in A.DTYPES):
            raise ValueError(f"group_norm_act: {name} {tuple(t.shape)} {t.dtype} for {C} channels")
    S = x.numel() // (N * C) if N else 0
    if not _fits(N, C, S):
        raise L.DbevHipError(f"group_norm_act: {N} images of {C} channels, {tuple(x.shape)}; at most 2^22 and 2^16, of 2^30 pixels and 2^36 values")
    if not eps >= 0:
        raise ValueError(f"group_norm_act: eps {eps}")
    if N * S * C == G:                                            # F.group_norm's own refusal
        raise ValueError(f"Expected more than 1 value per channel when training, got input size {tuple(x.shape)}")
    if special or torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                               or (bias is not None and bias.requires_grad)):
        x = _maps(x)[0]                                               # (a copy of another layout is a step of the graph by itself)
        return (_GroupNormAct8 if checkpoint else _GroupNormAct).apply(x, weight, bias, G, float(eps), act, checkpoint)     # (raises if special)
    with L.on(dev):
        xd, N, C, S = _maps(x.detach())
        return _forward(xd, N, C, S, G, _f32(weight), _f32(bias), float(eps), act, None, False)[0]


def _ready(x, gn):
    if not (torch.is_tensor(x) and x.is_cuda and x.numel() and x.dim() >= 2):
        return False
    why = None
    if x.dtype not in A.DTYPES or (gn.weight is not None and gn.weight.dtype not in A.DTYPES):
        why = f"dtype {x.dtype}"
    elif torch.is_autocast_enabled("cuda"):
        why = "autocast"
    elif A.transformed():
        why = "traced or transformed"
    elif not _fits(x.shape[0], x.shape[1], x.numel() // (x.shape[0] * x.shape[1])):
        why = f"size {tuple(x.shape)}"
    if why:
        L.note_fallback("gn_act", why)
    return why is None


def _channels_last(x):
    if x.dim() == 2 or x.numel() == x.shape[0] * x.shape[1]:                # one pixel
        return x.is_contiguous()
    return (x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last)
            or x.dim() == 5 and x.is_contiguous(memory_format=torch.channels_last_3d))


def gn_act(x, gn, act="none", checkpoint=None):
    """act(gn(x)) with the module `gn`'s parameters: the kernels for device tensors they take, the stock operators otherwise.  A channels-last map
    (or [N, C]) stays one.  A tensor of another layout gives a contiguous one, as torch's operator does, and goes to the kernels -- by copies
    in and out -- only to keep a checkpoint or where the parameters are of another type than x, which torch's does not take"""
    A._act(act)
    if checkpoint is not None:
        A._fmt(checkpoint)
    if _ready(x, gn):
        args = (gn.num_groups, gn.weight, gn.bias, gn.eps, act, checkpoint)
        if _channels_last(x):
            return group_norm_act(x, *args)
        if checkpoint is not None and A._recording(x, gn.weight, gn.bias) or gn.weight is not None and gn.weight.dtype != x.dtype:
            return group_norm_act(x, *args).contiguous()
        L.note_fallback("gn_act", f"layout {tuple(x.shape)} {x.stride()}")
    return _STOCK[act](F.group_norm(x, gn.num_groups, gn.weight, gn.bias, gn.eps))


def norm_act(x, norm, act="none"):
    """act(norm(x)) for any norm module; `act`: a name or an activation module.  One operator where the norm is a GroupNormAct without an activation
    of its own and the activation is one of act8.ACTS -- for blocks that hold the two as separate attributes (nets.BasicBlock, Bottleneck)"""
    name = act if isinstance(act, str) else act.act if type(act) is A.Act8Activation and not A.hooked(act) else A.act_name(act)
    if type(norm) is GroupNormAct and norm.act == "none" and name and not A.hooked(norm):
        return gn_act(x, norm, name, norm.act8_format)
    y = norm(x)
    return _STOCK[act](y) if isinstance(act, str) else act(y)


class GroupNormAct(nn.GroupNorm):
    """nn.GroupNorm that also applies the activation behind it (`act`, one of act8.ACTS) and may keep its input as an 8-bit checkpoint
    (`act8_format`: None, "int8" or "e4m3"); parameters and state-dict keys are nn.GroupNorm's"""
    act, act8_format = "none", None

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, act="none", checkpoint=None, **kwargs):
        super().__init__(num_groups, num_channels, eps, affine, **kwargs)
        A._act(act)
        if checkpoint is not None:
            A._fmt(checkpoint)
        self.act, self.act8_format = act, checkpoint

    def forward(self, x):
        return gn_act(x, self, self.act, self.act8_format)

    def extra_repr(self):
        return super().extra_repr() + f", act={self.act}, act8={self.act8_format}"


def fuse_gn_act_modules(model, checkpoint=None):
    """Rewire the nn.GroupNorm modules of nn.Sequential stacks and ConvModules onto the kernels, together with the ReLU / SiLU / GELU right
    behind them (replaced by nn.Identity; keys unchanged); other GroupNorm modules become GroupNormAct without an activation (the residual
    blocks of nets.py put theirs in by `norm_act`).
    A norm that several places share, or that carries hooks, keeps the activation behind it as a module; so does an activation with hooks, and a
    stack whose forward is not its class's.  `checkpoint`: the format in which all norms of the model keep their input; None leaves that to
    each norm (a GroupNormAct's own `act8_format`; plain norms keep x).  Returns how many norms changed.  Idempotent."""
    from .registry import ConvModule
    from .wino import ConvNormSequential
    if checkpoint is not None:
        A._fmt(checkpoint)
    n = 0
    places = {}
    for mod in model.modules():
        for kid in mod._modules.values():
            places[id(kid)] = places.get(id(kid), 0) + 1

    def take(norm, act):
        norm.__class__ = GroupNormAct
        norm.act, norm.act8_format = act, checkpoint

    def alone(norm):
        return places[id(norm)] == 1 and not A.hooked(norm)

    for mod in list(model.modules()):
        if "forward" in mod.__dict__:
            continue
        if type(mod).forward in (nn.Sequential.forward, ConvNormSequential.forward):
            kids = list(mod._modules.items())
            for (_, a), (kb, b) in zip(kids, kids[1:]):
                if type(a) is nn.GroupNorm and alone(a) and A.act_name(b):
                    take(a, A.act_name(b))
                    mod._modules[kb] = nn.Identity()
                    n += 1
        elif type(mod).forward is ConvModule.forward and mod.with_norm and type(mod.norm) is nn.GroupNorm:
            act = A.act_name(mod.activate) if mod.with_activation and alone(mod.norm) else None
            take(mod.norm, act or "none")
            if act:
                mod.activate = nn.Identity()
            n += 1
    for mod in model.modules():
        if type(mod) is nn.GroupNorm:
            take(mod, "none")
            n += 1
        elif type(mod) is GroupNormAct and checkpoint is not None:
            mod.act8_format = checkpoint
    return n
