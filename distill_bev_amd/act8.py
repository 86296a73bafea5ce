"""8-bit activation checkpoints and the layers that train on them (csrc/act8.hip, csrc/act8_wgrad.hip).

What a backward pass needs of a layer's input is kept as one byte per value and one scale byte per 32 neighbouring channels -- 1.03 bytes
instead of 2 or 4 -- and read back by the kernels that use it.  The reference's own means of saving activation memory is recomputation
(``with_cp`` -> torch.utils.checkpoint, mmdet3d/models/bricks/res_block.py:11-230), which costs a second forward pass; a checkpoint
costs the rounding of the values that the GRADIENTS see (the forward pass itself is untouched).

    ck = pack(x, "int8")                 # x [..., C]; or a channels-last [N, C, H, W]
    unpack(ck)                           # the values it stands for, in x's shape, layout and type
    activation(x, "gelu", "int8")        # differentiable; keeps the checkpoint of x instead of x
    linear(x, weight, bias, "int8")      # differentiable F.linear; likewise
    conv1x1(x, weight, bias, "int8")     # differentiable 1x1 F.conv2d on a channels-last map; likewise
    weight_gradient(ck, gy, bias=True)   # (gy^T x^, column sums of gy) -- what linear's backward calls

Formats: with a = max |x| of a block of 32 channels and one power of two 2^k per block,
    "int8"   k = floor(log2 a) - 6: whole numbers -127..127; |x - x^| <= 2^(k-1) (2^k where clamped), i.e. a / 128 (a / 64)
    "e4m3"   k = floor(log2 a) - 8 or -7: floats with four significant bits; |x - x^| <= |x| / 16 down to a / 2^14; the topmost values of a
             type, above 63488 in fp16 and 248 * 2^120 in fp32 and bf16, round up to an infinity of it
int8 is the finer one for values that fill their block's range, e4m3 for blocks with outliers.  A block that holds an infinity or a NaN
restores as NaN.  ReLU's derivative is taken at x^, where a positive value below half of the smallest code is zero.

`use_act8(model, fmt)` swaps these layers into a built model; parameters and state-dict keys stay.  The functions above raise on what the
kernels cannot take (linear and conv1x1 under autocast too: they compute in their arguments' type); the modules leave CPU and float64 tensors,
autocast, layers of more than 2^20 channels or 2^31 weights, and calls under torch.jit.trace, forward-mode differentiation or a torch.func
transform to the stock operators (device tensors are counted in the fallback ledger)."""
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch._prims_common import suggest_memory_format
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .gemm_bf6 import Bf6Conv2d, Bf6Linear

FORMATS = {"int8": 1, "e4m3": 2}                               # DBEV_ACT8_*
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}            # DBEV_ACT_*
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # DBEV_DT_*
BLOCK = 32
_tracing_state, _transform_stack = torch._C._get_tracing_state, torch._C._functorch.peek_interpreter_stack      # None outside


def _fmt(fmt):
    if fmt not in FORMATS:
        raise ValueError(f"checkpoint format {fmt!r}: one of {', '.join(FORMATS)}")
    return FORMATS[fmt]


def _act(act):
    if act not in ACTS:
        raise ValueError(f"activation {act!r}: one of {', '.join(ACTS)}")
    return ACTS[act]


def _dtype(t, what="x"):
    if t.dtype not in DTYPES:
        raise L.DbevHipError(f"{what}: float32, bfloat16 or float16 expected, got {t.dtype}")
    return DTYPES[t.dtype]


def transformed(*tensors):
    """is this call traced, differentiated forward (with `tensors`: is one of them a dual tensor), or inside a torch.func transform?  The kernels
    fill tensors through their addresses, which none of these sees: such a call takes the stock operators (modules) or raises (functions)"""
    if _tracing_state() is not None or _transform_stack() is not None:
        return True
    return forward_ad._current_level >= 0 and (not tensors or any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors))


def no_trace(what):
    if _tracing_state() is not None:
        raise L.DbevHipError(f"{what}: torch.jit.trace cannot record it (the modules trace as the stock operators)")


def _no_derivative(what, x):
    no_trace(what)
    if transformed(x):
        raise L.DbevHipError(f"{what}: not under forward-mode differentiation or a torch.func transform (it has no derivative)")


def dense_dim(x):
    """the dimension along which a tensor's blocks of 32 run: the one whose neighbours are neighbours in memory (1 for channels-last maps),
    the last one longer than 1 if there is none"""
    if x.dim() and x.shape[-1] > 1 and x.stride(-1) == 1:
        return x.dim() - 1
    dims = [d for d in range(x.dim()) if x.shape[d] > 1]
    unit = [d for d in dims if x.stride(d) == 1]
    return (unit or dims or [x.dim() - 1])[-1]


def _strides(shape, dim):
    """strides of a dense tensor of `shape` with `dim` innermost, the others in order"""
    st, n = [0] * len(shape), 1
    for d in [dim] + [d for d in range(len(shape) - 1, -1, -1) if d != dim]:
        st[d] = n
        n *= max(1, shape[d])
    return st


def empty_dense(shape, dim, dtype, device):
    if dim == len(shape) - 1:
        return torch.empty(shape, dtype=dtype, device=device)
    return torch.empty_strided(tuple(shape), _strides(shape, dim), dtype=dtype, device=device)


def rows_of(x, dim):
    """x as (tensor to keep alive, rows, C, row stride) with `dim` as the unit-stride channel dimension: a view wherever the other
    dimensions are evenly spaced, a dense copy otherwise (expanded, transposed, unevenly sliced tensors)"""
    C = x.shape[dim]
    rows = x.numel() // C if C else 0
    if C == 0 or rows == 0:
        return x, 0, C, C
    if C > 1 << 30:
        raise L.DbevHipError(f"act8: {C} channels, at most 2^30")
    if dim == x.dim() - 1 and x.is_contiguous():
        return x.view(rows, C), rows, C, C
    t = x.movedim(dim, -1)
    if C == 1 or t.stride(-1) == 1:
        try:
            v = t.view(rows, C)
            stride = v.stride(0) if rows > 1 else C
            if stride >= C:
                return v, rows, C, stride
        except RuntimeError:
            pass
    v = t.contiguous().view(rows, C)
    return v, rows, C, C


class Checkpoint8:
    """What `pack` keeps of a tensor: one uint8 buffer -- the codes [rows, C], then the scale bytes [rows, ceil(C / 32)] --, the format, and
    the tensor's shape, channel dimension and type."""
    __slots__ = ("buf", "rows", "C", "fmt", "shape", "dim", "dtype")

    def __init__(self, buf, rows, C, fmt, shape, dim, dtype):
        self.buf, self.rows, self.C, self.fmt, self.shape, self.dim, self.dtype = buf, rows, C, fmt, tuple(shape), dim, dtype

    @property
    def codes(self):
        return self.buf[:self.rows * self.C].view(self.rows, self.C)

    @property
    def scales(self):
        return self.buf[self.rows * self.C:].view(self.rows, -(-self.C // BLOCK))

    @property
    def nbytes(self):
        return self.buf.numel()

    def __repr__(self):
        return f"Checkpoint8({self.fmt}, shape={self.shape}, {self.dtype}, {self.nbytes} bytes)"


def _buffer(rows, C, dev):
    return torch.empty((rows * (C + -(-C // BLOCK)),), dtype=torch.uint8, device=dev)


def _dim(x, channel_dim):
    if x.dim() == 0:
        raise ValueError("a checkpoint needs a tensor of at least one dimension")
    if channel_dim is None:
        return dense_dim(x)
    if not -x.dim() <= channel_dim < x.dim():
        raise ValueError(f"channel_dim {channel_dim} of a {x.dim()}-dimensional tensor")
    return channel_dim % x.dim()


def pack(x, fmt="int8", channel_dim=None):
    """the 8-bit checkpoint of a device tensor (no autograd).  `channel_dim`: the dimension along which the blocks of 32 run; by default
    the one that is dense in memory (`dense_dim`)."""
    f, dt = _fmt(fmt), _dtype(x)
    _no_derivative("pack", x)
    dev = L.require_cuda(x)
    dim = _dim(x, channel_dim)
    with L.on(dev):
        v, rows, C, stride = rows_of(x.detach(), dim)
        buf = _buffer(rows, C, dev)
        if rows:
            p = buf.data_ptr()
            L.call("dbev_act8_pack", v.data_ptr(), dt, rows, C, stride, f, p, p + rows * C, L.raw_stream(dev))
    return Checkpoint8(buf, rows, C, fmt, x.shape, dim, x.dtype)


def unpack(ck, dtype=None):
    """the values a checkpoint stands for, in the shape and (dense) layout of the packed tensor; `dtype`: the packed tensor's by default"""
    dtype = ck.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise L.DbevHipError(f"unpack: float32, bfloat16 or float16 expected, got {dtype}")
    _no_derivative("unpack", ck.buf)
    dev = L.require_cuda(ck.buf)
    with L.on(dev):
        out = empty_dense(ck.shape, ck.dim, dtype, dev)
        if ck.buf.numel():
            p = ck.buf.data_ptr()
            L.call("dbev_act8_unpack", p, p + ck.rows * ck.C, FORMATS[ck.fmt], ck.rows, ck.C, out.data_ptr(), DTYPES[dtype], L.raw_stream(dev))
    return out


def _act_forward(x, act, fmt, dim):
    """-> act(x), the checkpoint's buffer (None without `fmt`), rows, C"""
    dev = x.device
    with L.on(dev):
        v, rows, C, stride = rows_of(x, dim)
        y = empty_dense(x.shape, dim, x.dtype, dev)
        buf = p = q = None
        if fmt is not None:
            buf = _buffer(rows, C, dev)
            p = buf.data_ptr()
            q = p + rows * C
        if rows:
            L.call("dbev_act8_activation_forward", v.data_ptr(), DTYPES[x.dtype], rows, C, stride, ACTS[act], FORMATS[fmt] if fmt else 0,
                   y.data_ptr(), p, q, L.raw_stream(dev))
    return y, buf, rows, C


class _Activation8(Function):
    @staticmethod
    def forward(ctx, x, act, fmt, dim):
        y, buf, rows, C = _act_forward(x, act, fmt, dim)
        ctx.save_for_backward(buf)
        ctx.cfg = (act, fmt, dim, rows, C)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        buf, = ctx.saved_tensors
        act, fmt, dim, rows, C = ctx.cfg
        dev = gy.device
        with L.on(dev):
            g, _, _, stride = rows_of(gy, dim)
            dx = empty_dense(gy.shape, dim, gy.dtype, dev)
            if rows:
                p = buf.data_ptr()
                L.call("dbev_act8_activation_backward", g.data_ptr(), DTYPES[gy.dtype], stride, p, p + rows * C, FORMATS[fmt], rows, C,
                       ACTS[act], dx.data_ptr(), L.raw_stream(dev))
        return dx, None, None, None


def activation(x, act="gelu", checkpoint="int8", channel_dim=None):
    """act(x), act one of `ACTS` (gelu: the erf form); under autograd the 8-bit checkpoint of x is kept and dx = gy * act'(x^)"""
    no_trace("activation")
    _act(act), _fmt(checkpoint), _dtype(x)
    L.require_cuda(x)
    dim = _dim(x, channel_dim)
    if x.requires_grad and torch.is_grad_enabled() or transformed():        # (transformed: the function raises)
        return _Activation8.apply(x, act, checkpoint, dim)
    return _act_forward(x.detach(), act, None, dim)[0]


def _gradient_fits(Ci, Co):
    return Ci <= 1 << 20 and Co <= 1 << 20 and Ci * Co <= 1 << 31


def _gradient_ok(Ci, Co):
    if not _gradient_fits(Ci, Co):
        raise L.DbevHipError(f"act8: weight gradient of {Ci} -> {Co} channels; at most 2^20 and 2^31 weights")


def _weight_gradient(buf, fmt, Ci, gy2, bias):
    """checkpoint buffer of [M, Ci], gy2 [M, Co] dense -> (gw [Co, Ci], gb [Co] or None) in gy2's type"""
    dev = gy2.device
    M, Co = gy2.shape
    with L.on(dev):
        _gradient_ok(Ci, Co)
        gw = torch.empty((Co, Ci), dtype=gy2.dtype, device=dev)
        gb = torch.empty((Co,), dtype=gy2.dtype, device=dev) if bias else None
        if Co and Ci:
            nbytes = int(L.call("dbev_act8_weight_gradient_workspace_bytes", M, Ci, Co))
            if nbytes == 0:
                raise L.DbevHipError(f"weight_gradient: unsupported sizes {M} x {Ci} -> {Co}")
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
            p = buf.data_ptr()
            L.call("dbev_act8_weight_gradient", gy2.data_ptr(), DTYPES[gy2.dtype], p, p + M * Ci, FORMATS[fmt], M, Ci, Co, gw.data_ptr(),
                   gb.data_ptr() if bias else None, ws.data_ptr(), nbytes, L.raw_stream(dev))
        elif bias and Co:
            gb = gy2.sum(0)
    return gw, gb


def weight_gradient(ck, gy, bias=False):
    """gy^T x^ [Co, Ci] (and with `bias` the sums of gy over its rows, [Co]) in gy's type, for the checkpoint of a layer's input and the
    gradient of its output: gy has the checkpoint's shape but for the channel dimension.  fp32 sums, fp32 accuracy for fp32 gy."""
    _dtype(gy, "gy")
    _no_derivative("weight_gradient", gy)
    dev = L.require_cuda(ck.buf, gy)
    dim, want = ck.dim, ck.shape
    if gy.dim() != len(want) or any(gy.shape[d] != want[d] for d in range(len(want)) if d != dim):
        raise ValueError(f"weight_gradient: gy {tuple(gy.shape)} does not match a checkpoint of {ck.shape} with channels in dimension {dim}")
    with L.on(dev):
        g, rows, Co, stride = rows_of(gy.detach(), dim)
        if rows == 0:
            g = gy.new_empty((0, Co))
        elif stride != Co:
            g = g.contiguous()
        gw, gb = _weight_gradient(ck.buf, ck.fmt, ck.C, g, bias)
    return (gw, gb) if bias else gw


def _check_layer(x, weight, bias, what):
    L.require_cuda(x, weight, bias)
    _dtype(x)
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise L.DbevHipError(f"{what}: x, weight and bias of one type expected, got {x.dtype}, {weight.dtype}"
                             + ("" if bias is None else f", {bias.dtype}"))
    if torch.is_autocast_enabled("cuda"):
        raise L.DbevHipError(f"{what}: not under autocast (the products would be in another type than the arguments)")
    if _recording(weight):
        _gradient_ok(int(weight.shape[1]), int(weight.shape[0]))
    if bias is not None and bias.shape != (weight.shape[0],):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} for {weight.shape[0]} outputs")


def _bias_grad(gy2):
    from . import colsum
    return colsum.channel_sum(gy2) if gy2.dtype == torch.float32 and colsum.eligible(gy2) else gy2.sum(0)


class _Linear8(Function):
    """F.linear on rows x2 [M, K]; the products forward and for the data gradient are those of gemm_bf6.Bf6Linear (the bf16x6 GEMM where its
    shape rule says so, else the library's), the weight and bias gradient come from the checkpoint of x2."""

    @staticmethod
    def forward(ctx, x2, weight, bias, fmt, keep):
        from . import gemm_bf6 as G
        if G.eligible_linear(x2, weight):
            M, K = x2.shape
            if ctx.needs_input_grad[0] and G.shape_ok(M, int(weight.shape[0]), K):
                G.pack_both(weight, M)
            y = G._rows_product(x2, weight, False, bias if bias is not None and bias.is_contiguous() else None)
            if bias is not None and not bias.is_contiguous():
                y.add_(bias)
        else:
            y = F.linear(x2, weight, bias)
        ck = pack(x2, fmt, -1) if keep else None
        ctx.save_for_backward(weight, None if ck is None else ck.buf)
        ctx.fmt = fmt
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        from . import gemm_bf6 as G
        weight, buf = ctx.saved_tensors
        gx = gw = gb = None
        with L.on(gy.device):
            gy = gy.contiguous()
            if ctx.needs_input_grad[0]:
                if (G._ON and G._LIN and gy.dtype == torch.float32 and weight.is_contiguous() and gy.numel() < 2 ** 31
                        and G.shape_ok(gy.shape[0], int(weight.shape[0]), int(weight.shape[1]))):
                    gx = G._rows_product(gy, weight, True)
                else:
                    gx = gy @ weight
            if ctx.needs_input_grad[1]:
                gw, gb = _weight_gradient(buf, ctx.fmt, int(weight.shape[1]), gy, ctx.needs_input_grad[2])
            elif ctx.needs_input_grad[2]:
                gb = _bias_grad(gy)
        return gx, gw, gb, None, None


def linear(x, weight, bias=None, checkpoint="int8"):
    """F.linear(x, weight, bias), differentiable; the 8-bit checkpoint of x is what the weight gradient is computed from"""
    no_trace("linear")
    _fmt(checkpoint)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.shape[1] == 0:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    _check_layer(x, weight, bias, "linear")
    with L.on(x.device):
        x2 = x.reshape(-1, weight.shape[1])
        x2 = x2 if x2.is_contiguous() else x2.contiguous()
        return _Linear8.apply(x2, weight, bias, checkpoint, _recording(weight)).view(*x.shape[:-1], weight.shape[0])


class _Conv1x1_8(Function):
    """F.conv2d(x, weight, bias) for a 1x1 filter on a channels-last map, products as in gemm_bf6, weight and bias gradient from the
    checkpoint of x.  `stats` (bias-free layers): also the output's partial BatchNorm statistics rows, from the epilogue of the bf16x6 GEMM
    ("bf6") or of the fp32 one ("f32", bn_act.conv1x1_stats); the caller has asked that kernel's rule"""

    @staticmethod
    def forward(ctx, x, weight, bias, fmt, keep, stats=None):
        from . import gemm_bf6 as G
        part = None
        if stats == "f32":
            from .bn_act import conv1x1_stats_product
            y, part = conv1x1_stats_product(x, weight)
        elif G.eligible(x, weight):
            M = x.shape[0] * x.shape[2] * x.shape[3]
            if ctx.needs_input_grad[0] and G.shape_ok(M, int(weight.shape[0]), int(weight.shape[1])):
                G.pack_both(weight, M)
            if stats:
                y, part = G.product(x, weight, stats=True)
            else:
                y = G.product(x, weight, bias=bias if bias is not None and bias.is_contiguous() else None)
            if bias is not None and not bias.is_contiguous():
                y.add_(bias.view(1, -1, 1, 1))
        else:
            y = F.conv2d(x, weight, bias)
        ck = pack(x, fmt, 1) if keep else None
        ctx.save_for_backward(weight, None if ck is None else ck.buf)
        ctx.fmt, ctx.x_shape = fmt, tuple(x.shape)
        if stats is None:
            return y
        ctx.mark_non_differentiable(part)
        ctx.set_materialize_grads(False)                                  # no zero tensor for the statistics' (never used) gradient
        return y, part

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, _gpart=None):
        from . import gemm_bf6 as G
        weight, buf = ctx.saved_tensors
        gx = gw = gb = None
        if gy is None:
            return None, None, None, None, None, None
        with L.on(gy.device):
            gy = gy.contiguous(memory_format=torch.channels_last)
            gy2 = gy.permute(0, 2, 3, 1).reshape(-1, gy.shape[1])
            if ctx.needs_input_grad[0]:
                gx = G.data_gradient(gy, weight) if weight.dtype == torch.float32 else None
                if gx is None:
                    x_like = gy.new_empty(1).expand(ctx.x_shape)          # (only its shape is read)
                    gx = torch.ops.aten.convolution_backward(gy, x_like, weight, None, [1, 1], [0, 0], [1, 1], False, [0, 0], 1, [True, False, False])[0]
            if ctx.needs_input_grad[1]:
                gw, gb = _weight_gradient(buf, ctx.fmt, int(weight.shape[1]), gy2, ctx.needs_input_grad[2])
                gw = gw.view(weight.shape)                                # [Co, Ci] in memory: dense in both memory formats of a 1x1 filter
            elif ctx.needs_input_grad[2]:
                gb = _bias_grad(gy2)
        return gx, gw, gb, None, None, None


def conv1x1(x, weight, bias=None, checkpoint="int8"):
    """F.conv2d(x, weight, bias) for a 1x1 filter, stride 1, differentiable; x is taken as (or copied to) a channels-last map and its 8-bit
    checkpoint is what the weight gradient is computed from"""
    no_trace("conv1x1")
    _fmt(checkpoint)
    if weight.dim() != 4 or tuple(weight.shape[2:]) != (1, 1) or x.dim() != 4 or x.shape[1] != weight.shape[1]:
        raise ValueError(f"conv1x1: x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    _check_layer(x, weight, bias, "conv1x1")
    with L.on(x.device):
        return _Conv1x1_8.apply(x.contiguous(memory_format=torch.channels_last), weight, bias, checkpoint, _recording(weight))


def conv1x1_stats(conv, x, kernel):
    """(conv(x), partial BatchNorm statistics rows of it) for a layer that `keeps` x, by the epilogue of `kernel` ("bf6": gemm_bf6.eligible
    says so; "f32": bn_act.conv1x1_bn_ready does)"""
    return _Conv1x1_8.apply(x, conv.weight, None, conv.act8_format, True, kernel)


def conv1x1_module(conv, x):
    """the forward of a 1x1 convolution module that `keeps` x: conv1x1 in the layout that F.conv2d would give (contiguous unless the map or the
    filter is channels-last)"""
    y = conv1x1(x, conv.weight, conv.bias, conv.act8_format)
    if x.is_contiguous(memory_format=torch.channels_last) or suggest_memory_format(conv.weight) == torch.channels_last:
        return y
    return y.contiguous()


def keeps(conv, x):
    """does this call of a 1x1 convolution module keep x as an 8-bit checkpoint?  For code that runs a module's product without its forward
    (nets.Bottleneck, colsum.conv_bn_cancelled_bias)"""
    return (getattr(conv, "act8_format", None) is not None and _plain_1x1(conv) and _recording(conv.weight) and x.dim() == 4 and x.numel() > 0
            and _module_ready(x, conv.weight, conv.bias))


# ---- modules ------------------------------------------------------------------------------------------------------------------------
def _module_ready(x, weight=None, bias=None):
    """may a module's call go to the kernels?  Device tensors of one supported type, a weight whose gradient fits; a device tensor that may not is
    counted."""
    if not (torch.is_tensor(x) and x.is_cuda):
        return False
    why = None
    if x.dtype not in DTYPES or any(p is not None and p.dtype != x.dtype for p in (weight, bias)) or torch.is_autocast_enabled("cuda"):
        why = f"dtype {x.dtype}" + (" under autocast" if torch.is_autocast_enabled("cuda") else "")
    elif weight is not None and not _gradient_fits(int(weight.shape[1]), int(weight.shape[0])):
        why = f"{int(weight.shape[1])} -> {int(weight.shape[0])} channels"
    elif transformed():
        why = "traced or transformed"
    if why:
        L.note_fallback("act8", why)
    return why is None


def _recording(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class Act8Linear(Bf6Linear):
    """nn.Linear (its products: Bf6Linear's) that keeps its input as an 8-bit checkpoint (`act8_format`) while gradients of the weight are recorded; same parameters
    and state-dict keys"""
    act8_format = "int8"

    def forward(self, x):
        if _recording(self.weight) and x.numel() and _module_ready(x, self.weight, self.bias):
            return linear(x, self.weight, self.bias, self.act8_format)
        return super().forward(x)

    def extra_repr(self):
        return super().extra_repr() + f", act8={self.act8_format}"


def _plain_1x1(m):
    return m.kernel_size == (1, 1) and m.stride == (1, 1) and m.padding == (0, 0) and m.dilation == (1, 1) and m.groups == 1


class Act8Conv2d(Bf6Conv2d):
    """1x1, stride-1 nn.Conv2d that keeps its input as an 8-bit checkpoint while gradients of the weight are recorded"""
    act8_format = "int8"

    def forward(self, x):
        if keeps(self, x):
            return conv1x1_module(self, x)
        return super().forward(x)

    def extra_repr(self):
        return super().extra_repr() + f", act8={self.act8_format}"


class Act8Activation(nn.Module):
    """SiLU / GELU (erf) / ReLU that keeps its input as an 8-bit checkpoint while its gradient is recorded"""

    def __init__(self, act, fmt="int8"):
        super().__init__()
        _act(act), _fmt(fmt)
        self.act, self.act8_format = act, fmt

    def forward(self, x):
        if _recording(x) and x.numel() and _module_ready(x):
            return activation(x, self.act, self.act8_format)
        return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[self.act](x)

    def extra_repr(self):
        return f"{self.act}, act8={self.act8_format}"


def hooked(m):
    """has somebody registered hooks on this module, or given it a forward of its own?  They would not run if the module were left out, or see
    other values if it did more"""
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks or "forward" in m.__dict__)


def act_name(m):
    """the `ACTS` name of a plain activation module without hooks, or None"""
    if m is None or hooked(m):
        return None
    if type(m) is nn.ReLU:
        return "relu"
    if type(m) is nn.SiLU:
        return "silu"
    if type(m) is nn.GELU and m.approximate == "none":
        return "gelu"
    return None


def use_act8(model, fmt="int8"):
    """Let the plain Linear and 1x1 / stride-1 convolution modules of `model` (bf16x6 ones included) keep their input as an 8-bit checkpoint,
    and the activations whose input nothing else keeps: every SiLU / GELU, and a ReLU right behind one of those layers in an nn.Sequential
    (elsewhere a ReLU's output is kept by the layer behind it anyway; one that carries hooks stays as it is).  nn.MultiheadAttention reads
    its projections' weights itself and stays as it is.  Returns how many modules changed class.  Idempotent for one format.
    The biased 1x1 layers of a model that has been through train_step.accelerate_modules (BiasSumConv2d) stay what they are and are given the
    format; two kernels that take such a layer as a whole keep its input their own way: the depth head's and the adaptation loss's."""
    from .colsum import BiasSumConv2d
    _fmt(fmt)
    n = 0
    for mod in model.modules():
        to = None
        if type(mod) in (nn.Linear, Bf6Linear):
            to = Act8Linear
        elif type(mod) in (nn.Conv2d, Bf6Conv2d) and _plain_1x1(mod):
            to = Act8Conv2d
        if to is not None:
            mod.__class__ = to
            n += 1
        if isinstance(mod, (Act8Linear, Act8Conv2d, Act8Activation)) or type(mod) is BiasSumConv2d and _plain_1x1(mod):
            mod.act8_format = fmt
    for mod in list(model.modules()):
        kids = list(mod._modules.items())
        for i, (name, child) in enumerate(kids):
            act = act_name(child)
            behind = isinstance(mod, nn.Sequential) and i > 0 and isinstance(kids[i - 1][1], (Act8Linear, Act8Conv2d))
            if act in ("silu", "gelu") or (act == "relu" and behind):
                mod._modules[name] = Act8Activation(act, fmt)
                n += 1
    return n
