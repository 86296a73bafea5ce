"""Group norm in the residual blocks of nets.py on the GPU (nets -> bn_act / norm_act -> gn_act), against the same modules in 64 bits."""
import copy

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("act", ["ReLU", "SiLU", "GELU"])
@pytest.mark.parametrize("kind", ["BasicBlock", "Bottleneck"])
def test_blocks_with_group_norm(kind, act, monkeypatch):
    """the activations inside the block are the norms' epilogues (the last one follows the addition), nothing is counted as a fallback.  fp32 against
    64 bits: three layers of sums of up to 2304 products and the norms between them, 1e-5 of an output's or gradient's norm"""
    from distill_bev_amd import _lib as L
    from distill_bev_amd import act8 as A
    from distill_bev_amd import gn_act as GN
    from distill_bev_amd import nets
    torch.manual_seed(1)
    cls, width = getattr(nets, kind), 64
    down = nn.Sequential(nn.Conv2d(48, width * cls.expansion, 1, bias=False), nn.GroupNorm(8, width * cls.expansion))
    ref = cls(48, width, downsample=down, norm_cfg=dict(type="GN", num_groups=8), act_cfg=dict(type=act)).double()
    for m in ref.modules():
        if isinstance(m, nn.GroupNorm):
            nn.init.normal_(m.weight, 1, 0.2), nn.init.normal_(m.bias, 0, 0.2)
    mod = copy.deepcopy(ref).float().to(DEV).to(memory_format=torch.channels_last)
    norms = 3 if kind == "BasicBlock" else 4
    assert GN.fuse_gn_act_modules(mod) == norms
    calls = []
    call = L.call
    monkeypatch.setattr(L, "call", lambda name, *a, **k: calls.append((name, a)) or call(name, *a, **k))
    x, gy = torch.randn(2, 48, 20, 24), torch.randn(2, width * cls.expansion, 20, 24)
    xa = x.to(DEV).to(memory_format=torch.channels_last).requires_grad_(True)
    L.fallback_reset()
    y = mod(xa)
    y.backward(gy.to(DEV).to(memory_format=torch.channels_last))
    acts = sorted(a[9] for n, a in calls if n == "dbev_gn_act_forward")
    assert acts == sorted([0, 0] + [A.ACTS[act.lower()]] * (norms - 2))      # the last norm and the identity branch's: no activation
    assert L.fallback_counts()["total"] == 0
    xd = x.double().requires_grad_(True)
    yd = ref(xd)
    yd.backward(gy.double())
    rel = lambda a, r: float((a.detach().cpu().double() - r).norm() / r.norm())        # noqa: E731
    assert rel(y, yd.detach()) < 1e-5 and rel(xa.grad, xd.grad) < (1e-5 if act != "ReLU" else 1e-3)   # (a ReLU next to zero may open the other way)
    for (name, p), q in zip(mod.named_parameters(), ref.parameters()):
        assert rel(p.grad, q.grad) < (1e-5 if act != "ReLU" else 1e-3), name


def test_block_norms_keep_checkpoints():
    """with a format the block's norms keep 8 bits of their inputs: 4 - 33 / 32 bytes a value less for every norm"""
    from distill_bev_amd import gn_act as GN
    from distill_bev_amd import nets
    x = torch.randn(2, 256, 40, 40, device=DEV).to(memory_format=torch.channels_last)

    def kept(fmt):
        torch.manual_seed(2)
        m = nets.Bottleneck(256, 64, norm_cfg=dict(type="GN", num_groups=8), act_cfg=dict(type="SiLU")).to(DEV).to(memory_format=torch.channels_last)
        GN.fuse_gn_act_modules(m, fmt)
        own = {q.untyped_storage().data_ptr() for q in m.parameters()}
        held, alive = {}, []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: alive.append(t) or held.__setitem__(t.untyped_storage().data_ptr(),
                                                                                                   t.untyped_storage().nbytes()) or t, lambda t: t):
            y = m(x.clone().requires_grad_(True))
        return y.detach(), sum(b for p, b in held.items() if p not in own)

    y, a = kept(None)
    y8, b = kept("int8")
    assert torch.equal(y, y8)
    assert a - b >= 2 * 1600 * (64 + 64 + 256) * (4 - 33 / 32) - (1 << 14)
