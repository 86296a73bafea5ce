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
