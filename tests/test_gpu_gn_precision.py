"""Group norm statistics of data with outliers and offsets (GPU) against 64 bits, in each of the forms that a size can take."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _data(N, S, C, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(N, S, C, generator=g), 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)


def _maps(t, H):
    N, S, C = t.shape
    return t.to(DEV).view(N, H, S // H, C).permute(0, 3, 1, 2)


def _rows(t):
    return t.detach().cpu().movedim(1, -1).reshape(t.shape[0], -1, t.shape[1]).double()


def _reference(x, G, w, b):
    return F.group_norm(x.double().movedim(1, 2), G, w.double(), b.double(), 1e-5).movedim(1, 2)


@pytest.mark.parametrize("size", [100.0, 1e4])
@pytest.mark.parametrize("N,S,H,C,G", [(1, 2000, 40, 8, 2), (2, 9000, 90, 64, 8), (2, 2500, 50, 33, 3), (1, 40000, 200, 96, 12)])
def test_an_outlier_in_the_first_pixel(N, S, H, C, G, size):
    """Two launches.  M2 is a sum of positive terms throughout: a thread's rows (at most some 40 batches, three roundings each), up to 64 row phases, a
    group's channels (11 at most here): 200 additions at most, each within 2^-24 of the sum so far, i.e. 200 * 2^-24 of the variance and half
    that of rstd; sequential worst cases, so half of it again is ample.  The outlier's own y is D rstd w, where the mean's error (5 * 2^-24 D
    in a chunk, test_gpu_gn_act.py) counts 5 * 2^-24 of it"""
    from distill_bev_amd import gn_act as GN
    x, w, b = _data(N, S, C, 9)
    x[:, 0] = size
    y = _rows(GN.group_norm_act(_maps(x, H), G, w.to(DEV), b.to(DEV), 1e-5))
    ref = _reference(x, G, w, b)
    rel = ((y - ref).abs() / (ref - b.double()).abs())[:, 0]
    assert float(rel.max()) < 55 * 2.0 ** -24, float(rel.max())
