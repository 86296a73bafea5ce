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


def _mean(x, G):
    """the mean that the forward pass keeps, [N, G], of x [N, S, C] on the device"""
    from distill_bev_amd import _lib as L
    N, S, C = x.shape
    y, st = torch.empty_like(x), torch.empty((2, N, G), device=DEV)
    ws = torch.empty((int(L.call("dbev_gn_act_workspace_bytes", N, S, C, G)),), dtype=torch.uint8, device=DEV)
    L.call("dbev_gn_act_forward", x.data_ptr(), 0, N, S, C, G, None, None, 1e-5, 0, y.data_ptr(), st[0].data_ptr(), st[1].data_ptr(), 0, None, None,
           ws.data_ptr(), ws.numel(), L.raw_stream(DEV))
    return st[0], y


@pytest.mark.parametrize("N,S,C,G,roundings", [(2, 500, 64, 8, 1), (6, 176, 256, 32, 1), (12, 11440, 256, 32, 2), (40, 4200, 64, 8, 2), (2, 3000, 64, 8, 3),
                                               (1, 9000, 30, 2, 3)])
def test_large_offsets_leave_the_mean_its_digits(N, S, C, G, roundings):
    """mean / spread = 1000, a step of the mean is 2^-14 spreads: one rounding, 2^-15, where a workgroup holds the image; one in every tile and
    one behind their sum in the one-pass form; one of a channel's mean, one of the group's, one of all chunks' in the two launches.
    A thread of the first two forms adds up 16 rows of its channels, in pairs, and takes the offset off the sum: eight roundings of sums up to
    16000, root mean square 3.8e-5 of a row, independent over the 32 or more threads and channels that a group has: 7e-6, two
    of them 2^-16 (the tiles' average out).  Everything else is computed on differences of the size of the spread"""
    x = torch.randn(N, S, C, generator=torch.Generator().manual_seed(3)).add_(1000.0).to(DEV)
    mean, y = _mean(x, G)
    ref = x.double().view(N, S, G, C // G).mean((1, 3))
    assert float((mean.double() - ref).abs().max()) <= roundings * 2.0 ** -15 + 2.0 ** -16
    # y: that, times rstd, and the rounding of mean * rstd, which may be beyond 1024, in its constant term
    z = x.double().view(N, S, G, C // G)
    z = (z - ref[:, None, :, None]) / torch.sqrt(z.var((1, 3), correction=0, keepdim=True) + 1e-5)
    assert float((y.double() - z.view(N, S, C)).abs().max()) <= 1.1 * (roundings * 2.0 ** -15 + 2.0 ** -16) + 2.0 ** -14 + 2.0 ** -18
