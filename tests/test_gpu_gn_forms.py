"""Group norm on the GPU: which of its forms a size takes, and the sizes at which they change, against oracle/act8.py."""
import pytest
import torch

from test_gpu_gn_act import ONE, test_forward_and_backward as _check, test_large_batches as _check_large

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,S,H,C,G", [(600, 16, 4, 256, 32), (520, 25, 5, 200, 25), (512, 64, 8, 72, 9), (511, 9, 3, 96, 3), (530, 65, 5, 64, 2), (700, 33, 11, 40, 5)])
def test_many_small_images(N, S, H, C, G, dtype, fmt):
    """enough images to fill the chip with one workgroup each: several rows a thread over all channels"""
    _check(N, S, H, C, G, dtype, fmt)


def _form(dtype, N, S, C, G, fmt=None, backward=False):
    from distill_bev_amd import _lib as L
    from distill_bev_amd import act8 as A
    return L.call("dbev_gn_act_form", A.DTYPES[dtype], N, S, C, G, A.FORMATS[fmt] if fmt else 0, int(backward))


# like ONE, with the image count that brings every type's tiles to 2048: 512 groups of two channels, several groups a wave of a collector
MANY_GROUPS = (33, 2111, 1, 1024, 512)


@pytest.mark.parametrize("dtype,fmt,act", [(torch.float32, None, "silu"), (torch.bfloat16, None, "gelu"), (torch.bfloat16, "int8", "silu"),
                                           (torch.float16, "e4m3", "gelu")])
def test_many_groups_in_one_pass(dtype, fmt, act):
    N, S, H, C, G = MANY_GROUPS
    assert _form(dtype, N, S, C, G, fmt) == 2
    _check_large(N, S, H, C, G, dtype, fmt, act)


def test_the_sizes_of_the_tests_take_the_forms_that_they_are_meant_for():
    for N, S, H, C, G in ONE:
        assert _form(torch.float32, N, S, C, G) == 2 and _form(torch.float32, N, S, C, G, "int8", True) == 2
        if C != 1024:                                                      # (MANY_GROUPS is its 16-bit counterpart)
            assert _form(torch.bfloat16, N, S, C, G) == 2 and _form(torch.float16, N, S, C, G, "e4m3") == 2
        assert _form(torch.bfloat16, N, S, C, G, None, True) == 0          # 16-bit gradients: two launches
    for N, S, C, G in ((3, 300, 200, 25), (2, 512, 72, 9), (600, 16, 256, 32), (40, 9, 32, 32)):
        assert _form(torch.float32, N, S, C, G) == 1 and _form(torch.float32, N, S, C, G, None, True) == 0
    assert _form(torch.float32, 2, 513, 32, 4) == 0 and _form(torch.float32, 2, 512, 32, 4) == 1
    assert _form(torch.float32, 2, 12, 33, 4) == -1 and _form(torch.float32, 0, 12, 32, 4) == -1


@pytest.mark.parametrize("fmt", [None, "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,S,H,C,G", [(1, 40, 4, 3000, 3000), (2, 33, 3, 2058, 343), (1, 70, 7, 1030, 10), (2, 21, 3, 4104, 27), (1, 12, 3, 65536, 65536)])
def test_groups_across_column_ranges(N, S, H, C, G, dtype, fmt):
    """rows of several workgroups' channels: groups of one channel, groups that lie in two ranges, a group in many"""
    assert _form(dtype, N, S, C, G, fmt, True) == 0
    _check(N, S, H, C, G, dtype, fmt)
