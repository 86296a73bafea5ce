"""Group norm on the GPU: which of its forms a size takes, and the sizes at which they change, against oracle/act8.py."""
import pytest
import torch

from test_gpu_gn_act import test_forward_and_backward as _check

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,S,H,C,G", [(600, 16, 4, 256, 32), (520, 25, 5, 200, 25), (512, 64, 8, 72, 9), (511, 9, 3, 96, 3), (530, 65, 5, 64, 2), (700, 33, 11, 40, 5)])
def test_many_small_images(N, S, H, C, G, dtype, fmt):
    """enough images to fill the chip with one workgroup each: several rows a thread over all channels"""
    _check(N, S, H, C, G, dtype, fmt)
