"""qkv_norm_rope at every form that a head's width, its pairs and the rows' alignment choose, against 64 bits; linear's few tokens at either form."""
import pytest
import torch

from speed3r_b200 import _lib, ops
from test_gpu_dense_ops import ACTS, BF16, F16, FP32, Linear, Qkv

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_status():
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


# channels, axes, pairs: vectors of two, two or three of them for each of 8, 16, 32 threads; single elements, three or four for each of 8, 16, 32
WIDTHS = [(40, 2, 10), (60, 1, 30), (72, 2, 18), (88, 2, 22), (100, 1, 50), (120, 2, 30), (152, 2, 38), (184, 2, 46), (200, 2, 50), (248, 2, 62), (256, 1, 126),
          (30, 1, 15), (34, 2, 8), (46, 1, 23), (50, 1, 25), (64, 3, 5), (66, 1, 33), (90, 2, 21), (100, 2, 25), (126, 1, 63), (130, 1, 65), (190, 2, 47),
          (194, 1, 97), (250, 2, 62), (252, 2, 63)]


@pytest.mark.parametrize("x", (BF16, F16, FP32))
@pytest.mark.parametrize("d, axes, pairs", WIDTHS)
def test_widths(d, axes, pairs, x):
    Qkv(2, 21, 3, 1, d, x=x, axes=axes, pairs=pairs).train()


# the first size has a quarter of the threads without columns, and more of them than fill the GPU: vectors of two take over
@pytest.mark.parametrize("d, T", [(96, 5200), (80, 5200), (192, 2600), (96, 3000), (128, 5200)])
def test_widths_of_many_tokens(d, T):
    Qkv(1, T, 2, 1, d, axes=2).train()


@pytest.mark.parametrize("M", (1, 2, 3, 5, 8))
@pytest.mark.parametrize("N", (1183, 1184, 1185, 2401))
def test_few_tokens_by_channels(M, N):
    """One channel per warp up to eight per SM, two beyond."""
    Linear(M, N, 264, act=ACTS[M % 4], bias=BF16, scale=FP32, residual=F16, out=BF16).train()


@pytest.mark.parametrize("kinds", [(BF16, F16), (F16, BF16), (FP32, BF16)])
@pytest.mark.parametrize("M", (300, 64))
def test_types_of_factors(M, kinds):
    bias, scale = kinds
    for act in ACTS:
        Linear(M, 200, 2056, act=act, bias=bias, scale=scale).train()
