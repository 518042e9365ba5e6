"""The norm and dropout on the GPU at the edge of what they take: rows that are not finite, and arrays large enough
to be stored past the caches."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ferrum_gpu.norm import NormPlan
from gpu_tensor import fill, up, use, values
import test_gpu_norm as small

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_device(gpu_device):
    yield from use(gpu_device)


@pytest.mark.parametrize("width,dtype", [(200, "bfloat16"), (600, "float32"), (4096, "bfloat16"), (17001, "bfloat16")])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_every_scale_of_a_row_that_is_not_finite_is_nan(gpu_device, width, dtype, group):
    """An infinity, one where the weight is 0, a NaN, finite values whose squares pass float32; the other rows' are not."""
    x, weight = small.rows((6, width), dtype, 1), torch.randn(width)
    weight[width // 2] = 0
    x[1, -1], x[2, width // 2], x[3, 0], x[4] = float("inf"), -float("inf"), float("nan"), 1e25
    plan = NormPlan(6, width, gpu_device, dtype=dtype, group=group)
    out, scales = fill((6, width), "uint8"), fill((6, -(-width // group) if group else 1))
    plan.forward(up(x), out, weight=up(weight), scales=scales)
    got = values(scales)
    assert np.isnan(got[1:5]).all() and (got[[0, 5]] > 0).all()


LARGE = 16 << 20  # bytes of rows from which on they are stored past the caches


@pytest.mark.parametrize("n,width,dtype", [(2050, 4096, "bfloat16"), (4200, 1001, "float32"), (1030, 8200, "float16"),
                                           (9000, 960, "bfloat16"), (520, 17001, "bfloat16"), (600, 9000, "float32")])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_large_arrays(gpu_device, n, width, dtype, p):
    assert n * width * small.TYPES[dtype].itemsize >= LARGE
    small.test_forward_and_backward(gpu_device, n, width, dtype, p)


@pytest.mark.parametrize("n,width,dtype", [(2050, 4096, "bfloat16"), (4200, 1001, "float32"), (530, 16400, "float16")])
@pytest.mark.parametrize("group", [0, 128])
def test_large_arrays_to_eight_bits(gpu_device, n, width, dtype, group):
    assert n * width * small.TYPES[dtype].itemsize >= LARGE
    small.test_eight_bits(gpu_device, n, width, dtype, group)


@pytest.mark.parametrize("n,dtype", [((8 << 20) + 3, "bfloat16"), ((4 << 20) + 1, "float32")])
def test_large_arrays_dropped(gpu_device, n, dtype):
    assert n * small.TYPES[dtype].itemsize >= LARGE
    small.test_dropout(gpu_device, dtype, n, 0.1)
