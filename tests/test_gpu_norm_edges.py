"""The norm and dropout on the GPU at the edge of what they take: rows that are not finite, and arrays large enough
to be stored past the caches."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from ferrum_gpu.norm import NormPlan
from gpu_tensor import fill, up, use, values
from test_gpu_norm import rows

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_device(gpu_device):
    yield from use(gpu_device)


@pytest.mark.parametrize("width,dtype", [(200, "bfloat16"), (600, "float32"), (4096, "bfloat16"), (17001, "bfloat16")])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_every_scale_of_a_row_that_is_not_finite_is_nan(gpu_device, width, dtype, group):
    """An infinity, one where the weight is 0, a NaN, finite values whose squares pass float32; the other rows' are not."""
    x, weight = rows((6, width), dtype, 1), torch.randn(width)
    weight[width // 2] = 0
    x[1, -1], x[2, width // 2], x[3, 0], x[4] = float("inf"), -float("inf"), float("nan"), 1e25
    plan = NormPlan(6, width, gpu_device, dtype=dtype, group=group)
    out, scales = fill((6, width), "uint8"), fill((6, -(-width // group) if group else 1))
    plan.forward(up(x), out, weight=up(weight), scales=scales)
    got = values(scales)
    assert np.isnan(got[1:5]).all() and (got[[0, 5]] > 0).all()
