"""The norm that clipping returns where a gradient is not finite."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [10, 50000, 100001])
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_norm_of_what_is_not_finite(cuda, n, norm_type, dtype):
    from voodoo_quant.training.grad_clip import clip_grad_norm_, grad_norm

    for bad in (math.nan, math.inf, -math.inf):
        for at in (0, n // 2, n - 1):
            p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda))
            p.grad = torch.ones(n, dtype=dtype, device=cuda)
            p.grad[at] = bad
            for norm in (grad_norm([p.grad], norm_type), clip_grad_norm_([p], math.inf, norm_type),
                         clip_grad_norm_([p], 1.0, norm_type)):
                assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
