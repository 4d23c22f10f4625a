"""What lines_delta refuses of its numbers before it looks at its tensors."""
import math

import pytest
import torch

from drama3_b200 import kernels


@pytest.mark.parametrize("eps", [-1e-6, -1.0, -math.inf, math.nan])
def test_eps_below_zero_is_refused(eps):
    """The C ABI's form of rows as they are, which None says here."""
    x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    plan = kernels.LinesPlan(None, None, None, torch.zeros(2, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), None, None,
                             None, 64, 1)
    with pytest.raises(ValueError, match="eps"):
        kernels.lines_delta(x, x, x, x[..., 0], torch.zeros((1, 4, 64, 64)), plan, eps=eps)
