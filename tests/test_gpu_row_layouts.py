"""GPU tests of row-wise operators on tensors whose dimensions of one element
have strides of their own (one decoding step, time first), and on no rows."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0, 40), (3, 0, 40)])
def test_rms_norm_of_no_rows(cuda, shape):
    """A batch without rows has an empty gradient and the weight's is zero."""
    from hydra_amd.kernels import fused_rms_norm

    x = torch.zeros(shape, device=cuda, requires_grad=True)
    weight = torch.ones(40, device=cuda, requires_grad=True)
    y = fused_rms_norm(x, weight)
    gx, gw = torch.autograd.grad(y.sum(), [x, weight])
    assert y.shape == gx.shape == shape and gw.shape == (40,) and not gw.any()
