"""GPU tests of the serving operators at their edges: values that are no
numbers behind vanishing weights, derivatives that no kernel gives, launches
beyond one grid, idle rows of blocks."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("length,columns", [(400, 25), (9000, 600)])  # one workgroup, and split
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_values_behind_vanishing_weights(cuda, dtype, length, columns, bad):
    """A value that is seen is in the sum however small its weight is: 0 x NaN
    and 0 x inf are NaN, whichever part of a split context they lie in."""
    from hydra_amd.attention import paged_attention

    page, hd = 16, 32
    pages = -(-length // page)
    kp, vp = torch.zeros(pages, 1, page, hd), torch.ones(pages, 1, page, hd)
    kp[..., 0] = -40.0
    kp[0, 0, :, 0] = 40.0  # scores 400 apart: the weights of all but the first 16 keys vanish in fp32
    vp[(length - 5) // page, 0, (length - 5) % page, 3] = bad
    q = torch.zeros(1, 2, hd)
    q[..., 0] = 5.0
    table = torch.full((1, columns), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages, dtype=torch.int32)
    got = paged_attention(q.to(cuda, dtype), kp.to(cuda, dtype), vp.to(cuda, dtype), table.to(cuda),
                          torch.tensor([length], dtype=torch.int32, device=cuda), scale=1.0).cpu()
    rest = [c for c in range(hd) if c != 3]
    assert not got[..., 3].isfinite().any()
    assert (got[..., rest] == 1).all()
