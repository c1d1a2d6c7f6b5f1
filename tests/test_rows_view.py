"""CPU checks of how the row-wise operators see a tensor as rows: whatever the
strides of its dimensions of one element are."""
from __future__ import annotations

import pytest
import torch

from hydra_amd.kernels.fused_ops import _as_rows

LAYOUTS = {
    "contiguous": torch.randn(3, 4, 7),
    "vector": torch.randn(7),
    "one step, time first": torch.randn(1, 4, 7).transpose(0, 1),
    "one sequence": torch.randn(5, 1, 7).transpose(0, 1),
    "one row of a wide one": torch.randn(1, 1, 20)[..., 3:10],
    "ones everywhere": torch.randn(2, 1, 3, 1, 7).permute(1, 0, 3, 2, 4),
    "halves": torch.randn(3, 4, 14)[..., :7],
    "one column": torch.randn(1, 5).t(),
    "one column, three dims": torch.randn(1, 2, 5).permute(1, 2, 0),
    "one element": torch.randn(1, 1, 1),
    "shifted": torch.randn(3, 4, 7)[:, :-1],
    "turned": torch.randn(7, 4).t(),
    "broadcast": torch.randn(7).expand(3, 4, 7),
    "no rows": torch.zeros(3, 0, 7).transpose(0, 1),
    "no batch, turned": torch.zeros(0, 4, 3, 7).transpose(1, 2),
    "no columns": torch.zeros(0, 4).t(),
    "no sequence": torch.zeros(0, 5, 7).transpose(0, 1),
}


@pytest.mark.parametrize("name", list(LAYOUTS))
def test_rows_of_any_layout(name):
    t = LAYOUTS[name]
    x, (rows, stride) = _as_rows(t)
    assert x.shape == t.shape and torch.equal(x, t)
    assert rows * t.shape[-1] == t.numel()
    if t.numel():
        assert torch.equal(torch.as_strided(x, (rows, t.shape[-1]), (stride, 1), x.storage_offset()),
                           t.reshape(-1, t.shape[-1]))


@pytest.mark.parametrize("name", ["contiguous", "one step, time first", "one sequence", "halves", "one column",
                                  "ones everywhere"])
def test_rows_that_need_no_copy(name):
    assert _as_rows(LAYOUTS[name])[0] is LAYOUTS[name]
