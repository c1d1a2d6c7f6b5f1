"""What HydraBlock passes on to an attention of the caller's (CPU)."""
from __future__ import annotations

import torch


class Plain(torch.nn.Module):
    """An attention that knows neither pages of 8 bits nor shared prefixes."""

    def new_cache(self, pool, dtype=None):
        return pool, dtype

    def decode(self, x, cache, plan):
        return x, cache, plan


class Sharing(Plain):
    def new_cache(self, pool, dtype=None, page_dtype=None):
        return pool, dtype, page_dtype

    def decode(self, x, cache, plan, shared=None):
        return x, cache, plan, shared


def test_arguments_that_are_not_given_are_not_passed_on(monkeypatch):
    from hydra_amd.model.framework import HydraBlock

    block = HydraBlock(64, n_heads=4, n_kv_heads=1)
    block.norm1 = torch.nn.Identity()
    monkeypatch.setattr(block, "_rest", lambda x, a: a)
    block.attention = Plain()
    assert block.new_cache("pool") == ("pool", None)
    assert block.new_cache("pool", torch.float16) == ("pool", torch.float16)
    assert block.decode(1, 2, 3) == (1, 2, 3)
    block.attention = Sharing()
    assert block.new_cache("pool", None, torch.int8) == ("pool", None, torch.int8)
    assert block.new_cache("pool", page_dtype=torch.int8) == ("pool", None, torch.int8)
    assert block.decode(1, 2, 3) == (1, 2, 3, None)
    assert block.decode(1, 2, 3, 4) == block.decode(1, 2, 3, shared=4) == (1, 2, 3, 4)
