"""CPU checks of the sizes that the serving operators take, and of what they
refuse before a request enters."""
from __future__ import annotations

import pytest
import torch

FAKE = 4096  # an address that a refused call never uses


def test_requests_of_a_plan_and_a_release():
    """Loops over the requests are counted in an int, and every workgroup of a
    plan goes over the requests before its own."""
    from hydra_amd import _lib

    for N in ((1 << 24) + 1, (1 << 31) - 1):
        with pytest.raises(ValueError, match="too large"):
            _lib.call("hydra_page_plan", FAKE, FAKE, FAKE, 1, FAKE, 8, FAKE, FAKE, 2 * FAKE, FAKE, FAKE, FAKE, 3 * FAKE,
                      N, 1, 1, 16, 0, None)
        with pytest.raises(ValueError, match="too large"):
            _lib.call("hydra_page_release", FAKE, FAKE, FAKE, 1, FAKE, 8, FAKE, N, 1, 16, None)
        with pytest.raises(ValueError, match="too large"):
            _lib.call("hydra_pool_release", FAKE, FAKE, FAKE, 1, FAKE, 8, FAKE, N, 1, 16, 4, None)


def test_pools_that_no_layer_decodes():
    """A pool whose requests decode would refuse is refused by new_cache."""
    from hydra_amd.attention import CCGQAAttention, PagePool

    with torch.device("meta"):
        narrow = CCGQAAttention(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=64)
        wide = CCGQAAttention(dim=32768, n_heads=64, n_kv_heads=2, max_seq_len=64)
        endless = CCGQAAttention(dim=256, n_heads=4, n_kv_heads=2, use_rope=False)
    many = PagePool(65536, 16, 4, 16, device="cpu")
    with pytest.raises(ValueError, match="65535 requests"):
        narrow.new_cache(many)
    with pytest.raises(ValueError, match="2\\^30"):
        endless.new_cache(PagePool(1, (1 << 30) + 1, 4, 4096, device="cpu"))
    # rings of 8192 + 512 channels in fp32: 5 rows of 34816 bytes a request
    assert 24672 * 5 * 34816 < 1 << 32 <= 24673 * 5 * 34816
    with pytest.raises(ValueError, match="4 GiB"):
        wide.new_cache(PagePool(24673, 16, 4, 16, device="cpu"))
    for layer, pool in ((narrow, PagePool(65535, 16, 4, 16, device="cpu")), (wide, PagePool(24672, 16, 4, 16, device="cpu")),
                        (endless, PagePool(1, 1 << 30, 4, 4096, device="cpu"))):
        with pytest.raises(RuntimeError, match="the pool is on cpu"):  # nothing else against them
            layer.new_cache(pool)


def test_workspace_of_sizes_that_are_refused():
    """A query of heads whose channels pass 64 bits ended the process in a
    division by zero."""
    from hydra_amd import _lib

    for N, Hq, Hkv in ((1024, 1 << 62, 1), (1 << 62, 8, 2), (1, 4097, 1), (65536, 8, 2), (1, 2, 4)):
        assert _lib.query("hydra_ccgqa_decode_prep_workspace", N, Hq, Hkv, 32, 3, 1, 1) == 0
    assert _lib.query("hydra_ccgqa_decode_prep_workspace", 16, 16, 4, 64, 3, 1, 1) > 0


def test_prep_of_an_unknown_type():
    """It took the alignment of weights by a size of 0."""
    from hydra_amd import _lib

    for dtype in (-1, 3, 7):
        with pytest.raises(ValueError, match="unknown dtype"):
            _lib.call("hydra_ccgqa_prep_fwd", FAKE, 192, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16, FAKE, FAKE, FAKE, 3,
                      128, 8, 2, 16, 3, 1, dtype, None)
