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
