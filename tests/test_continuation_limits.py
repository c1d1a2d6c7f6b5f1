"""Sizes that whole numbers of 32 bits do not hold are refused before any launch (CPU)."""
from __future__ import annotations

import ctypes

import pytest


def test_beam_selection_counts_in_32_bits():
    from hydra_amd import _lib

    need = ctypes.c_int64(0)
    ask = lambda B, W, V, n: _lib.call("hydra_beam_select_workspace", B, W, V, n, 1, ctypes.byref(need))  # noqa: E731
    ask(1, 1, (1 << 31) - (1 << 14), 1)
    with pytest.raises(ValueError, match="vocabulary"):
        ask(1, 1, (1 << 31) - (1 << 14) + 1, 1)


def test_shared_prefixes_of_very_many_heads_go_in_pieces():
    """The rows of a launch stay below 2^25: the workspace of more requests grows no further."""
    from hydra_amd import _lib

    need = ctypes.c_int64(0)

    def ask(N, H):
        _lib.call("hydra_prefix_attn_workspace", 1, N, H, 1, 16, 1, 16, 1, 1, ctypes.byref(need))
        return need.value

    assert ask(64, 1 << 19) == ask(2048, 1 << 19) > ask(32, 1 << 19)
