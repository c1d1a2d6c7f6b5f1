"""CPU checks of calls whose launch would pass 2^32 threads: HIP runs what is
left modulo 2^32 of them without an error, so the host refuses them."""
from __future__ import annotations

import pytest

FAKE = 4096   # an address that a refused call never uses
ODD = 4096 + 4

NONE = None
BIG, ROWS = 1 << 32, 1 << 24

CASES = {
    # name, arguments: no 16-byte rows, so that an element (or a row) takes a thread (or a wave)
    "rms_norm": ("hydra_rms_norm_fwd", (FAKE, FAKE, FAKE, 1 << 26, 3, 3, 3, 1e-6, 0, NONE)),
    "residual_norm": ("hydra_residual_norm_fwd", (FAKE, 3, NONE, 0, 1.0, NONE, NONE, FAKE, 1e-6, 1, NONE, 0, FAKE, 3,
                                                  1 << 26, 3, 0, 0, NONE)),
    "swiglu": ("hydra_swiglu_fwd", (FAKE, FAKE, FAKE, 1 << 20, 4097, 4097, 4097, 4097, 1, NONE)),
    "swiglu_bwd": ("hydra_swiglu_bwd", (FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 20, 4097, 4097, 4097, 4097, 4097, 4097, 1,
                                        NONE)),
    "qk_norm": ("hydra_qk_norm_fwd", (FAKE, FAKE, FAKE, FAKE, BIG, 1, 3, 1.0, 1.0, 1, NONE)),
    "qk_norm, whole rows": ("hydra_qk_norm_fwd", (FAKE, FAKE, FAKE, FAKE, BIG >> 3, 1, 64, 1.0, 1.0, 1, NONE)),
    "qk_norm_bwd": ("hydra_qk_norm_bwd", (FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, BIG, 1, 3, 1.0, 1.0, 1, NONE)),
    "embedding": ("hydra_embedding_fwd", (FAKE, 1 << 20, FAKE, 10, 4097, 4097, 1.0, FAKE, 4097, 1, NONE)),
    "mor_update": ("hydra_mor_update", (FAKE, 4097, FAKE, 4097, FAKE, 4097, FAKE, 1 << 20, 4097, 0, 1, NONE)),
    "mor_route": ("hydra_mor_route", (FAKE, BIG, NONE, NONE, FAKE, 4, 0, 1, NONE)),
    "ce_rows": ("hydra_ce_rows", (FAKE, ROWS, 8, 8, FAKE, -100, FAKE, FAKE, NONE, 0, NONE, 1, NONE)),
    "ce_grad_planes": ("hydra_ce_grad_planes", (FAKE, ROWS, 8, 8, FAKE, -100, ODD, 8, ROWS * 8, FAKE, NONE)),
    "mod_gather": ("hydra_mod_gather", (FAKE, FAKE, FAKE, 1, 1 << 21, 1 << 20, 4097, 4097 << 21, 4097, 1, NONE)),
    "mod_scatter": ("hydra_mod_scatter", (FAKE, FAKE, FAKE, NONE, 1, 1 << 21, 1 << 20, 4097, 4097 << 21, 4097, 0, 1, NONE)),
    "mod_scatter_bwd": ("hydra_mod_scatter_bwd", (FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 1 << 27, 1 << 26, 8, 8 << 27, 8,
                                                  1, NONE)),
    "causal_im2col": ("hydra_causal_im2col", (FAKE, 64, FAKE, 32, 1 << 20, 1, 64, 3, 1, NONE)),
    "causal_col2im": ("hydra_causal_col2im", (FAKE, FAKE, 64, 64, 1 << 20, 1, 64, 3, 0, 1, NONE)),
    "stream_copy": ("hydra_stream_copy", (FAKE, FAKE, 1 << 36, NONE)),
}


@pytest.mark.parametrize("name", list(CASES))
def test_more_threads_than_a_launch_counts(name):
    from hydra_amd import _lib

    entry, args = CASES[name]
    with pytest.raises(ValueError, match="too large|too many|bad size"):
        _lib.call(entry, *args)
