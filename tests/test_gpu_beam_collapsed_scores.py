"""GPU tests of beams whose scores are so large that fp64 no longer tells their
continuations apart: these are equal, and the lowest beam and token come first."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_beam_select import DTYPES, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", [-1e30, 1e30, float(torch.finfo(torch.float32).min)])
@pytest.mark.parametrize("W,V,count", [(1, 50257, 4), (3, 9001, 20), (2, 20000, 128), (40, 300, 9), (2, 5, 8)])
def test_all_beams(cuda, dtype, score, W, V, count):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(2 * W, V, generator=g) * 2.5).to(dtype)
    got = check(cuda, x, torch.full((2, W), score), count)
    first = torch.arange(count)
    assert torch.equal(got.tokens.cpu(), (first % V).expand(2, -1)) and torch.equal(got.beams.cpu(), (first // V).expand(2, -1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_tokens(cuda, dtype):
    """Of a row with -inf the other tokens in order, then -inf from the lowest beam on."""
    g = torch.Generator().manual_seed(1)
    x = torch.full((3, 20000), -math.inf, dtype=dtype)
    for row, allowed in enumerate((50, 7, 9000)):
        x[row, torch.randperm(20000, generator=g)[:allowed]] = torch.randn(allowed, generator=g).to(dtype)
    for count in (5, 50, 57, 128):
        check(cuda, x, torch.full((1, 3), -1e30), count)
    check(cuda, x[:2], torch.full((1, 2), -1e30), 128)


@pytest.mark.parametrize("dtype", DTYPES)
def test_beside_beams_that_count(cuda, dtype):
    """One beam with fewer allowed tokens than are asked for, the others at the type's lowest."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 30000, generator=g).to(dtype)
    x[0, 3:] = -math.inf
    scores = torch.full((1, 4), -1e30)
    scores[0, 0] = -1.0
    for count in (3, 4, 12, 100):
        check(cuda, x, scores, count)


@pytest.mark.parametrize("score", [0.0, -20.0])
def test_logits_too_small_to_count(cuda, score):
    """Logits of 1e-30 beside a large one: their differences are lost in any score."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 12000, generator=g) * 1e-30
    x[:, 7000] = 5.0
    check(cuda, x, torch.full((1, 2), score), 40)
    check(cuda, torch.randn(2, 12000, generator=g) * 1e-30, torch.full((1, 2), score), 40)
