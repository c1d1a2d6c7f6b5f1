"""GPU tests of a step of beam search against the oracle in fp64; the bound of
the scores is derived in oracle/beam.py."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import beam as ob

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(cuda, logits, scores, count, form=lambda t: t):
    """Scores within the bound, rank by rank; beams and tokens those of the oracle, unless
    two scores are closer than twice the bound (then the one chosen has that
    rank's score within the bound, and nothing is chosen twice)."""
    from hydra_amd.kernels import beam_select

    want, beams, tokens = ob.select(logits, scores, count)
    bound = ob.score_bound(logits, scores, want)
    got = beam_select(form(logits.to(cuda)), scores.to(cuda), count)
    B, W = scores.shape
    s, b, t, r = (x.cpu() for x in got)
    assert s.shape == b.shape == t.shape == r.shape == (B, count)
    assert (s.dtype, b.dtype, t.dtype, r.dtype) == (torch.float32, torch.int64, torch.int64, torch.int32)
    assert torch.equal(s.isnan(), want.isnan()) and torch.equal(s == -math.inf, want == -math.inf)
    fine = torch.isfinite(want)
    assert bool(((s.double() - want).abs() <= bound)[fine].all()), float((s.double() - want).abs()[fine].max())
    assert torch.equal(r.long(), torch.arange(B)[:, None] * W + b)
    other = (b != beams) | (t != tokens)
    assert not bool(other[~fine].any())
    flat = b * logits.shape[1] + t
    assert all(len(set(x)) == count for x in flat.tolist())
    if bool(other.any()):
        at = other.nonzero()
        lp = torch.log_softmax(logits.double(), -1)
        for i, j in at.tolist():
            mine = float(scores[i, b[i, j]].double() + lp[i * W + b[i, j], t[i, j]])
            assert 0 < abs(mine - float(want[i, j])) <= 2 * float(bound[i, j]), (i, j)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,W,V,count", [(1, 1, 1, 1), (1, 4, 50257, 4), (3, 5, 1003, 10), (2, 16, 4099, 32), (1, 1, 7, 7),
                                         (32, 8, 2000, 16), (1, 2, 300000, 128), (2, 1024, 33, 128), (600, 1, 50, 3),
                                         (1, 3, 2048, 65)])
def test_sizes(cuda, dtype, B, W, V, count):
    g = torch.Generator().manual_seed(V + W)
    check(cuda, (torch.randn(B * W, V, generator=g) * 2.5).to(dtype), torch.randn(B, W, generator=g) * 2 - 20, count)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_scores(cuda, dtype):
    """The lowest beam, then the lowest token."""
    x = torch.zeros(6, 3000, dtype=dtype)
    check(cuda, x, torch.zeros(2, 3), 100)
    x[:, 1::2] = -0.0
    check(cuda, x, torch.zeros(2, 3), 100)
    x[1, 2500:] = 1
    x[4, :3] = 1
    check(cuda, x, torch.tensor([[0.0, 0.0, 0.0], [0.0, 0.0, -1e-3]]), 128)
    g = torch.Generator().manual_seed(1)
    check(cuda, torch.randint(0, 3, (4, 20000), generator=g).to(dtype), torch.zeros(1, 4), 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [-math.inf, "lowest"])
def test_masked_tokens(cuda, dtype, masked):
    """Few tokens allowed, none in a row, more asked for than allowed."""
    low = torch.finfo(dtype).min if masked == "lowest" else masked
    g = torch.Generator().manual_seed(7)
    x = torch.full((6, 30011), low, dtype=dtype)
    for row, allowed in enumerate((12, 1, 3, 40, 0, 2)):
        x[row, torch.randperm(30011, generator=g)[:allowed]] = torch.randn(allowed, generator=g).to(dtype)
    check(cuda, x, torch.tensor([[0.0, -1.0, -2.0], [-3.0, -0.5, 0.0]]), 20)
    check(cuda, x[:, :5], torch.tensor([[0.0, -1.0, -2.0], [-3.0, -0.5, 0.0]]), 15)


def test_beams_that_do_not_count_yet(cuda):
    """A text's first step: one beam with a score, the others -inf; fewer tokens than continuations."""
    g = torch.Generator().manual_seed(2)
    scores = torch.full((2, 4), -math.inf)
    scores[:, 0] = 0
    check(cuda, torch.randn(8, 5000, generator=g), scores, 8)
    check(cuda, torch.randn(8, 3, generator=g), scores, 10)
    check(cuda, torch.randn(8, 3, generator=g), torch.full((2, 4), -math.inf), 12)


@pytest.mark.parametrize("bad", [float("nan"), math.inf])
def test_rows_and_scores_that_are_not_numbers(cuda, bad):
    """They come first, and show."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, 4000, generator=g)
    x[4, 3999] = bad
    x[8] = bad
    scores = torch.randn(3, 3, generator=g)
    got = check(cuda, x, scores, 6)
    assert got.scores[1].isnan().all() and got.beams[1].tolist() == [1] * 6 and got.tokens[1].tolist() == list(range(6))
    scores[0, 2] = float("nan")
    assert check(cuda, x, scores, 6).beams[0].tolist() == [2] * 6


def test_far_scores_keep_their_order(cuda):
    """Scores of thousands, where fp32 has no room for the logits' differences."""
    g = torch.Generator().manual_seed(5)
    check(cuda, torch.randn(4, 999, generator=g) * 1e-3, torch.tensor([[-70000.0, -70000.0, -70000.5, -70000.0]]), 40)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(cuda, dtype):
    """Rows that begin anywhere, of a wider tensor, transposed, broadcast."""
    g = torch.Generator().manual_seed(6)
    x, s = torch.randn(6, 1001, generator=g).to(dtype), torch.randn(2, 3, generator=g)
    for first in range(8):
        def form(t, first=first):
            wide = torch.full((6, 1001 + 17), 99.0, dtype=dtype, device=t.device)
            wide[:, first:first + 1001] = t
            return wide[:, first:first + 1001]
        check(cuda, x, s, 9, form)
    check(cuda, x, s, 9, lambda t: t.t().contiguous().t())
    check(cuda, x[:1].expand(6, 1001), s, 9, lambda t: t[:1].expand(6, 1001))


def test_no_texts(cuda):
    from hydra_amd.kernels import beam_select

    got = beam_select(torch.zeros(0, 50, device=cuda), torch.zeros(0, 4, device=cuda), 5)
    assert got.scores.shape == got.rows.shape == (0, 5)


def test_refusals(cuda):
    from hydra_amd.kernels import beam_select

    x, s = torch.zeros(8, 50, device=cuda), torch.zeros(2, 4, device=cuda)
    for args, text in (((x[0], s, 1), "must be"), ((x, s[:1], 1), "must be"), ((x, s.double(), 1), "float32"),
                       ((x, s, 0), "at most"), ((x, s, 129), "at most"), ((x[:, :3], s, 13), "at most")):
        with pytest.raises(ValueError, match=text):
            beam_select(*args)
    with pytest.raises(TypeError, match="dtype"):
        beam_select(x.double(), s, 1)
    with pytest.raises(RuntimeError, match="no gradient"):
        beam_select(x.requires_grad_(), s, 1)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        beam_select(x.detach().cpu(), s, 1)
