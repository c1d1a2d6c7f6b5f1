"""GPU tests of calls of the attention over shared prefixes and 8-bit pages and of beam
selection that the other files' sizes pass over, against the oracles in fp64."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_beam_select import check as check_beams
from test_gpu_prefix_attention import DTYPES, EIGHT, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [1, 7, 20, 65, 72, 100, 250])
def test_head_dims_off_16_bytes(cuda, dtype, eight, hd):
    Case([[0, 1, 40, 300], [130, 131, 5, 200]], [40, 129], 6, 2, hd, 16, dtype, eight, seed=hd).check(cuda)
    if eight is not None:
        Case([[n] for n in (0, 1, 33, 400)], [0] * 4, 6, 2, hd, 16, dtype, eight, seed=hd).check(cuda, shared=False)
    Case([[90 + i for i in range(40)]], [80], 8, 2, hd, 32, dtype, eight, seed=hd).check(cuda)


@pytest.mark.parametrize("hd,length", [(16, 1025), (64, 1025), (128, 513), (256, 257), (256, 300)])
@pytest.mark.parametrize("N", [1, 3, 80])
def test_where_requests_begin_to_be_split(cuda, N, hd, length):
    """One workgroup a request up to a number of keys that goes by the heads."""
    for L in (length - 1, length):
        Case([[L - 3 * (i % 5)] for i in range(N)], [0] * N, 4, 1, hd, 16, torch.bfloat16, torch.int8, seed=L,
             P=-(-L // 16)).check(cuda, shared=False)


def test_scale_is_read_in_each_call(cuda):
    case = Case([[60, 61, 62]], [50], 4, 2, 32, 16, torch.float32, seed=2)
    scale = torch.tensor(0.25)
    first = case.call(cuda, scale=scale)
    scale.fill_(0.5)
    assert torch.equal(case.call(cuda, scale=scale), case.call(cuda, scale=0.5))
    assert torch.equal(first, case.call(cuda, scale=0.25))


def test_no_requests(cuda):
    from hydra_amd.attention import paged_attention

    pages = torch.zeros(2, 2, 16, 32, device=cuda)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.zeros(0, 4, 32, device=cuda)
    assert paged_attention(q, pages, pages, ints(0, 3), ints(0), shared=ints(0)).shape == (0, 4, 32)
    scales = torch.ones(2, 2, 16, device=cuda)
    eight = pages.to(torch.int8)
    assert paged_attention(q, eight, eight, ints(0, 3), ints(0), scales=(scales, scales), shared=ints(0)).shape == (0, 4, 32)
    with pytest.raises(ValueError, match="groups"):
        paged_attention(torch.zeros(2, 4, 32, device=cuda), pages, pages, ints(2, 3), ints(2), shared=ints(0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 4, 8, 9, 100, 128])
def test_one_beam_holds_the_best(cuda, dtype, count):
    """Beams of very different scores, of which one or a few have all that is chosen."""
    g = torch.Generator().manual_seed(count)
    scores = -40.0 * torch.arange(64).float().view(1, 64)
    scores[0, 37], scores[0, 11] = 3.0, 2.5
    check_beams(cuda, (torch.randn(64, 9000, generator=g) * 2.5).to(dtype), scores, count)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_equal_ones_than_are_collected(cuda, dtype):
    """In a row (9000 of one value, and again with better ones behind them), over beams (64
    alike), and with few that differ."""
    x = torch.full((2, 9000), -1.5, dtype=dtype)
    x[1, 8000:8100] = 2.0
    check_beams(cuda, x, torch.zeros(2, 1), 128)
    x = torch.zeros(64, 700, dtype=dtype)
    check_beams(cuda, x, torch.zeros(1, 64), 128)
    x[40, 3] = x[63, 699] = 1.0
    check_beams(cuda, x, torch.zeros(1, 64), 64)
    x = torch.full((4, 20000), -math.inf, dtype=dtype)
    x[0, 19999], x[3, 5:4000] = 0.0, 0.0
    check_beams(cuda, x, torch.zeros(1, 4), 100)


@pytest.mark.parametrize("order", [1, -1])
def test_rows_in_order(cuda, order):
    """Ascending and descending logits: neighbours are much alike."""
    x = torch.linspace(-8, 8, 20000).mul(order).expand(6, -1).contiguous()
    check_beams(cuda, x + torch.arange(6).float()[:, None] / 7, torch.tensor([[0.0, -0.1, -3.0], [0.0, 0.0, 0.01]]), 128)
