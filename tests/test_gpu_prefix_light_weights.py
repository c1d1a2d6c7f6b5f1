"""GPU tests of fp16 values under many weights that are small beside the largest one:
each is far below fp16's least step, together they are the result."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def run(cuda, hd, G, W, prefix, own, light, groups=64, K=8, page=64):
    """Position 0 has a weight of 1 and a value of 0, every other one a weight of about
    2^light and values near 1000.  All groups read the same pages.  (got, the exact
    result and its bound, [hd])."""
    from hydra_amd.attention import paged_attention

    n = prefix + own
    pages = -(-n // page)
    g = torch.Generator().manual_seed(hd + prefix)
    k = torch.zeros(pages * page, hd, dtype=torch.float16)
    k[1:, 0] = light * math.log(2.0)
    v = (torch.rand(pages * page, hd, generator=g) * 500 + 750).to(torch.float16)
    v[0] = 0
    shape = lambda t: t.view(pages, 1, page, hd).expand(-1, K, -1, -1).contiguous().to(cuda)  # noqa: E731
    N = groups * W
    q = torch.zeros(N, K * G, hd, dtype=torch.float16)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32).expand(N, -1).contiguous()
    got = paged_attention(q.to(cuda), shape(k), shape(v), table.to(cuda), torch.full((N,), n, dtype=torch.int32, device=cuda),
                          scale=1.0, shared=torch.full((groups,), prefix, dtype=torch.int32, device=cuda))
    x = k[:n, 0].double()
    e = torch.exp(x)
    want = (e[:, None] * v[:n].double()).sum(0) / e.sum()
    # A score is one product, exact; times log2 e, less the reference and e to it: within
    # 1 +- 16 u (2 |x| + 1), u = 2^-24, in numerator and sum, which add n terms (u each)
    # and some joins.  The weights as two terms: 2^-22 of each, and 2^-25 of a step where
    # they are below fp16's least one, under a lift of 2^13 that is 2^-38 of the largest.
    u = 2.0 ** -24
    bound = 2 * (16 * u * (2 * float(x.abs().max()) + 1) + (n + 64) * u + 2.0 ** -22) * want.abs() + \
        2.0 ** -38 * n * float(v.max()) + 2.0 ** -11 * want.abs() * 1.01
    return got.cpu().double(), want, bound


# few rows over a prefix (waves in turn) and many (rows of their own, by direct loads; of rows
# off 16 bytes by the general form), at each number of channels
@pytest.mark.parametrize("light", [-20.0, -25.5, -29.0])
@pytest.mark.parametrize("hd,G,W", [(64, 2, 2), (64, 4, 16), (32, 8, 9), (128, 4, 40), (256, 2, 20), (20, 2, 3), (20, 8, 9)])
def test_of_a_prefix(cuda, hd, G, W, light):
    got, want, bound = run(cuda, hd, G, W, 32768, 5, light, groups=64 if hd < 128 else 16)
    err = (got - want).abs()
    assert bool((err <= bound).all()), f"error {err.max():.3e} of {want.max():.3e}, bound {bound.max():.3e}"


@pytest.mark.parametrize("light", [-20.0, -25.5, -29.0])
@pytest.mark.parametrize("hd", [64, 20])
def test_behind_a_prefix(cuda, hd, light):
    got, want, bound = run(cuda, hd, 2, 2, 0, 32768, light, groups=64)
    err = (got - want).abs()
    assert bool((err <= bound).all()), f"error {err.max():.3e} of {want.max():.3e}, bound {bound.max():.3e}"
