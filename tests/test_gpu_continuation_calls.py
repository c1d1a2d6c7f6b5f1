"""GPU tests of calls of the operators that continue several texts which their
documentation allows and the other files pass over."""
from __future__ import annotations

import pytest
import torch

from test_gpu_prefix_attention import EIGHT, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", EIGHT)
def test_nothing_to_do_of_any_strides(cuda, eight):
    """An empty tensor counts as contiguous whatever its strides are."""
    from hydra_amd.attention import paged_attention, store_pages

    pages = torch.zeros(2, 2, 16, 8, device=cuda).to(eight)
    scales = tuple(torch.ones(2, 2, 16, device=cuda) for _ in range(2))
    before = pages.view(torch.int8).clone()
    for n, s in ((0, 4), (3, 0), (0, 0)):
        k = torch.zeros(n, 2, 8, s, device=cuda).transpose(2, 3)
        assert k.stride(-1) != 1 or s == 0
        wide = torch.zeros(n, 2, s, 16, device=cuda)[..., ::2]
        slots = torch.zeros(n, s, dtype=torch.int64, device=cuda)
        for rows in (k, wide):
            store_pages(rows, rows, pages, pages.clone(), slots, scales=scales)
    assert torch.equal(pages.view(torch.int8), before)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=cuda)  # noqa: E731
    for q in (torch.zeros(0, 8, 4, device=cuda).transpose(1, 2), torch.zeros(0, 4, 16, device=cuda)[..., ::2]):
        for kw in (dict(scales=scales), dict(scales=scales, shared=ints(0))):
            assert paged_attention(q, pages, pages, ints(0, 3), ints(0), **kw).shape == (0, 4, 8)
        plain = torch.zeros(2, 2, 16, 8, device=cuda)
        assert paged_attention(q, plain, plain, ints(0, 3), ints(0), shared=ints(0)).shape == (0, 4, 8)


def test_recorded_scales_are_refused(cuda):
    """As recorded pages are: their gradient would be lost without a word."""
    from hydra_amd.attention import copy_pages, paged_attention, read_pages, store_pages

    case = Case([[40, 50], [33, 60]], [32, 16], 4, 2, 32, 16, torch.bfloat16, torch.int8, seed=1)
    q, kp, vp, table, lengths, shared = (t.to(cuda) for t in (case.q, case.kp, case.vp, case.table, case.lengths, case.shared))
    rows, slots = torch.zeros(1, 2, 3, 32, device=cuda), torch.arange(3, device=cuda)[None]
    pair = torch.tensor([0], dtype=torch.int32, device=cuda), torch.tensor([1], dtype=torch.int32, device=cuda)
    for which in (0, 1):
        scales = [s.to(cuda) for s in case.scales]
        scales[which].requires_grad_()
        calls = (lambda: paged_attention(q, kp, vp, table, lengths, scales=scales),
                 lambda: paged_attention(q, kp, vp, table, lengths, scales=scales, shared=shared),
                 lambda: store_pages(rows, rows, kp, vp, slots, scales=scales),
                 lambda: read_pages(kp, vp, slots, scales=scales, dtype=torch.bfloat16),
                 lambda: copy_pages(kp, vp, *pair, scales=scales))
        for call in calls:
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad():
                call()
        scales[which].requires_grad_(False)
        with torch.autograd.forward_ad.dual_level():
            scales[which] = torch.autograd.forward_ad.make_dual(scales[which], torch.ones_like(scales[which]))
            for call in calls:
                with pytest.raises(RuntimeError, match="no forward-mode"):
                    call()


@pytest.mark.parametrize("rows", [4, 300])
def test_a_page_that_a_row_holds_twice(cuda, rows):
    """Goes back once."""
    from hydra_amd.attention import fork_pages

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    lengths, extra = [48] + [0] * (rows - 1), [0] * 9
    table = [[3, 5, 3, -1]] + [[-1] * 4] * (rows - 1)
    extra[3] = 1
    t = [i32(lengths), i32(table), i32([8, 0, 0, 0, 0]), i32([1]), i32(extra)]
    fork = fork_pages(i32([-1] + list(range(1, rows))), *t, 16)
    assert t[3].item() == 3 and t[2].tolist()[:3] == [8, 3, 5]
    assert not t[4].any() and not t[0].any() and (t[1] == -1).all() and fork.granted.all()


@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("W", [2, 40])
def test_a_scale_that_is_no_number(cuda, eight, W):
    """Shows in every result, also of requests that end with the prefix, whichever form
    the rows go through."""
    case = Case([[192 + i % 3 for i in range(W)]], [192], 4, 2, 64, 16, torch.bfloat16, eight, seed=1)
    assert case.call(cuda, scale=float("nan")).isnan().all()
    for scale in (1e-39, -1e-39):  # below fp32's normal numbers
        case.check(cuda, scale=scale)
