"""GPU tests of requests that go on from what others hold: tables, stacks and
holders against the oracle's lists, pages and rows against plain indexing."""
from __future__ import annotations

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu


def state(groups, width, page, seed, spare=20, P=12, empty=False):
    """Requests in groups that share full pages, as forks leave them."""
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))  # noqa: E731
    lengths, rows, extra = [], [], {}
    ids = iter(torch.randperm(groups * (width + 1) * P + spare, generator=g).tolist())
    for _ in range(groups):
        prefix = r(0, (P - 3) * page)
        common = [next(ids) for _ in range(prefix // page)]
        holders = 0
        for _ in range(width):
            if empty and r(0, 3) == 0:
                lengths.append(0)
                rows.append([-1] * P)
                continue
            n = prefix + r(0, 2 * page)
            mine = common + [next(ids) for _ in range(-(-n // page) - len(common))]
            holders += 1
            lengths.append(n)
            rows.append(mine + [7] * (P - len(mine)))  # what lies behind a request's pages does not matter
        for p in common:
            extra[p] = max(holders - 1, 0)
        if not holders:
            spare += len(common)
    left = list(ids)[:spare]
    pages = groups * (width + 1) * P + spare + 20
    return lengths, rows, left, [extra.get(p, 0) for p in range(pages)], pages


def run(cuda, parents, lengths, rows, stack, count, extra, page):
    from hydra_amd.attention import fork_pages

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    t = [i32(lengths), i32(rows), i32(stack), i32([count]), i32(extra)]
    fork = fork_pages(i32(parents), *t, page)
    got = [t[0].tolist(), t[1].tolist(), t[2].tolist(), t[3].item(), t[4].tolist(), fork.sources.tolist(),
           fork.copies.tolist(), fork.parents.tolist(), fork.granted.tolist()]
    want = op.fork(parents, lengths, rows, stack, count, extra, page)
    top = want[3]
    names = ("lengths", "table", "stack", "count", "extra", "sources", "copies", "parents", "granted")
    for name, a, b in zip(names, got, want):
        if name == "stack":
            a, b = a[:top], b[:top]
        assert a == b, name
    return got


@pytest.mark.parametrize("empty", [False, True])
@pytest.mark.parametrize("groups,width,page", [(1, 1, 16), (1, 4, 64), (5, 3, 16), (40, 8, 32), (300, 2, 16)])
def test_forks(cuda, groups, width, page, empty):
    """Within the groups, twice (what the first leaves is a state too)."""
    lengths, rows, stack, extra, pages = state(groups, width, page, groups + width, empty=empty, spare=2 * groups * width)
    g = torch.Generator().manual_seed(3)
    stack = stack + [0] * (pages - len(stack))
    count = 2 * groups * width
    for _ in range(2):
        parents = [i // width * width + int(torch.randint(0, width, (1,), generator=g)) for i in range(groups * width)]
        got = run(cuda, parents, lengths, rows, stack, count, extra, page)
        lengths, rows, stack, count, extra = got[:5]


def test_parents_of_any_kind(cuda):
    """Outside the rows (they end), across groups, all from one, everyone his own."""
    lengths, rows, stack, extra, pages = state(4, 4, 16, 8, spare=40)
    N = 16
    g = torch.Generator().manual_seed(5)
    for parents in ([-1] * N, list(range(N)), [3] * N, [N, -2**31, 2**31 - 1] + list(range(3, N)),
                    torch.randperm(N, generator=g).tolist(), torch.randint(-2, N + 2, (N,), generator=g).tolist()):
        run(cuda, parents, lengths, rows, stack + [0] * (pages - 40), 40, extra, 16)


def test_pages_run_out(cuda):
    """Copies beyond the stack are refused, rows in order, and give up their share."""
    for free in (0, 1, 2):
        run(cuda, [0] * 6, [40] + [0] * 5, [[3, 4, 5, -1]] + [[-1] * 4] * 5, [9, 8, 0, 0, 0], free, [0] * 10, 16)
    run(cuda, [0, 0, 1, 1], [20, 25, 7, 0], [[0, 1], [2, 3], [4, -1], [-1, -1]], [0] * 6, 0, [0] * 6, 16)
    # negative and too large counts, a stack that is too small for what comes back
    run(cuda, [-1, -1], [32, 32], [[0, 1], [2, 3]], [5], -4, [0] * 6, 16)
    run(cuda, [-1, -1], [32, 32], [[0, 1], [2, 3]], [5, 4, 4], 2, [0] * 6, 16)


def test_entries_and_lengths_that_are_wrong(cuda):
    run(cuda, [0, 0, 2, 1], [40, -5, 10**6, 16], [[99, -1, 98, 3], [0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 1, 1]],
        [10, 11, 0, 0], 2, [0] * 12, 16)


def test_pages_go_back_with_their_last_holder(cuda):
    """Shared pages outlive all holders but one."""
    N, page = 4, 16
    lengths, rows, stack, extra, count = [40, 0, 0, 0], [[0, 1, 2]] + [[-1] * 3] * 3, [5, 6, 7] + [0] * 9, [0] * 12, 3
    for parents in ([0] * 4, [-1, 1, 2, 3], [0, -1, 2, 3], [0, 1, 3, 2], [0, 1, 2, -1], [0, 1, -1, 3]):
        got = run(cuda, parents, lengths, rows, stack, count, extra, page)
        lengths, rows, stack, count, extra = got[:5]
    assert count == 6 and sorted(stack[:6]) == [0, 1, 2, 5, 6, 7] and lengths == [0] * 4 and not any(extra)


@pytest.mark.parametrize("N", [2047, 8192])
def test_many_rows(cuda, N):
    g = torch.Generator().manual_seed(N)
    lengths = torch.randint(0, 49, (N,), generator=g).tolist()
    ids = iter(range(N * 3))
    rows = [[next(ids) if c < -(-n // 16) else -1 for c in range(3)] for n in lengths]
    used = next(ids)
    pages = used + N
    stack = list(range(used, pages)) + [0] * used
    run(cuda, torch.randint(-1, N, (N,), generator=g).tolist(), lengths, rows, stack, N, [0] * pages, 16)


EIGHT = [torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, *EIGHT])
@pytest.mark.parametrize("K,page,hd", [(2, 16, 64), (1, 64, 3), (3, 16, 20), (1, 4096, 16)])
def test_copied_pages(cuda, dtype, K, page, hd):
    from hydra_amd.attention import copy_pages

    g = torch.Generator().manual_seed(page)
    fresh = lambda: torch.randint(-100, 100, (11, K, page, hd), generator=g, dtype=torch.int8)  # noqa: E731
    kp, vp = ((x.view(dtype) if dtype in EIGHT else x.to(dtype)).to(cuda) for x in (fresh(), fresh()))
    scales = [torch.rand(11, K, page, generator=g).to(cuda) for _ in range(2)] if dtype in EIGHT else None
    want = [t.clone() for t in (kp, vp, *(scales or ()))]
    sources, copies = [4, -1, 2, 11, 0, 4, 5], [7, 8, -1, 9, 11, 10, 3]
    for a, b in ((4, 7), (4, 10), (5, 3)):
        for t in want:
            (t.view(torch.int8) if dtype in EIGHT and t.dtype == dtype else t)[b] = \
                (t.view(torch.int8) if dtype in EIGHT and t.dtype == dtype else t)[a]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    # pages in a pool of other strides
    kp = kp.view(torch.int8).view(dtype).transpose(1, 2).contiguous().transpose(1, 2) if dtype not in EIGHT else kp
    copy_pages(kp, vp, i32(sources), i32(copies), scales=scales)
    raw = lambda t: t.view(torch.int8) if t.dtype in EIGHT else t  # noqa: E731
    for got, exp in zip((kp, vp, *(scales or ())), want):
        assert torch.equal(raw(got), raw(exp))


@pytest.mark.parametrize("N,shape,dtype", [(1, (4,), torch.float32), (2, (3,), torch.int64), (5, (7, 96), torch.bfloat16),
                                           (256, (5, 1536), torch.bfloat16), (300, (1,), torch.uint8), (8192, (33,), torch.int16),
                                           (33, (100003,), torch.uint8), (1000, (), torch.bool), (17, (4, 4), torch.float64)])
def test_rows_taken_along(cuda, N, shape, dtype):
    from hydra_amd.attention import take_rows

    g = torch.Generator().manual_seed(N)
    x = torch.randint(0, 2 if dtype == torch.bool else 100, (N, *shape), generator=g).to(dtype).to(cuda)
    parents = torch.randint(-1, N + 1, (N,), generator=g)
    keep = (parents < 0) | (parents >= N)
    want = x[torch.where(keep, torch.arange(N), parents).to(cuda)]
    take_rows(x, parents.to(torch.int32).to(cuda))
    assert torch.equal(x, want)


def test_rows_of_a_wider_tensor(cuda):
    from hydra_amd.attention import take_rows

    x = torch.arange(40 * 64, device=cuda).view(40, 64)
    want = x.clone()
    parents = torch.arange(39, -1, -1, dtype=torch.int32, device=cuda)
    want[:, 10:30] = x.flip(0)[:, 10:30]
    take_rows(x[:, 10:30], parents)
    assert torch.equal(x, want)
    with pytest.raises(ValueError, match="not contiguous"):
        take_rows(x[:, ::2], parents)
    with pytest.raises(ValueError, match="not contiguous"):
        take_rows(x[:1].expand(40, 64), parents)
