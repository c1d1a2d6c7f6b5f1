"""GPU tests of what bounds a pool of pages: entries that are no page."""
from __future__ import annotations

import random

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("N,P,page", [(1, 1, 16), (1, 2500, 16), (7, 5, 32), (256, 9, 16), (700, 40, 16), (3, 1024, 64)])
@pytest.mark.parametrize("pool", [False, True])
def test_release_of_entries_that_are_no_page(cuda, N, P, page, pool):
    """They do not come back; the pages beside them do, in their order."""
    from hydra_amd.attention import release_pages

    rng = random.Random(N * 31 + P)
    for share in (0.0, 0.1, 1.0):
        lengths = [rng.choice([0, 1, P * page, rng.randint(0, P * page), -3, 2**31 - 1]) for _ in range(N)]
        table = [[rng.randrange(5000) for _ in range(P)] for _ in range(N)]
        for row in table:
            for c in range(P):
                if rng.random() < share:
                    row[c] = rng.choice([-1, -9, -2**31] + ([5000, 2**31 - 1] if pool else []))
        done = [rng.random() < 0.7 for _ in range(N)]
        cap = rng.choice([N * P + 3, max(1, N * P // 3)])
        stack, free = [7777] * cap, rng.randint(0, 3)
        free = min(free, cap)
        bound = 5000 if pool else None
        want = op.release(done, lengths, table, stack, free, page, bound)
        ln, t, st, fc = ints(lengths, cuda), ints(table, cuda), ints(stack, cuda), ints([free], cuda)
        release_pages(torch.tensor(done, device=cuda), ln, t, st, fc, page, **({"pages": bound} if pool else {}))
        assert fc.tolist() == [want[3]]
        assert st.tolist() == want[2] and ln.tolist() == want[0] and t.tolist() == want[1]


def test_a_damaged_entry_costs_its_own_request_alone(cuda):
    """Two entries of one request are overwritten with what is no page of the
    pool; after its release no other request is handed them."""
    from hydra_amd.attention import PagePool

    pool = PagePool(3, 64, 8, 16, device=cuda)
    pool.plan(ints([64, 0, 0], cuda), width=64)
    pool.table[0, 1], pool.table[0, 2] = -1, 8
    pool.release(torch.tensor([True, False, False], device=cuda))
    assert pool.free_count.tolist() == [6]
    assert sorted(set(range(8)) - set(pool.free_pages.tolist()[:6])) and all(0 <= p < 8 for p in pool.free_pages.tolist()[:6])
    plan = pool.plan(ints([0, 64, 32], cuda), width=64)
    assert plan.granted.all()
    held = plan.slots[1].tolist() + plan.slots[2, :32].tolist()
    assert all(0 <= s < 8 * 16 for s in held) and len(set(held)) == 96
