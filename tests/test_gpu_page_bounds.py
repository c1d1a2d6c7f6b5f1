"""GPU tests of what bounds a pool of pages: entries that are no page,
stacks near the reach of an int, the longest request, tables of one row or column."""
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


def test_release_onto_a_full_stack_of_the_largest_size(cuda):
    """What finds no room is dropped, also where the stack's height and the
    pages together pass an int."""
    from hydra_amd.attention import release_pages

    cap = 2**31 - 1
    stack = torch.empty(cap, dtype=torch.int32, device=cuda)
    stack[-100:] = 7
    for free in (cap, cap - 2, cap - 40, cap - 90):
        table = torch.arange(80, dtype=torch.int32, device=cuda).view(2, 40)
        lengths, height = ints([640, 600], cuda), ints([free], cuda)
        release_pages(torch.tensor([True, True], device=cuda), lengths, table, stack, height, 16)
        assert height.tolist() == [min(cap, free + 78)] and lengths.tolist() == [0, 0]
        want = [7] * 100
        for j, page in enumerate([*range(40), *range(40, 78)]):
            if free + j < cap:
                want[100 - (cap - free) + j] = page
        assert stack[-100:].tolist() == want
        assert table.tolist() == [[-1] * 40, [-1] * 38 + [78, 79]]
        stack[-100:] = 7


def test_requests_end_at_max_length(cuda):
    """A length that is no whole number of pages."""
    from hydra_amd.attention import PagePool

    for N in (2, 300):  # planned in place, and by several workgroups
        pool = PagePool(N, 20, 2 * N, 16, device=cuda)
        assert pool.max_length == 20 and pool.table.shape == (N, 2)
        plan = pool.plan(ints([21] + [20] * (N - 1), cuda), width=32, from_empty=True)
        assert plan.granted.tolist() == [False] + [True] * (N - 1)
        assert pool.lengths.tolist() == [0] + [20] * (N - 1) and pool.free_count.tolist() == [2]
        plan = pool.plan(ints([19] + [0] * (N - 1), cuda), width=32, from_empty=True)
        assert plan.granted.all()
        plan = pool.plan(ints([1] * N, cuda))
        assert plan.granted.tolist() == [True] + [False] * (N - 1) and plan.slots[1:].eq(-1).all()
        assert not pool.plan(ints([1] * N, cuda)).granted.any()
        assert pool.lengths.tolist() == [20] * N


def test_layer_at_its_full_length(cuda):
    """A layer whose rotation table ends inside a page, served up to its end."""
    from hydra_amd.attention import CCGQAAttention, PagePool
    from oracle import ccgqa as oc

    cfg = oc.CCGQAConfig(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=20)
    params = oc.init_params(cfg, torch.Generator().manual_seed(1), std=0.05)
    m = CCGQAAttention(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=20)
    m.load_state_dict(params)
    m = m.to(cuda).eval()
    pool = PagePool(2, 20, 4, 16, device=cuda)
    cache = m.new_cache(pool)
    x = torch.randn(2, 20, 256, generator=torch.Generator().manual_seed(2))
    want = oc.forward(params, x, cfg)
    plan = pool.plan(ints([18, 20], cuda), width=20, from_empty=True)
    out = m.prefill(x.to(cuda), cache, plan)
    top = want.abs().max()
    assert (out[1].cpu() - want[1]).abs().max() / top < 1e-5  # the layer's own tolerance in fp32
    for s in (18, 19):
        plan = pool.plan(ints([1, 1], cuda))
        assert plan.granted.tolist() == [True, False]
        out = m.decode(x[:, s].to(cuda), cache, plan)
        assert (out[0].cpu() - want[0, s]).abs().max() / top < 1e-5 and not out[1].any()
    assert not pool.plan(ints([1, 1], cuda)).granted.any()


@pytest.mark.parametrize("N,P", [(3, 1), (1, 4), (1, 1)])
def test_tables_of_one_row_or_column(cuda, N, P):
    """The stride of a dimension of one element says nothing."""
    from hydra_amd.attention import paged_attention, plan_pages, release_pages

    g = torch.Generator().manual_seed(1)
    kp, vp = (torch.randn(8, 1, 16, 16, generator=g).to(cuda) for _ in range(2))
    q = torch.randn(N, 2, 16, generator=g).to(cuda)
    outs = []
    for table in (ints([[-1] * P] * N, cuda), ints([[-1] * N] * P, cuda).t(),
                  torch.empty_strided((N, P), (1, 5) if P == 1 else (0, 1), dtype=torch.int32, device=cuda).fill_(-1)):
        stack, height, lengths = ints(range(8), cuda), ints([8], cuda), ints([0] * N, cuda)
        plan = plan_pages(lengths, ints([P * 16 - 3] * N, cuda), table, stack, height, 16, width=P * 16)
        out = paged_attention(q, kp, vp, table, plan.seen)
        assert plan.granted.all()
        held = table.clone()
        after, count = plan.lengths.clone(), plan.free_count.clone()
        release_pages(torch.ones(N, dtype=torch.bool, device=cuda), after, table, stack, count, 16)
        assert table.eq(-1).all() and count.tolist() == [8] and not after.any()
        outs.append((out, plan.slots, held, stack))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))
