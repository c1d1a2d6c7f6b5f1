"""GPU tests of the page plans, their release and the page store: whole
numbers and copies, equal to the oracle's."""
from __future__ import annotations

import random

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu


def ints(v, cuda):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def make(rng, N, P, page, width, spare, wrong=False):
    """A pool in use: lengths, new tokens, a table of distinct pages (-1 behind
    them) and a stack."""
    lengths = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, P * page)]) for _ in range(N)]
    lengths = [min(n, P * page) for n in lengths]
    new = [rng.choice([0, 1, width, rng.randint(0, width)]) for _ in range(N)]
    ids = list(range(sum(-(-n // page) for n in lengths) + spare))
    rng.shuffle(ids)
    table = []
    for n in lengths:
        c = -(-n // page)
        table.append([ids.pop() for _ in range(c)] + [-1] * (P - c))
    if wrong:
        for i in range(N):
            if rng.random() < 0.2:
                lengths[i] = rng.choice([-1, -2**31, P * page + 1, 2**31 - 1])
            if rng.random() < 0.2:
                new[i] = rng.choice([-1, width + 1, 2**31 - 1])
    return lengths, new, table, ids + [rng.randrange(99) for _ in range(rng.randint(0, 3))], len(ids)


def check(plan, table, want, cuda):
    slots, after, seen, granted, left, rows = want
    assert plan.slots.tolist() == slots
    assert plan.lengths.tolist() == after
    assert plan.seen.tolist() == seen
    assert plan.granted.tolist() == granted
    assert plan.free_count.tolist() == [left]
    assert table.tolist() == rows


@pytest.mark.parametrize("N,P,page,width", [
    (1, 1, 16, 1), (1, 3, 16, 40), (7, 5, 32, 1), (255, 4, 16, 3), (256, 4, 16, 1), (257, 4, 16, 1), (1000, 8, 64, 1),
    (300, 6, 16, 40), (3, 700, 16, 9000), (2, 3, 4096, 5000), (65, 9, 128, 64),
])
@pytest.mark.parametrize("from_empty", [False, True])
def test_plan_matches_oracle(cuda, N, P, page, width, from_empty):
    from hydra_amd.attention import plan_pages

    rng = random.Random(N * 131 + P * 7 + width)
    for spare in (0, 1, N // 2 + 1, N * (width // page + 2)):
        for wrong in (False, True):
            lengths, new, table, stack, free = make(rng, N, P, page, width, spare, wrong)
            t, ln, nw = ints(table, cuda), ints(lengths, cuda), ints(new, cuda)
            fp, fc = ints(stack, cuda), ints([free], cuda)
            want = op.plan(lengths, new, table, stack, free, page, width, from_empty)
            for _ in range(2):  # the inputs stay: a second call says the same
                plan = plan_pages(ln, nw, t, fp, fc, page, width=width, from_empty=from_empty)
                check(plan, t, want, cuda)
                assert plan.positions.tolist() == lengths
                assert ln.tolist() == lengths and fc.tolist() == [free]


@pytest.mark.parametrize("free", [-5, 0, 3, 1000])
def test_plan_with_a_wrong_stack_height(cuda, free):
    """A count outside the stack is taken as its nearest end."""
    from hydra_amd.attention import plan_pages

    stack = [5, 3, 8]
    t = ints([[-1, -1], [-1, -1]], cuda)
    plan = plan_pages(ints([0, 0], cuda), ints([20, 16], cuda), t, ints(stack, cuda), ints([free], cuda), 16, width=20)
    check(plan, t, op.plan([0, 0], [20, 16], [[-1, -1]] * 2, stack, free, 16, 20), cuda)


def test_plan_of_a_strided_table_and_an_entry_that_is_no_page(cuda):
    from hydra_amd.attention import plan_pages

    wide = ints([[4, -1, 77, 77], [-9, -1, 77, 77]], cuda)
    plan = plan_pages(ints([3, 3], cuda), ints([2, 2], cuda), wide[:, :2], ints([], cuda), ints([0], cuda), 16, width=3)
    assert plan.slots.tolist() == [[67, 68, -1], [-1, -1, -1]]
    assert wide.tolist() == [[4, -1, 77, 77], [-9, -1, 77, 77]]


@pytest.mark.parametrize("N", [1, 5, 256, 700])
def test_pool_over_many_steps(cuda, N):
    """Plans taken and pages released, step after step, against the oracle; no
    page is ever held twice."""
    from hydra_amd.attention import PagePool

    rng = random.Random(N)
    page, P = 16, 5
    pages = N * 3 + 1
    pool = PagePool(N, P * page, pages, page)
    lengths, table = [0] * N, [[-1] * P for _ in range(N)]
    stack, free = list(range(pages - 1, -1, -1)), pages
    for step in range(12):
        width = rng.choice([1, 1, 30])
        new = [rng.choice([0, 1, width, rng.randint(0, width)]) for _ in range(N)]
        before = list(lengths)
        plan = pool.plan(ints(new, cuda), width=width)
        slots, lengths, seen, granted, free, table = op.plan(lengths, new, table, stack, free, page, width)
        check(plan, pool.table, (slots, lengths, seen, granted, free, table), cuda)
        assert plan.positions.tolist() == before and pool.lengths.tolist() == lengths
        done = [rng.random() < 0.2 for _ in range(N)]
        pool.release(torch.tensor(done, device=cuda))
        lengths, table, stack, free = op.release(done, lengths, table, stack, free, page)
        assert pool.lengths.tolist() == lengths and pool.table.tolist() == table
        assert pool.free_pages.tolist()[:free] == stack[:free] and pool.free_count.tolist() == [free]
        held = [p for i, n in enumerate(lengths) for p in table[i][:-(-n // page)]] + stack[:free]
        assert sorted(held) == list(range(pages))


def test_pool_step_captured(cuda):
    """A captured plan moves the pool on at every replay."""
    from hydra_amd.attention import PagePool

    for N in (6, 300):  # planned in place, and by several workgroups
        pool, eager = (PagePool(N, 64, 4 * N, 16) for _ in range(2))
        new = torch.ones(N, dtype=torch.int32, device=cuda)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            pool.plan(torch.zeros_like(new))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan = pool.plan(new)
        for step in range(70):  # past the end of the rows: refused
            graph.replay()
            want = eager.plan(new)
            assert torch.equal(plan.slots, want.slots) and torch.equal(pool.lengths, eager.lengths), step
            assert torch.equal(plan.seen, want.seen) and torch.equal(pool.table, eager.table)
            assert torch.equal(plan.granted, want.granted)
        assert pool.lengths.tolist() == [64] * N and not plan.granted.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,K,S,hd,page", [(1, 1, 1, 16, 16), (2, 4, 37, 16, 16), (3, 2, 130, 64, 64),
                                           (2, 1, 33, 20, 32), (1, 3, 50, 1, 16), (2, 2, 17, 256, 16)])
def test_store(cuda, dtype, N, K, S, hd, page):
    from hydra_amd.attention import store_pages

    g = torch.Generator().manual_seed(S * hd + K)
    pages = -(-N * S // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:N * S].view(N, S)
    slots[torch.rand(N, S, generator=g) < 0.3] = -1
    slots[0, 0] = pages * page  # outside the pool: nowhere
    slots[-1, -1] = -2**62
    forms = {
        "plain": lambda t: t,
        "tokens first": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
        "turned": lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
        "unaligned": lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape),
    }
    for name, form in forms.items():
        k, v = (torch.randn(N, K, S, hd, generator=g).to(dtype) for _ in range(2))
        kp, vp = (torch.randn(pages, K, page, hd, generator=g).to(dtype) for _ in range(2))
        got = [form(t.to(cuda)) if name != "turned" else t.to(cuda) for t in (kp, vp)]
        store_pages(form(k.to(cuda)), form(v.to(cuda)), *got, slots.to(cuda))
        for n in range(N):
            for s in range(S):
                slot = int(slots[n, s])
                if 0 <= slot < pages * page:
                    kp[slot // page, :, slot % page] = k[n, :, s]
                    vp[slot // page, :, slot % page] = v[n, :, s]
        assert torch.equal(got[0].cpu(), kp) and torch.equal(got[1].cpu(), vp), name


def test_store_by_rows(cuda):
    """Prompts that belong to some of the requests, in any order; rows outside
    the slots store nothing."""
    from hydra_amd.attention import store_pages

    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(160, generator=g)[:70].view(7, 10)
    k, v = (torch.randn(5, 2, 10, 8, generator=g) for _ in range(2))
    kp, vp = (torch.zeros(10, 2, 16, 8) for _ in range(2))
    got = kp.to(cuda), vp.to(cuda)
    rows = [6, -1, 2, 7, 0]
    store_pages(k.to(cuda), v.to(cuda), *got, slots.to(cuda), rows=torch.tensor(rows, device=cuda))
    for n, r in enumerate(rows):
        for s in range(10 if 0 <= r < 7 else 0):
            slot = int(slots[r, s])
            kp[slot // 16, :, slot % 16] = k[n, :, s]
            vp[slot // 16, :, slot % 16] = v[n, :, s]
    assert torch.equal(got[0].cpu(), kp) and torch.equal(got[1].cpu(), vp)
    for bad in (torch.zeros(4, dtype=torch.long, device=cuda), torch.zeros(5, dtype=torch.int32, device=cuda)):
        with pytest.raises(ValueError, match="rows"):
            store_pages(k.to(cuda), v.to(cuda), *got, slots.to(cuda), rows=bad)


def test_store_past_32_bits(cuda):
    """The last page of a pool of more than 2^32 bytes and 2^31 elements."""
    from hydra_amd.attention import store_pages

    page, K, hd = 4096, 8, 128
    pages = (1 << 32) // (page * K * hd * 2) + 8
    kp, vp = (torch.zeros(pages, K, page, hd, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    assert kp.numel() > 2**31
    k, v = (torch.randn(1, K, 3, hd, generator=torch.Generator().manual_seed(i)).to(cuda, torch.bfloat16) for i in (1, 2))
    last = pages * page - 1
    store_pages(k, v, kp, vp, torch.tensor([[last, last + 1, last - page]], device=cuda))
    for pool, x in ((kp, k), (vp, v)):
        assert torch.equal(pool[-1, :, -1], x[0, :, 0]) and torch.equal(pool[-2, :, -1], x[0, :, 2])
        assert not pool[:-2].any() and not pool[-2:, :, :-1].any()


def test_refusals(cuda):
    from hydra_amd.attention import plan_pages, release_pages, store_pages

    z = ints([0, 0], cuda)
    t = ints([[0, 1], [2, 3]], cuda)
    for args, text in (((z, z[:1], t, z, z[:1], 16), "new_tokens"), ((z.long(), z, t, z, z[:1], 16), "lengths"),
                       ((z, z, t.long(), z, z[:1], 16), "table"), ((z, z, t[:1], z, z[:1], 16), "table"),
                       ((z, z, t.t(), z, z[:1], 16), "table"), ((z, z, t[:1].expand(2, 2), z, z[:1], 16), "overlap"),
                       ((z, z, t, z, z, 16), "free_count"), ((z, z, t, z, z[:1], 24), "power of two"),
                       ((z, z, t, z, z[:1], 16, 0), "width"), ((z, z, t[:, :0], z, z[:1], 16), "pages each")):
        with pytest.raises(ValueError, match=text):
            plan_pages(*args)
    two = torch.zeros(4, dtype=torch.int32, device=cuda)[::2]
    with pytest.raises(ValueError, match="contiguous"):
        release_pages(z.bool(), two, t, z, z[:1], 16)
    with pytest.raises(ValueError, match="done"):
        release_pages(z, z, t, z, z[:1], 16)
    kv = torch.zeros(4, 2, 16, 8, device=cuda)
    rows, slots = torch.zeros(1, 2, 3, 8, device=cuda), torch.zeros(1, 3, dtype=torch.long, device=cuda)
    for args, text in (((rows, rows, kv, kv.half(), slots), "alike"), ((rows, rows[:, :, :2], kv, kv, slots), "must be"),
                       ((rows.half(), rows.half(), kv, kv, slots), "share a dtype"),
                       ((rows, rows, kv, kv, slots.int()), "slots"), ((rows, rows, kv, kv, slots[:, :2]), "slots"),
                       ((rows, rows, kv[:1].expand(4, 2, 16, 8), kv, slots), "overlap"),
                       ((rows, rows, kv[:0], kv[:0], slots), "empty pool"),
                       ((rows[..., :6], rows[..., :6], kv[:, :, :12].transpose(2, 3)[..., :6],
                         kv[:, :, :12].transpose(2, 3)[..., :6], slots), "must be|unit stride")):
        with pytest.raises(ValueError, match=text):
            store_pages(*args)
    for i in range(4):
        args = [rows, rows, kv, kv]
        args[i] = args[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            store_pages(*args, slots)
