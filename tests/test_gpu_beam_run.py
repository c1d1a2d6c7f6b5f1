"""Beam search over blocks: prompts prefilled once, requests forked from them
with their pages in common, tokens decoded over the shared prefixes, the best
continuations selected and everything taken along; each step against the
oracle's forward of the whole sequences.  The same in caches of 8 bits against
what those hold, and a step captured and replayed."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import blocks as ob
from oracle import ccgqa as oc
from oracle import paged as op

pytestmark = pytest.mark.gpu

DIM, VOCAB = 256, 301


def test_beam_search(cuda):
    from hydra_amd.attention import PagePool, take_rows
    from hydra_amd.kernels import beam_select
    from hydra_amd.layers import RMSNorm
    from hydra_amd.model.framework import HydraBlock, embedding_lookup

    torch.manual_seed(3)
    cfg = oc.CCGQAConfig(dim=DIM, n_heads=4, n_kv_heads=2, max_seq_len=128)
    blocks = [HydraBlock(DIM, n_heads=4, n_kv_heads=2, max_seq_len=128) for _ in range(2)]
    refs = [{k: v.detach().clone() for k, v in b.state_dict().items()} for b in blocks]
    table = torch.randn(VOCAB, DIM) * 0.05
    blocks = [b.to(cuda).eval() for b in blocks]
    norm, emb = RMSNorm(DIM).to(cuda), table.to(cuda)

    def oracle(ids):
        h = ob.embedding(table, torch.tensor(ids), math.sqrt(DIM))
        for ref in refs:
            h = ob.hydra_block(ref, h, cfg)
        return F.linear(ob.rms_norm(h, torch.ones(DIM)), table)[:, -1]

    B, W, steps = 2, 3, 13
    N = B * W
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    g = torch.Generator().manual_seed(4)
    pool = PagePool(N, 64, 20, 16, device=cuda, sharing=True)
    caches = [b.new_cache(pool) for b in blocks]
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (20, 33)]

    with torch.no_grad():
        ids = torch.zeros(B, 33, dtype=torch.long)
        for b, p in enumerate(prompts):
            ids[b, :len(p)] = torch.tensor(p)
        plan = pool.plan(i32([20, 0, 0, 33, 0, 0]), width=33, from_empty=True)
        h = embedding_lookup(emb, ids.to(cuda), math.sqrt(DIM))
        for b, c in zip(blocks, caches):
            h = b.prefill(h, c, plan, rows=torch.tensor([0, W], device=cuda))
        logits = F.linear(norm(torch.stack([h[b, len(p) - 1] for b, p in enumerate(prompts)])), emb)
        logits = logits.repeat_interleave(W, 0)
        scores = torch.full((B, W), -math.inf, device=cuda)
        scores[:, 0] = 0
        shared, ones = i32([20, 33]), i32([1] * N)
        history = torch.zeros(N, steps, dtype=torch.long, device=cuda)
        texts, sums = [list(prompts[n // W]) for n in range(N)], [0.0] * N
        free = []
        for step in range(steps):
            best = beam_select(logits, scores, W)
            rows, tokens, scores = best.rows.view(-1), best.tokens.view(-1), best.scores
            fork = pool.fork(rows)
            assert fork.granted.all()
            for c in caches:
                c.fork(fork)
            take_rows(history, rows)
            history[:, step] = tokens
            plan = pool.plan(ones)
            assert plan.granted.all()
            h = embedding_lookup(emb, tokens, math.sqrt(DIM))
            for b, c in zip(blocks, caches):
                h = b.decode(h, c, plan, shared=shared)
            logits = F.linear(norm(h), emb)
            # the oracle's texts, and what their logits and sums of log probabilities are
            at, tok = rows.tolist(), tokens.tolist()
            logp = [torch.log_softmax(oracle([texts[n]])[0].double(), -1) for n in range(N)]
            sums = [sums[p] + float(logp[p][t]) for p, t in zip(at, tok)]
            texts = [texts[p] + [t] for p, t in zip(at, tok)]
            assert len({tuple(t) for t in texts}) == N
            assert [prompts[n // W] + history[n, :step + 1].tolist() for n in range(N)] == texts
            # two fp32 evaluations: 1e-5 of the largest logit each, in every step's log probability
            want = torch.cat([oracle([t]) for t in texts])
            tol = 4e-5 * float(want.abs().max()) + 1e-5
            assert (logits.cpu() - want).abs().max() < tol
            assert max(abs(a - b) for a, b in zip(scores.view(-1).tolist(), sums)) < tol * (step + 1)
            free.append(pool.free_count.item())
        # the prompts' full pages once, then each beam's own, at most
        assert min(free) >= 20 - (1 + 2) - N * 2
        pool.release(torch.tensor([True] * 3 + [False] * 3, device=cuda))
        assert pool.lengths.tolist() == [0] * 3 + [33 + steps] * 3
        pool.release(torch.ones(N, dtype=torch.bool, device=cuda))
        assert pool.free_count.item() == 20 and sorted(pool.free_pages.tolist()) == list(range(20))
        assert not pool.extra.any() and (pool.table == -1).all()


@pytest.mark.parametrize("eight", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_caches_of_eight_bits(cuda, eight, dtype):
    """A layer that decodes and forks in one: the rows that the full cache holds,
    quantised; the attention over what that stands for."""
    from hydra_amd.attention import CCGQAAttention, PagePool, paged_attention

    torch.manual_seed(1)
    layer = CCGQAAttention(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=128).to(cuda, dtype).eval()
    N, page = 5, 16
    pools = [PagePool(N, 96, 40, page, device=cuda, sharing=True) for _ in range(2)]
    caches = [layer.new_cache(pools[0]), layer.new_cache(pools[1], page_dtype=eight)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    x = torch.randn(2, 37, 256, device=cuda).to(dtype)
    outs = []
    for pool, cache in zip(pools, caches):
        plan = pool.plan(i32([37, 21, 0, 0, 0]), width=37, from_empty=True)
        outs.append(layer.prefill(x, cache, plan, rows=torch.tensor([0, 1], device=cuda)))
        cache.fork(pool.fork(i32([0, 1, 0, 1, -1])))
    assert torch.equal(*outs)  # prompts are answered from their own rows
    for step in range(20):
        new = i32([1, 1, 1, 1 if step % 3 else 0, 0])  # one request idles at times, one for good
        x = torch.randn(N, 256, device=cuda).to(dtype)
        for pool, cache in zip(pools, caches):
            plan = pool.plan(new)
            outs[pools.index(pool)] = layer.decode(x, cache, plan)
        full, small = caches
        assert torch.equal(pools[0].table, pools[1].table) and torch.equal(full.ring, small.ring)
        for n in range(N):
            L = int(pools[0].lengths[n])
            for t in range(L) if step in (0, 19) else range(max(L - 1, 0), L):
                p = int(pools[0].table[n, t // page])
                for a, b, s in zip((full.k_pages, full.v_pages), (small.k_pages, small.v_pages), small.scales):
                    q, scales = op.quantise(a[p, :, t % page].cpu(), eight)
                    assert torch.equal(b.view(torch.int8)[p, :, t % page].cpu(),
                                       (q.to(eight) if eight == torch.int8 else q.float().to(eight)).view(torch.int8))
                    assert torch.equal(s[p, :, t % page].cpu(), scales)
        wide = [(p.float() * s[..., None]) for p, s in zip((small.k_pages, small.v_pages), small.scales)]
        # the same attention of fp32 pages: q is within outs' rounding, so go through a probe of the layer's own
        probe = torch.randn(N, 4, 16, device=cuda).to(dtype)
        got = paged_attention(probe, small.k_pages, small.v_pages, small.table, plan.seen, scales=small.scales)
        want, weight = op.attention(probe.cpu(), wide[0].cpu(), wide[1].cpu(), small.table.cpu(), plan.seen.cpu())
        bound = op.attention_bound(probe.cpu(), wide[0].cpu(), weight, want, plan.seen.cpu(), dtype) + \
            op.two_term_bound(weight, wide[1].cpu(), plan.seen.cpu(), eight, dtype)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
        assert not outs[1][plan.seen == 0].any()
        if step % 5 == 4:
            for pool, cache in zip(pools, caches):
                cache.fork(pool.fork(i32([[2, 1, 0, 0, -1], [1, 1, 2, 3, -1]][step % 2])))


def test_shared_prefix_of_a_layer(cuda):
    """decode with and without `shared`: two orders of the same sums."""
    from hydra_amd.attention import CCGQAAttention, PagePool

    torch.manual_seed(2)
    layer = CCGQAAttention(dim=512, n_heads=8, n_kv_heads=2, max_seq_len=512).to(cuda).eval()
    pool = PagePool(8, 400, 100, 16, device=cuda, sharing=True)
    cache = layer.new_cache(pool)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    plan = pool.plan(i32([300, 0, 0, 0, 123, 0, 0, 0]), width=300, from_empty=True)
    layer.prefill(torch.randn(2, 300, 512, device=cuda), cache, plan, rows=torch.tensor([0, 4], device=cuda))
    cache.fork(pool.fork(i32([0] * 4 + [4] * 4)))
    for _ in range(3):
        x = torch.randn(8, 512, device=cuda)
        plan = pool.plan(i32([1] * 8))
        ring = cache.ring.clone()
        a = layer.decode(x, cache, plan)
        cache.ring.copy_(ring)
        b = layer.decode(x, cache, plan, shared=i32([300, 123]))
        # both within 1e-5 of the largest output (the fp32 tolerance of the layer's forward)
        assert (a - b).abs().max() <= 2e-5 * a.abs().max()


def test_step_captured(cuda):
    """beam_select, fork_pages, copy_pages, take_rows, store_pages and both forms of the
    attention in one graph, replayed between eager runs of the same on other states."""
    from hydra_amd.attention import copy_pages, fork_pages, paged_attention, read_pages, store_pages, take_rows
    from hydra_amd.kernels import beam_select

    g = torch.Generator().manual_seed(3)
    B, W, K, H, hd, page, P = 3, 4, 2, 8, 64, 16, 150
    N, pages = B * W, 900
    rand = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda)  # noqa: E731

    def fresh(seed):
        r = torch.Generator().manual_seed(seed)
        lengths = torch.randint(1, 1000, (N,), generator=r)
        ids = iter(torch.randperm(pages, generator=r).tolist())
        table = [[next(ids) if c < -(-n // page) else -1 for c in range(P)] for n in lengths.tolist()]
        left = list(ids)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
        return [i32(lengths.tolist()), i32(table), i32(left + [0] * (pages - len(left))), i32([len(left)]),
                i32([0] * pages), torch.randn(N, 500, generator=r).to(cuda), torch.randn(B, W, generator=r).to(cuda),
                torch.randint(0, pages * page, (2, 30), generator=r).unique()[:30][None].to(cuda),
                torch.randint(1, 400, (B,), generator=r).to(torch.int32).to(cuda), torch.randn(N, 9, 20, generator=r).to(cuda)]

    q, k, v, k16, v16 = rand(N, H, hd), rand(1, K, 30, hd), rand(1, K, 30, hd), rand(pages, K, page, hd), rand(pages, K, page, hd)
    k8, v8 = (torch.randint(-100, 100, (pages, K, page, hd), generator=g, dtype=torch.int8).to(cuda) for _ in range(2))
    scales = [torch.rand(pages, K, page, generator=g).to(cuda) for _ in range(2)]
    keep = [t.clone() for t in (k8, v8, *scales, k16, v16)]
    state = fresh(0)

    def step():
        lengths, table, stack, count, extra, logits, scores, slots, shared, rows = state
        best = beam_select(logits, scores, W)
        fork = fork_pages(best.rows.view(-1), lengths, table, stack, count, extra, page)
        copy_pages(k8, v8, fork.sources, fork.copies, scales=scales)
        copy_pages(k16, v16, fork.sources, fork.copies)
        take_rows(rows, fork.parents)
        store_pages(k, v, k8, v8, slots, scales=scales)
        return [*best, *fork, *read_pages(k8, v8, slots, scales=scales, dtype=torch.float32),
                paged_attention(q, k8, v8, table, lengths, scales=scales),
                paged_attention(q, k16, v16, table, lengths, shared=shared),
                paged_attention(q, k8, v8, table, lengths, scales=scales, shared=shared)]

    def set_to(seed):
        for t, s in zip(state, fresh(seed)):
            t.copy_(s)
        for t, s in zip((k8, v8, *scales, k16, v16), keep):
            t.copy_(s)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(1, 5):
        set_to(seed)
        want = [t.clone() for t in step()]
        after = [t.clone() for t in state]
        set_to(seed)
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(state, after))
