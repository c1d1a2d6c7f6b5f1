"""GPU tests of the serving operators at their edges: values that are no
numbers behind vanishing weights, derivatives that no kernel gives, launches
beyond one grid, idle rows of blocks."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("length,columns", [(400, 25), (9000, 600)])  # one workgroup, and split
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_values_behind_vanishing_weights(cuda, dtype, length, columns, bad):
    """A value that is seen is in the sum however small its weight is: 0 x NaN
    and 0 x inf are NaN, whichever part of a split context they lie in."""
    from hydra_amd.attention import paged_attention

    page, hd = 16, 32
    pages = -(-length // page)
    kp, vp = torch.zeros(pages, 1, page, hd), torch.ones(pages, 1, page, hd)
    kp[..., 0] = -40.0
    kp[0, 0, :, 0] = 40.0  # scores 400 apart: the weights of all but the first 16 keys vanish in fp32
    vp[(length - 5) // page, 0, (length - 5) % page, 3] = bad
    q = torch.zeros(1, 2, hd)
    q[..., 0] = 5.0
    table = torch.full((1, columns), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages, dtype=torch.int32)
    got = paged_attention(q.to(cuda, dtype), kp.to(cuda, dtype), vp.to(cuda, dtype), table.to(cuda),
                          torch.tensor([length], dtype=torch.int32, device=cuda), scale=1.0).cpu()
    rest = [c for c in range(hd) if c != 3]
    assert not got[..., 3].isfinite().any()
    assert (got[..., rest] == 1).all()


class Step(torch.nn.Module):
    def __init__(self, layer):
        super().__init__()
        self.layer = layer

    def forward(self, *args):
        return self.layer.decode(*args)


def test_derivatives_that_nothing_gives_are_refused(cuda):
    """A recorded gradient of a weight or of `out`, and forward-mode tangents
    of anything, are an error and not lost."""
    import torch.autograd.forward_ad as fwad

    from hydra_amd.attention import CCGQAAttention, PagePool, paged_attention, store_pages
    from hydra_amd.attention.backends.ccgqa.ops import CCGQA_CONVS, CCGQA_QK_NORM, ccgqa_decode_prep, ccgqa_ring_fill
    from hydra_amd.kernels import token_logprobs

    new = lambda *s: torch.ones(*s, device=cuda)  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    kp, vp, q, table = new(4, 1, 16, 16), new(4, 1, 16, 16), new(1, 2, 16), i32(0, 1, 2)[None]
    ring, row, slot = new(1, 5, 64), new(1, 64), torch.zeros(1, 1, dtype=torch.long, device=cuda)
    w = [new(3, 32, 16), new(3, 32, 32), new(3, 16, 16), new(3, 16, 16)]
    tokens = torch.zeros(3, dtype=torch.long, device=cuda)

    def prep(row=row, ring=ring, w=w, temperature=new(1)):
        return ccgqa_decode_prep(row, ring, i32(5), slot, kp, vp, 2, 1, 16, CCGQA_CONVS | CCGQA_QK_NORM, *w,
                                 temperature=temperature, packed=True)

    prep()
    for i in range(4):
        recorded = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(w)]
        with pytest.raises(RuntimeError, match="no gradient"):
            prep(w=recorded)
        with torch.no_grad():
            prep(w=recorded)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention(q, kp, vp, table, i32(40), out=q.clone().requires_grad_())

    torch.manual_seed(0)
    m = CCGQAAttention(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=32).to(cuda).eval()
    pool = PagePool(2, 32, 4, 16, device=cuda)
    cache = m.new_cache(pool)
    plans = pool.plan(i32(4, 4), width=4, from_empty=True), pool.plan(i32(1, 1))
    x = new(2, 4, 256)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: token_logprobs(dual(new(3, 8)), tokens), lambda: token_logprobs(dual(new(3, 8).requires_grad_()), tokens),
                 lambda: prep(row=dual(row)), lambda: prep(ring=dual(ring)), lambda: prep(w=[dual(t) for t in w]),
                 lambda: prep(temperature=dual(new(1))), lambda: paged_attention(dual(q), kp, vp, table, i32(40)),
                 lambda: paged_attention(q, kp, dual(vp), table, i32(40)),
                 lambda: store_pages(dual(new(1, 1, 1, 16)), new(1, 1, 1, 16), kp, vp, slot),
                 lambda: ccgqa_ring_fill(dual(new(1, 4, 64)), ring, i32(4), 4),
                 lambda: m.prefill(dual(x), cache, plans[0]), lambda: m.decode(dual(x[:, 0]), cache, plans[1])]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        logits = new(3, 8).requires_grad_()
        out = token_logprobs(logits, tokens)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out.logprobs, logits, dual(new(3)))
        token_logprobs(new(3, 8), tokens), prep(), m.prefill(x, cache, plans[0])  # no tangents: as ever
        step = Step(m)
        params = {k: v.detach() for k, v in step.named_parameters()}
        torch.func.functional_call(step, params, (x[:, 0], cache, plans[1]))
        for name in ("q_conv.conv1.weight", "key_temperature", "o_proj.weight"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.func.functional_call(step, {**params, f"layer.{name}": dual(params[f"layer.{name}"])},
                                           (x[:, 0], cache, plans[1]))


@pytest.mark.parametrize("rows", [(1 << 22) + 1, (1 << 23) + 3])
def test_log_probabilities_of_more_rows_than_a_grid(cuda, rows):
    """HIP counts a launch's threads in 32 bits; rows past them are worked on
    like the first ones."""
    from hydra_amd.kernels import token_logprobs

    V, K = 12, 2
    x = torch.randn(rows, V, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(torch.bfloat16)
    tokens = torch.arange(rows, device=cuda) % V

    def step(x, tokens):
        x = x.clone().requires_grad_()
        out = token_logprobs(x, tokens, top_k=K)
        grad, = torch.autograd.grad([out.logprobs.sum() + 0.5 * out.entropy.sum() + out.top_logprobs.sum()], [x])
        return (*(t.detach() for t in out), grad)

    whole = step(x, tokens)
    for begin in range(0, rows, 1 << 20):
        part = slice(begin, begin + (1 << 20))
        for a, b in zip(whole, step(x[part], tokens[part])):
            assert torch.equal(a[part], b), begin
    assert torch.equal(token_logprobs(x, tokens).logprobs, whole[0])


def test_attention_of_more_items_than_a_grid(cuda):
    """Requests times key heads past what one launch's threads count."""
    from hydra_amd.attention import paged_attention

    N, K, hd, pages = (1 << 23) + 5, 2, 8, 64
    g = torch.Generator(device=cuda).manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device=cuda).to(torch.bfloat16)  # noqa: E731
    q, kp, vp = rand(N, K, hd), rand(pages, K, 16, hd), rand(pages, K, 16, hd)
    table = torch.randint(pages, (N, 1), generator=g, device=cuda, dtype=torch.int32)
    lengths = torch.randint(17, (N,), generator=g, device=cuda, dtype=torch.int32)
    whole = paged_attention(q, kp, vp, table, lengths, out=torch.full_like(q, 9.0))
    for begin in range(0, N, 1 << 20):
        part = slice(begin, begin + (1 << 20))
        assert torch.equal(whole[part], paged_attention(q[part], kp, vp, table[part], lengths[part])), begin


def test_blocks_with_idle_and_refused_requests(cuda):
    """Blocks over one pool, one request idle at every step and one refused in
    the end: the others' rows are those of blocks that serve them alone, an idle
    request's caches stay, and its own row is what the block makes of an
    attention of zeros: no result."""
    from hydra_amd.attention import PagePool
    from hydra_amd.model.framework import HydraBlock

    torch.manual_seed(0)
    dim, N, S = 256, 3, 12
    blocks = [HydraBlock(dim, n_heads=4, n_kv_heads=2, max_seq_len=64).to(cuda).eval() for _ in range(2)]
    x = torch.randn(N, 40, dim, generator=torch.Generator().manual_seed(1)).to(cuda)
    lens = [12, 5, 9]

    def serve(idle):
        """Rows [step][n]; request `idle(step)` has no token then."""
        pool = PagePool(N, 16, 3, 16, device=cuda)
        caches = [b.new_cache(pool) for b in blocks]
        h = x[:, :S]
        plan = pool.plan(torch.tensor(lens, dtype=torch.int32, device=cuda), width=S, from_empty=True)
        for b, c in zip(blocks, caches):
            h = b.prefill(h, c, plan)
        rows, at = [], list(lens)
        for step in range(6):
            who = idle(step)
            new = torch.tensor([int(n != who) for n in range(N)], dtype=torch.int32, device=cuda)
            before = [(c.ring[who].clone(), c.k_pages.clone()) for c in caches] if who is not None else None
            plan = pool.plan(new)
            h = token = torch.stack([x[n, at[n]] for n in range(N)])
            for b, c in zip(blocks, caches):
                h = b.decode(h, c, plan)
            rows.append(h)
            at = pool.lengths.tolist()
            if who is not None:
                page = int(pool.table[who, 0])
                for c, (ring, kp) in zip(caches, before):
                    assert torch.equal(c.ring[who], ring) and torch.equal(c.k_pages[page], kp[page])
                alone = token[who:who + 1]
                for b in blocks:
                    with torch.no_grad():
                        alone = b._rest(alone, torch.zeros_like(alone))
                assert plan.seen[who] == 0 and alone.any()
                assert (h[who] - alone[0]).abs().max() <= 1e-5 * alone.abs().max()
        return rows, plan

    whole, plan = serve(lambda step: None)
    assert plan.granted.tolist() == [False, True, True]  # 12 + 4 tokens fill the page: the last two are refused
    turns, _ = serve(lambda step: 1)
    for step in range(6):
        for n in (0, 2):
            assert torch.equal(turns[step][n], whole[step][n]), (step, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,head_dim,taps", [(1, 1, 2, 4), (1, 1, 2, 3), (2, 1, 2, 1), (1, 1, 14, 3),
                                                          (7, 7, 2, 2), (3, 1, 4, 5), (1, 1, 16, 3)])
def test_layers_of_few_channels(cuda, dtype, heads, kv_heads, head_dim, taps):
    """Fewer channels than a block of the matrix form (16): one token against
    the oracle's whole sequence."""
    import test_gpu_ccgqa_decode as td

    from oracle import ccgqa as oc

    cfg = oc.CCGQAConfig(dim=4 * heads * head_dim, n_heads=heads, n_kv_heads=kv_heads, conv_kernel_size=taps)
    positions = [0, 3, 9, 1]
    slots = [5, 17, 40, 33]
    params, rows, ring = td.case(cfg, positions, dtype, seed=heads * head_dim + taps)
    got = td.run(cuda, cfg, dtype, params, rows, ring, positions, slots, 3, 16)
    td.check(cfg, dtype, params, rows, ring, positions, slots, 16, got)
