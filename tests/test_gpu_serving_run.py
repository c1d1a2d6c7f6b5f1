"""A server's loop: prompts of unequal length through embedding, two blocks,
norm and LM head into a paged cache, then tokens chosen greedily and returned
with their log probabilities, entropy and alternatives; requests end and
others take their place.  Each step against the oracle's forward of the whole
sequence."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import blocks as ob
from oracle import ccgqa as oc
from oracle import logprobs as ol

pytestmark = pytest.mark.gpu

DIM, VOCAB, TOP = 256, 1003, 5


def test_greedy_generation(cuda):
    from hydra_amd.attention import PagePool
    from hydra_amd.kernels import token_logprobs
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
        h = ob.embedding(table, torch.tensor([ids]), math.sqrt(DIM))
        for ref in refs:
            h = ob.hydra_block(ref, h, cfg)
        return F.linear(ob.rms_norm(h, torch.ones(DIM)), table)[0, -1:]

    def answer(h):
        logits = F.linear(norm(h), emb)
        best = logits.argmax(-1)
        return best, token_logprobs(logits, best, top_k=TOP)

    def compare(ids, n, out):
        logits = oracle(ids)
        want = ol.forward(logits, out.top_tokens[n, :1].cpu(), TOP)
        # the logits are those of two fp32 evaluations: 1e-5 of the largest each
        tol = 4e-5 * float(logits.abs().max()) + 1e-5
        assert abs(float(out.logprobs[n].detach()) - float(want[0][0])) < tol
        assert abs(float(out.entropy[n].detach()) - float(want[1][0])) < tol * math.log(VOCAB)
        assert (out.top_logprobs[n].cpu().double() - want[2][0]).abs().max() < tol
        assert float(out.logprobs[n].detach()) == float(out.top_logprobs[n, 0].detach())

    g = torch.Generator().manual_seed(4)
    N = 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    pool = PagePool(N, 64, 8, 16, device=cuda)
    caches = [b.new_cache(pool) for b in blocks]
    texts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (20, 1, 33)]

    def prefill(rows):
        width = max(len(texts[n]) for n in rows)
        ids = torch.zeros(len(rows), width, dtype=torch.long)
        for m, n in enumerate(rows):
            ids[m, :len(texts[n])] = torch.tensor(texts[n])
        new = [len(texts[n]) if n in rows else 0 for n in range(N)]
        plan = pool.plan(i32(new), width=width, from_empty=True)
        assert plan.granted.all()
        h = embedding_lookup(emb, ids.to(cuda), math.sqrt(DIM))
        for b, c in zip(blocks, caches):
            h = b.prefill(h, c, plan, rows=torch.tensor(rows, device=cuda))
        last = torch.stack([h[m, len(texts[n]) - 1] for m, n in enumerate(rows)])
        best, out = answer(last)
        for m, n in enumerate(rows):
            compare(texts[n], m, out)
            texts[n].append(int(best[m]))

    prefill([0, 1, 2])
    for step in range(14):
        if step == 6:  # one request is done; a new one takes its row and pages
            pool.release(torch.tensor([False, False, True], device=cuda))
            texts[2] = torch.randint(0, VOCAB, (40,), generator=g).tolist()
            prefill([2])
        plan = pool.plan(i32([1] * N))
        assert plan.granted.all()
        h = embedding_lookup(emb, torch.tensor([t[-1] for t in texts], device=cuda), math.sqrt(DIM))
        for b, c in zip(blocks, caches):
            h = b.decode(h, c, plan)
        best, out = answer(h)
        for n in range(N):
            compare(texts[n], n, out)
            texts[n].append(int(best[n]))
    held = sum(-(-(len(t) - 1) // 16) for t in texts)
    assert pool.lengths.tolist() == [len(t) - 1 for t in texts] and pool.free_count.tolist() == [8 - held]


_CAPTURE_FIRST = """
import sys
import torch
sys.path.insert(0, sys.argv[1])
from hydra_amd.attention import paged_attention, plan_pages, store_pages
from hydra_amd.attention.backends.ccgqa.ops import CCGQA_CONVS, CCGQA_QK_MEAN, ccgqa_decode_prep
from hydra_amd.kernels import token_logprobs
g = torch.Generator().manual_seed(3)
rand = lambda *s: (torch.randn(*s, generator=g) / 8).to(torch.bfloat16).cuda()
i32 = lambda *s: torch.zeros(*s, dtype=torch.int32).cuda()
N, H, K, hd, page, P = 3, 16, 4, 64, 16, 300
L, KD = H * hd, K * hd
lengths, fresh, table = i32(N), i32(N) + 1, i32(N, P) - 1
stack, count = torch.arange(N * P, dtype=torch.int32).cuda(), i32(1) + N * P
kp, vp, ring, qkv = rand(N * P, K, page, hd), rand(N * P, K, page, hd), rand(N, 5, L + 2 * KD), rand(N, L + 2 * KD)
w = [rand(3, L, hd), rand(3, L, L), rand(3, KD, hd), rand(3, KD, KD)]
k, x, tokens = rand(1, K, 1, hd), rand(N, 5000), torch.zeros(N, dtype=torch.long).cuda()
slot = torch.full((1, 1), 16 * N * P - 1).cuda()

def step():
    plan = plan_pages(lengths, fresh, table, stack, count, page)
    store_pages(k, k, kp, vp, slot)
    q = ccgqa_decode_prep(qkv, ring, plan.positions, plan.slots, kp, vp, H, K, hd, CCGQA_CONVS | CCGQA_QK_MEAN, *w,
                          packed=True)
    return (plan.slots, q, paged_attention(q, kp, vp, table, plan.seen), *token_logprobs(x, tokens, top_k=3))

torch.cuda.synchronize()
graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side), torch.cuda.graph(graph):  # the process's first calls
    got = step()
torch.cuda.current_stream().wait_stream(side)
want = step()
for _ in range(3):
    for t in got:
        t.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    step()
print("capture-first ok")
"""


def test_step_captured_as_first_call(cuda):
    """A process whose first calls are inside a capture, in the forms with
    workspaces (split attention, shared heads' convs)."""
    import subprocess
    import sys
    from pathlib import Path

    root = str(Path(__file__).resolve().parents[1])
    res = subprocess.run([sys.executable, "-c", _CAPTURE_FIRST, root], capture_output=True, text=True, timeout=110)
    assert res.returncode == 0 and "capture-first ok" in res.stdout, res.stdout[-2000:] + res.stderr[-2000:]
