"""The operators of a serving step and of what it answers with, measured over
the sizes, types and directions that are used in earnest.

A case is a dict of plain values; its "kind" names the operator:

  plan   page tables and slot maps from the lengths of the requests
  store  the keys and values of a batch of prompts into their pages
  prep   one token's q, k and v of a CCGQA layer from its projected row, the
         rows before it and the convs' weights, k and v into the pages
  attn   the attention of one new token per request over its pages
  logp   log probabilities of given tokens, with the entropy and the top
         alternatives of their rows; as a training step with the gradient

`listed()` holds the named cases, `draw(rng)` gives others of the same
ranges, `exact()` restates each operator in 64 bits.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
TAPS = 3               # of the CCGQA convs
BACK = 2 * (TAPS - 1)  # rows that two of them reach back

# (dim, n_heads, n_kv_heads) of attention layers at 4x compression
LAYERS = [(512, 8, 2), (1024, 4, 1), (1024, 16, 4), (2048, 8, 2), (1792, 28, 4), (768, 6, 2), (1024, 8, 8),
          (2048, 4, 1)]
# (heads, kv_heads, head_dim) of their attention
HEADS = [(8, 2, 16), (4, 1, 64), (16, 4, 16), (8, 2, 64), (28, 4, 16), (6, 2, 32), (8, 8, 32), (4, 1, 128)]


def listed():
    return [
        # one decoding step's slots for a small server
        dict(name="plan_step", kind="plan", N=32, width=1, page=64, limit=4096, fresh=False, scarce=False),
        # a large batch of prompts of any length admitted at once
        dict(name="plan_prompts", kind="plan", N=256, width=4096, page=16, limit=8192, fresh=True, scarce=False),
        # one ragged prompt of a layer with small heads goes into the cache
        dict(name="store_prompt", kind="store", dtype="bf16", N=1, width=1003, kv_heads=4, head_dim=16, page=16),
        # a batch of long prompts
        dict(name="store_batch", kind="store", dtype="bf16", N=16, width=4096, kv_heads=2, head_dim=64, page=64),
        # a single user's token through the 250M model's layer
        dict(name="prep_one", kind="prep", dtype="bf16", N=1, dim=1024, heads=4, kv_heads=1, page=64, limit=4096),
        # a full server's step through a wide layer
        dict(name="prep_batch", kind="prep", dtype="bf16", N=256, dim=2048, heads=8, kv_heads=2, page=64, limit=8192),
        # a single user's token with a short context: latency
        dict(name="attn_one", kind="attn", dtype="bf16", N=1, heads=4, kv_heads=1, head_dim=64, page=64, length=700,
             ragged=False),
        # a server's requests of all lengths, seven heads to a key head of 16
        dict(name="attn_ragged", kind="attn", dtype="fp16", N=48, heads=28, kv_heads=4, head_dim=16, page=16,
             length=8192, ragged=True),
        # many long contexts: the largest reads of a step
        dict(name="attn_long", kind="attn", dtype="bf16", N=64, heads=8, kv_heads=2, head_dim=64, page=64,
             length=16384, ragged=False),
        # a program that keeps everything in fp32, a key head for each head
        dict(name="attn_fp32", kind="attn", dtype="fp32", N=5, heads=8, kv_heads=8, head_dim=32, page=32, length=3001,
             ragged=True),
        # what a server returns with each sampled token
        dict(name="logp_step", kind="logp", dtype="bf16", rows=16, vocab=50257, top=20, train=False, temperature=1.0),
        # a policy's training step on the tokens it sampled
        dict(name="logp_train", kind="logp", dtype="bf16", rows=8192, vocab=32000, top=0, train=True, temperature=0.7),
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "store", "prep", "attn", "attn", "logp", "logp"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "plan":
        N, fresh = _log_int(rng, 1, 1024), rng.random() < 0.5
        width = _log_int(rng, 2, min(4096, 1048576 // N)) if fresh else rng.choice([1, 1, 1, 5])
        return dict(kind=kind, N=N, width=width, page=page, limit=8192, fresh=fresh, scarce=rng.random() < 0.3)
    if kind == "store":
        H, K, hd = rng.choice(HEADS)
        N = _log_int(rng, 1, 64)
        return dict(kind=kind, dtype=dtype, N=N, width=_log_int(rng, 1, 65536 * 128 // (N * K * hd * SIZE[dtype] // 2)),
                    kv_heads=K, head_dim=hd, page=page)
    if kind == "prep":
        dim, H, K = rng.choice(LAYERS)
        return dict(kind=kind, dtype=dtype, N=_log_int(rng, 1, 256 if dtype != "fp32" else 64), dim=dim, heads=H,
                    kv_heads=K, page=page, limit=_log_int(rng, 256, 8192))
    if kind == "attn":
        H, K, hd = rng.choice(HEADS)
        N = _log_int(rng, 1, 256)
        most = (1 << 28) // (N * K * hd * SIZE[dtype])  # half of the longest listed case's bytes
        return dict(kind=kind, dtype=dtype, N=N, heads=H, kv_heads=K, head_dim=hd, page=page,
                    length=_log_int(rng, 1, max(1, min(32768, most // 2))), ragged=rng.random() < 0.6)
    vocab = rng.choice([4099, 16000, 32000, 50257])
    train = rng.random() < 0.5
    top = rng.choice([0, 1, 5, 20])
    rows = _log_int(rng, 1, min(4096, (1 << 27) // vocab) if train and not top else 512)
    return dict(kind=kind, dtype=dtype, rows=rows, vocab=vocab, top=top, train=train,
                temperature=rng.choice([1.0, 0.7, 1.5]))


# ------------------------------------------------------------------ inputs
class _Random:
    """Inputs on the GPU from a seed alone; sizes of requests from the CPU's
    generator."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))
        self.c = torch.Generator().manual_seed(int(seed) + 1)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std).add_(mean).to(dtype)

    def ints(self, hi, *shape, lo=0):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda")

    def lengths(self, n, most, ragged):
        """Lengths of n requests: all `most`, or even over the logarithm up to
        it, in any order."""
        if not ragged:
            return torch.full((n,), most)
        out = torch.exp((torch.arange(n) + 0.5) / n * math.log(most)).round().long().clamp(1, most)
        out[-1] = most
        return out[self.order(n)]

    def order(self, n):
        return torch.randperm(n, generator=self.c)


def _table(r, lengths, page, columns):
    """A table [N, columns] of pages handed out in no order, -1 where a request
    has none; the number of pages in the pool; the pages not handed out."""
    counts = (lengths + page - 1) // page
    used = int(counts.sum())
    total = used + 3
    ids = r.order(total)
    table = torch.full((len(lengths), columns), -1)
    at = torch.arange(columns)[None] < counts[:, None]
    table[at] = ids[:used]
    return table.to(torch.int32).cuda(), total, ids[used:]


def _rope_tables(head_dim, length):
    freqs = 1.0 / (10000.0 ** (torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim))
    ang = torch.outer(torch.arange(length, dtype=torch.float32), freqs)
    return ang.cos().cuda(), ang.sin().cuda()


def prepare(case, seed):
    r, kind = _Random(seed), case["kind"]
    s = {"case": case}
    if kind == "plan":
        N, W, page, limit = case["N"], case["width"], case["page"], case["limit"]
        columns = limit // page
        if case["fresh"]:  # some rows of the batch hold requests already
            lengths = torch.zeros(N, dtype=torch.long)
            new = r.lengths(N, W, True)
        else:
            lengths = r.lengths(N, limit - W, True)
            new = torch.randint(0, W + 1, (N,), generator=r.c) if W > 1 else (torch.rand(N, generator=r.c) < 0.9).long()
        s["table"], used, _ = _table(r, lengths, page, columns)
        need = int(((lengths + new + page - 1) // page - (lengths + page - 1) // page).sum())
        free = max(1, need // 2) if case["scarce"] else need + 7
        s["free_pages"] = (used + r.order(free + 5)).to(torch.int32).cuda()
        s["free_count"] = torch.tensor([free], dtype=torch.int32).cuda()
        s["lengths"], s["new"] = (t.to(torch.int32).cuda() for t in (lengths, new))
        return s
    dt = DTYPES[case["dtype"]]
    if kind == "store":
        N, W, K, hd, page = (case[n] for n in ("N", "width", "kv_heads", "head_dim", "page"))
        lengths = r.lengths(N, W, N > 1)
        table, pages, _ = _table(r, lengths, page, (W + page - 1) // page)
        at = torch.arange(W).cuda()
        slots = table.long()[:, at // page] * page + at % page
        s["slots"] = torch.where(at < lengths.cuda()[:, None], slots, -1)
        s["k"], s["v"] = (r.normal(N, K, W, hd, dtype=dt) for _ in range(2))
        s["pages"] = [r.normal(pages, K, page, hd, dtype=dt) for _ in range(2)]
    elif kind == "prep":
        N, dim, H, K, page, limit = (case[n] for n in ("N", "dim", "heads", "kv_heads", "page", "limit"))
        L = dim // 4
        hd = L // H
        kv = K * hd
        pos = r.lengths(N, limit, True) - 1
        s["qkv"] = r.normal(N, L + 2 * kv, dtype=dt)
        s["ring"] = r.normal(N, BACK + 1, L + 2 * kv, dtype=dt)
        s["positions"] = pos.to(torch.int32).cuda()
        s["slots"] = (r.order(N + 2)[:N] * page + pos % page).cuda()
        s["pages"] = [r.normal(N + 2, K, page, hd, dtype=dt) for _ in range(2)]
        s["weights"] = [r.normal(o, i, TAPS, std=0.02, dtype=dt) for o, i in ((L, hd), (L, L), (kv, hd), (kv, kv))]
        s["temperature"] = r.normal(1, std=0.1, mean=math.sqrt(hd), dtype=dt)
        s["rope"] = _rope_tables(hd, limit)
        if own:  # a program packs its weights once
            from hydra_amd._lib import CCGQA_W_TILED
            from hydra_amd.attention.backends.ccgqa.ops import (pack_conv_weight, pack_conv_weights_tiled, prep_flags,
                                                                tiled_weights_ok)
            tiled = tiled_weights_ok(H, K, hd, dt)
            s["flags"] = prep_flags(True, True, True, True, True) | (CCGQA_W_TILED if tiled else 0)
            s["packed"] = (pack_conv_weights_tiled(s["weights"], dt, H, K, hd) if tiled else
                           tuple(pack_conv_weight(w, dt) for w in s["weights"]))
    elif kind == "attn":
        N, H, K, hd, page = (case[n] for n in ("N", "heads", "kv_heads", "head_dim", "page"))
        lengths = r.lengths(N, case["length"], case["ragged"])
        s["table"], pages, _ = _table(r, lengths, page, (case["length"] + page - 1) // page)
        s["lengths"] = lengths.to(torch.int32).cuda()
        # unit queries, and keys of the length that the layers' temperature gives them
        s["q"] = F.normalize(r.normal(N, H, hd), dim=-1).to(dt)
        s["pages"] = [F.normalize(r.normal(pages, K, page, hd), dim=-1).mul_(4 * math.sqrt(hd)).to(dt),
                      r.normal(pages, K, page, hd, dtype=dt)]
    else:
        n, V = case["rows"], case["vocab"]
        s["logits"] = r.normal(n, V, std=2.5, dtype=dt).requires_grad_(case["train"])
        s["tokens"] = r.ints(V, n)
        if case["train"]:  # advantages of the tokens and a small weight of the entropy, over the batch
            s["grads"] = [r.normal(n, std=1.0 / n), r.normal(n, std=0.01 / n)]
    return s


# ------------------------------------------------------------ the plain forms
def _plan(s):
    case, table = s["case"], s["table"]
    W, page = case["width"], case["page"]
    N, P = table.shape
    dev = table.device
    length, new, free = s["lengths"].long(), s["new"].long(), s["free_count"].long()
    have = (length + page - 1) // page
    fits = (length + new <= P * page) & (new <= W)
    need = torch.where(fits, (length + new + page - 1) // page - have, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= free))
    most = (W + page - 1) // page + 1
    j = torch.arange(most, device=dev)
    takes = granted[:, None] & (j < need[:, None])
    source = (free - 1 - (upto - need)[:, None] - j).clamp(min=0, max=len(s["free_pages"]) - 1)
    column = torch.where(takes, have[:, None] + j, P)
    wide = F.pad(table, (0, 1))
    wide.scatter_(1, column, s["free_pages"][source])
    table.copy_(wide[:, :P])
    at = length[:, None] + torch.arange(W, device=dev)
    slots = table.long().gather(1, (at // page).clamp(max=P - 1)) * page + at % page
    slots = torch.where(granted[:, None] & (torch.arange(W, device=dev) < new[:, None]), slots, -1)
    after = torch.where(granted, length + new, length).to(torch.int32)
    seen = torch.where(granted & (new > 0), after, 0)
    left = (free - torch.where(granted, need, 0).sum()).to(torch.int32)
    return {"slots": slots, "lengths": after, "seen": seen, "granted": granted, "free_count": left, "table": table}


def _store(s):
    kept = s["slots"] >= 0
    slots, page = s["slots"][kept], s["case"]["page"]
    for rows, pages in zip((s["k"], s["v"]), s["pages"]):
        pages[slots // page, :, slots % page] = rows.transpose(1, 2)[kept]
    return list(s["pages"])


def _rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _conv_pair(x, w1, w2, groups):
    """The last row's output of two causal convs over x [N, 5, C]."""
    N, C, c = x.shape[0], x.shape[2], x.shape[2] // groups
    xg = x.view(N, BACK + 1, groups, c)
    w1 = w1.float().view(groups, c, c, TAPS)
    y = 0
    for t in range(TAPS):
        rows = xg[:, t:t + TAPS].permute(2, 0, 1, 3).reshape(groups, N * TAPS, c)
        y = y + torch.bmm(rows, w1[..., t].transpose(1, 2).contiguous())
    y = y.view(groups, N, TAPS, c).permute(1, 2, 0, 3).reshape(N, TAPS, C)
    return sum(y[:, t] @ w2.float()[..., t].t() for t in range(TAPS))


def _prep(s):
    case = s["case"]
    dt, N, H, K, page = DTYPES[case["dtype"]], case["N"], case["heads"], case["kv_heads"], case["page"]
    L = case["dim"] // 4
    hd = L // H
    kv = K * hd
    pos, row = s["positions"].long(), torch.arange(N, device="cuda")
    back = pos[:, None] - torch.arange(BACK, 0, -1, device="cuda")
    before = s["ring"][row[:, None], back % (BACK + 1)].float() * (back >= 0)[..., None]
    x = torch.cat([before, s["qkv"].float()[:, None]], 1)
    q = _conv_pair(x[..., :L], s["weights"][0], s["weights"][1], H).view(N, H, hd)
    k = _conv_pair(x[..., L:L + kv], s["weights"][2], s["weights"][3], K).view(N, K, hd)
    q0, k0 = x[:, -1, :L].view(N, H, hd), x[:, -1, L:L + kv].view(N, K, hd)
    if H == K:
        q, k = q + 0.5 * (q0 + k0), k + 0.5 * (q0 + k0)
    else:
        q, k = q + 0.5 * k0.mean(1, keepdim=True), k + 0.5 * q0.mean(1, keepdim=True)
    q = q / q.pow(2).sum(-1, keepdim=True).sqrt().clamp(min=1e-12)
    k = k / k.pow(2).sum(-1, keepdim=True).sqrt().clamp(min=1e-12) * s["temperature"].float()
    cos, sin = (t[pos][:, None] for t in s["rope"])
    q, k = _rotate(q, cos, sin).to(dt), _rotate(k, cos, sin).to(dt)
    half = kv // 2
    v = torch.cat([x[:, -1, L + kv:L + kv + half], x[:, -2, L + kv + half:]], -1).to(dt).view(N, K, hd)
    for rows, pages in zip((k, v), s["pages"]):
        pages[s["slots"] // page, :, s["slots"] % page] = rows
    s["ring"][row, pos % (BACK + 1)] = s["qkv"]
    return [q, *s["pages"], s["ring"]]


def _attend(s):
    q, table, lengths = s["q"], s["table"].long().clamp(min=0), s["lengths"].long()
    N, H, hd = q.shape
    pages, K, page, _ = s["pages"][0].shape
    G, S = H // K, table.shape[1] * page
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // (K * S * hd))
    for a in range(0, N, step):  # as many requests at a time as a gigabyte of keys holds
        ids, n = table[a:a + step], min(step, N - a)
        k, v = (p[ids].float().transpose(1, 2).reshape(n, K, S, hd) for p in s["pages"])
        past = (torch.arange(S, device=q.device) >= lengths[a:a + step, None])[:, None, None]
        x = q[a:a + step].float().view(n, K, G, hd) @ k.transpose(2, 3).contiguous() * hd ** -0.5
        x = x.masked_fill(past, -math.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        o = (e @ v) / e.sum(-1, keepdim=True)
        out[a:a + step] = o.view(n, H, hd).to(q.dtype)
    return out


def _logprobs(s):
    case, logits, tokens = s["case"], s["logits"].detach(), s["tokens"]
    x = logits.float() / case["temperature"]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    x = x - total.log()
    p = e / total
    entropy = -(p * x).sum(-1)
    out = [x.gather(1, tokens[:, None])[:, 0], entropy]
    if case["top"]:  # the lowest index first among equals
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out += [x.gather(1, order), order]
    if case["train"]:
        gl, ge = (g[:, None] for g in s["grads"])
        grad = -p * (gl + ge * (x + entropy[:, None]))
        grad.scatter_add_(1, tokens[:, None], gl)
        out.append((grad / case["temperature"]).to(logits.dtype))
    return out


# --------------------------------------------------------------- one pass
def _run_own(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "plan":
        from hydra_amd.attention import plan_pages
        plan = plan_pages(s["lengths"], s["new"], s["table"], s["free_pages"], s["free_count"], case["page"],
                          width=case["width"])
        return {"slots": plan.slots, "lengths": plan.lengths, "seen": plan.seen, "granted": plan.granted,
                "free_count": plan.free_count, "table": s["table"]}
    if kind == "store":
        from hydra_amd.attention import store_pages
        store_pages(s["k"], s["v"], *s["pages"], s["slots"])
        return list(s["pages"])
    if kind == "prep":
        from hydra_amd.attention.backends.ccgqa.ops import ccgqa_decode_prep
        hd = case["dim"] // 4 // case["heads"]
        q = ccgqa_decode_prep(s["qkv"], s["ring"], s["positions"], s["slots"], *s["pages"], case["heads"],
                              case["kv_heads"], hd, s["flags"], *s["packed"], temperature=s["temperature"],
                              cos=s["rope"][0], sin=s["rope"][1], packed=True)
        return [q, *s["pages"], s["ring"]]
    if kind == "attn":
        from hydra_amd.attention import paged_attention
        return paged_attention(s["q"], *s["pages"], s["table"], s["lengths"])
    from hydra_amd.kernels import token_logprobs
    got = token_logprobs(s["logits"], s["tokens"], top_k=case["top"], temperature=case["temperature"])
    out = [got.logprobs.detach(), got.entropy.detach()]
    if case["top"]:
        out += [got.top_logprobs.detach(), got.top_tokens]
    if case["train"]:
        out += torch.autograd.grad([got.logprobs, got.entropy], [s["logits"]], s["grads"])
    return out


_PLAIN = {"plan": _plan, "store": _store, "prep": _prep, "attn": _attend, "logp": _logprobs}


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


# ------------------------------------------------------ what a pass needs
def work(case):
    kind = case["kind"]
    r = _Random(0)
    if kind == "plan":
        n = case["N"] * case["width"]
        pages = n // case["page"] if case["fresh"] else case["N"] // case["page"]
        return {"bytes": 8 * n + 8 * pages + 17 * case["N"], "flops": 4 * n}
    e = SIZE[case["dtype"]]
    if kind == "store":
        n = int(r.lengths(case["N"], case["width"], case["N"] > 1).sum())
        return {"bytes": 4 * e * n * case["kv_heads"] * case["head_dim"] + 8 * case["N"] * case["width"], "flops": 0}
    if kind == "prep":
        N, H, K = case["N"], case["heads"], case["kv_heads"]
        L = case["dim"] // 4
        hd = L // H
        kv = K * hd
        weights = TAPS * (L * hd + L * L + kv * hd + kv * kv)
        macs = TAPS * N * (TAPS * L * hd + L * L + TAPS * kv * hd + kv * kv)
        rows = N * ((BACK + 2) * (L + 2 * kv) + L + 2 * kv)
        return {"bytes": e * (weights + rows), "flops": 2 * macs}
    if kind == "attn":
        keys = int(r.lengths(case["N"], case["length"], case["ragged"]).sum())
        rows = 2 * keys * case["kv_heads"] + 2 * case["N"] * case["heads"]
        return {"bytes": e * rows * case["head_dim"], "flops": 4 * keys * case["heads"] * case["head_dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": e * n * (3 if case["train"] else 1) + 24 * case["rows"], "flops": (16 if case["train"] else 6) * n}


# ------------------------------------------------------- in 64 bits
def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "plan":  # whole numbers
        return None
    if kind == "store":  # a copy, row by row of the batch
        for n in range(case["N"]):
            slots = s["slots"][n]
            at = (slots >= 0).nonzero()[:, 0]
            for rows, pages in zip((s["k"], s["v"]), s["pages"]):
                flat = pages.transpose(1, 2)
                flat[slots[at] // case["page"], slots[at] % case["page"]] = rows[n][:, at].transpose(0, 1)
        return [p.double() for p in s["pages"]]
    if kind == "prep":
        return _exact_prep(case, s)
    if kind == "attn":
        outs = []
        K, page = case["kv_heads"], case["page"]
        for n in range(case["N"]):
            S = int(s["lengths"][n])
            ids = s["table"][n, :(S + page - 1) // page].long()
            k, v = (p[ids].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :S] for p in s["pages"])
            q = s["q"][n].double().view(K, -1, case["head_dim"])
            x = torch.matmul(q, k.mT.contiguous()) / math.sqrt(case["head_dim"])
            outs.append(torch.matmul(torch.softmax(x, -1), v).flatten(0, 1))
        return torch.stack(outs)
    parts = []
    step = max(1, (1 << 26) // case["vocab"])
    for a in range(0, case["rows"], step):
        z = s["logits"][a:a + step].detach().double().requires_grad_(case["train"])
        t = s["tokens"][a:a + step, None]
        lp = torch.log_softmax(z / case["temperature"], -1)
        got = [lp.gather(1, t)[:, 0], -(lp.exp() * lp).sum(-1)]
        part = [g.detach() for g in got]
        if case["top"]:
            part += [lp.detach().sort(-1, descending=True).values[:, :case["top"]]]
        if case["train"]:
            part += torch.autograd.grad(got, [z], [g[a:a + step].double() for g in s["grads"]])
        parts.append(part)
    out = [torch.cat(p) for p in zip(*parts)]
    if case["top"]:
        out.insert(3, None)  # whole numbers
    return out


def _exact_prep(case, s):
    N, H, K, page = case["N"], case["heads"], case["kv_heads"], case["page"]
    L = case["dim"] // 4
    hd = L // H
    kv = K * hd
    rows = torch.zeros(N, BACK + 1, L + 2 * kv, dtype=torch.float64)
    ring, new, pos = s["ring"].double().cpu(), s["qkv"].double().cpu(), s["positions"].tolist()
    for n, p in enumerate(pos):
        for j in range(1, BACK + 1):
            if p >= j:
                rows[n, BACK - j] = ring[n, (p - j) % (BACK + 1)]
        rows[n, BACK] = new[n]
    w = [t.double().cpu() for t in s["weights"]]
    ang = torch.tensor(pos)
    cos, sin = (t.double().cpu()[ang] for t in s["rope"])
    x = rows.transpose(1, 2)
    qk = []
    for part, w1, w2, h in ((x[:, :L], w[0], w[1], H), (x[:, L:L + kv], w[2], w[3], K)):
        qk.append(F.conv1d(F.conv1d(part, w1, groups=h), w2)[..., 0].view(N, h, hd))
    q0, k0 = new[:, :L].view(N, H, hd), new[:, L:L + kv].view(N, K, hd)
    means = (0.5 * (q0 + k0),) * 2 if H == K else (0.5 * k0.mean(1, True), 0.5 * q0.mean(1, True))
    gains = (1.0, float(s["temperature"].double()))
    turned = []
    for y, m, g in zip(qk, means, gains):
        y = F.normalize(y + m, dim=-1) * g
        z = torch.view_as_complex(y.view(N, -1, hd // 2, 2)) * torch.complex(cos, sin)[:, None]
        turned.append(torch.view_as_real(z).flatten(-2).cuda())
    v = torch.cat([new[:, L + kv:L + kv + kv // 2], rows[:, BACK - 1, L + kv + kv // 2:]], 1).view(N, K, hd).cuda()
    pages = [p.double() for p in s["pages"]]
    for n, slot in enumerate(s["slots"].tolist()):
        pages[0][slot // page, :, slot % page] = turned[1][n]
        pages[1][slot // page, :, slot % page] = v[n]
        s["ring"][n, pos[n] % (BACK + 1)] = s["qkv"][n]
    return [turned[0], *pages, s["ring"].double()]
