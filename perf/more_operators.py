"""The operators that continue several texts from shared prompts over a cache
of 8 bits, measured over the sizes, types and directions that are used in
earnest.

A case is a dict of plain values; its "kind" names the operator:

  quant   keys and values of prompts into pages of 8 bits with a scale for
          each row, and read back
  attn    the attention of one new token per request over such pages
  shared  the attention of one new token per request where the requests of a
          group share a prefix, which is read once for all of them
  beam    a step of beam search: the best continuations over the beams and
          the vocabulary of each text
  fork    page tables, pages and states of requests that go on from what
          others hold, the pages shared as far as they are full

`listed()` holds the named cases, `draw(rng)` gives others of the same
ranges, `exact()` restates each operator in 64 bits.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EIGHT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LEAST = 2.0 ** -126  # of a scale

# (heads, kv_heads, head_dim)
HEADS = [(8, 2, 16), (4, 1, 64), (16, 4, 16), (8, 2, 64), (28, 4, 16), (6, 2, 32), (8, 8, 32), (4, 1, 128), (32, 8, 128)]


def listed():
    return [
        # one ragged prompt of a layer with small heads goes into the cache
        dict(name="quant_prompt", kind="quant", dtype="bf16", eight="int8", N=1, width=1003, kv_heads=4, head_dim=16,
             page=16),
        # a batch of long prompts
        dict(name="quant_batch", kind="quant", dtype="bf16", eight="e4m3", N=16, width=4096, kv_heads=2, head_dim=64,
             page=64),
        # a single user's token with a short context: latency
        dict(name="attn_one", kind="attn", dtype="bf16", eight="int8", N=1, heads=4, kv_heads=1, head_dim=64, page=64,
             length=700, ragged=False),
        # a server's requests of all lengths, seven heads to a key head of 16
        dict(name="attn_ragged", kind="attn", dtype="fp16", eight="int8", N=48, heads=28, kv_heads=4, head_dim=16,
             page=16, length=8192, ragged=True),
        # many long contexts: what the 8 bits are for
        dict(name="attn_long", kind="attn", dtype="bf16", eight="e4m3", N=64, heads=8, kv_heads=2, head_dim=64, page=64,
             length=16384, ragged=False),
        # four beams of each of eight texts, soon after their prompts
        dict(name="shared_beams", kind="shared", dtype="bf16", eight="", groups=8, width=4, heads=8, kv_heads=2,
             head_dim=64, page=64, prefix=1500, suffix=48),
        # every request of a full server begins with the same long instructions
        dict(name="shared_system", kind="shared", dtype="bf16", eight="", groups=1, width=256, heads=32, kv_heads=8,
             head_dim=128, page=64, prefix=32768, suffix=600),
        # a program that keeps everything in fp32, a key head for each head, samples 12 answers to each question
        dict(name="shared_fp32", kind="shared", dtype="fp32", eight="", groups=2, width=12, heads=8, kv_heads=8,
             head_dim=32, page=32, prefix=3001, suffix=200),
        # the first texts of a single user
        dict(name="beam_one", kind="beam", dtype="bf16", groups=1, width=4, vocab=50257, count=4),
        # a batch of texts with room for beams that end
        dict(name="beam_batch", kind="beam", dtype="bf16", groups=32, width=8, vocab=32000, count=16),
        # the same texts' tables, pages and states afterwards
        dict(name="fork_one", kind="fork", dtype="bf16", groups=1, width=4, kv_heads=1, head_dim=64, page=64, prefix=700,
             suffix=48, limit=4096),
        dict(name="fork_batch", kind="fork", dtype="bf16", groups=32, width=8, kv_heads=2, head_dim=64, page=16,
             prefix=2000, suffix=200, limit=8192),
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "attn", "attn", "shared", "shared", "beam", "fork"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    eight = rng.choice(["int8", "e4m3"])
    H, K, hd = rng.choice(HEADS)
    if kind == "quant":
        N = _log_int(rng, 1, 64)
        return dict(kind=kind, dtype=dtype, eight=eight, N=N, width=_log_int(rng, 1, 65536 * 64 // (N * K * hd)),
                    kv_heads=K, head_dim=hd, page=page)
    if kind == "attn":
        N = _log_int(rng, 1, 256)
        most = (1 << 28) // (N * K * hd)  # keys of as many bytes as the longest listed case reads in all
        return dict(kind=kind, dtype=dtype, eight=eight, N=N, heads=H, kv_heads=K, head_dim=hd, page=page,
                    length=_log_int(rng, 1, max(1, min(32768, most // 2))), ragged=rng.random() < 0.6)
    if kind == "shared":
        groups, width = _log_int(rng, 1, 16), _log_int(rng, 2, 64)
        suffix = _log_int(rng, 1, min(2048, (1 << 26) // (groups * width * K * hd)))
        return dict(kind=kind, dtype=dtype, eight=rng.choice(["", "", eight]), groups=groups, width=width, heads=H,
                    kv_heads=K, head_dim=hd, page=page, suffix=suffix,
                    prefix=_log_int(rng, 1, min(32768, (1 << 26) // (groups * K * hd))))
    if kind == "beam":
        groups, width = _log_int(rng, 1, 32), rng.randint(1, 16)
        return dict(kind=kind, dtype=dtype, groups=groups, width=width, vocab=rng.choice([4099, 16000, 32000, 50257]),
                    count=width * rng.choice([1, 2]))
    return dict(kind=kind, dtype=dtype, groups=_log_int(rng, 1, 32), width=rng.randint(2, 12), kv_heads=K,
                head_dim=min(hd, 64), page=page, prefix=_log_int(rng, 1, 4096), suffix=_log_int(rng, 1, 512), limit=8192)


# ------------------------------------------------------------------ inputs
class _Random:
    """Inputs on the GPU from a seed alone; sizes of requests from the CPU's
    generator."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))
        self.c = torch.Generator().manual_seed(int(seed) + 1)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std).add_(mean).to(dtype)

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
    has none; the number of pages in the pool."""
    counts = (lengths + page - 1) // page
    used = int(counts.sum())
    total = used + 3
    table = torch.full((len(lengths), columns), -1)
    table[torch.arange(columns)[None] < counts[:, None]] = r.order(total)[:used]
    return table.to(torch.int32).cuda(), total


def _scales(x, eight):
    """fp32 scales of rows x [..., hd] (fp32): int8 divides the row's largest
    value by 127; e4m3 takes the least power of two that brings it to 448."""
    top = x.abs().amax(-1)
    if eight == "int8":
        return (top / 127).clamp(min=LEAST)
    m, e = torch.frexp(top)
    return torch.ldexp(torch.ones_like(top), torch.where(m <= 0.875, e - 9, e - 8)).clamp(min=LEAST)


def _to_eight(x, scales, eight):
    """Rows x (fp32) in 8 bits.  A quotient beside the middle of two whole
    numbers needs 64 bits; by a power of two it is exact."""
    if eight == "int8":
        return (x.double() / scales[..., None].double()).round().clamp(-127, 127).to(torch.int8)
    return (x / scales[..., None]).to(torch.float8_e4m3fn)


def _eight_pages(r, rows, eight):
    """Pages of 8 bits and their scales from rows [pages, K, page, hd]."""
    scales = _scales(rows, eight)
    return _to_eight(rows, scales, eight), scales


def _pages(r, pages, K, page, hd, dt, eight):
    """Keys of the length that the layers' temperature gives them, values, and
    the scales of both (None in 16 and 32 bits)."""
    rows = [F.normalize(r.normal(pages, K, page, hd), dim=-1).mul_(4 * math.sqrt(hd)).to(dt), r.normal(pages, K, page, hd).to(dt)]
    if not eight:
        return rows, None
    (k, ks), (v, vs) = (_eight_pages(r, t.float(), eight) for t in rows)
    return [k, v], [ks, vs]


def _groups(r, case):
    """Tables [groups x width, columns] of requests that share their prefix's
    full pages and have all behind it for themselves; lengths of prefixes and
    requests; (from, to) pages that hold the same end of a prefix; pages."""
    B, W, page = case["groups"], case["width"], case["page"]
    prefix = r.lengths(B, case["prefix"], B > 1)
    lengths = prefix.repeat_interleave(W) + r.lengths(B * W, case["suffix"], True)
    columns = case.get("limit", int(lengths.max())) // page + 1
    full = prefix // page
    counts = (lengths + page - 1) // page - full.repeat_interleave(W)
    total = int(full.sum()) + B * W * (case["suffix"] // page + 2)  # whatever the order
    ids = r.order(total)
    table = torch.full((B * W, columns), -1)
    at, same = 0, []
    for b in range(B):
        table[b * W:(b + 1) * W, :full[b]] = ids[at:at + int(full[b])]
        at += int(full[b])
        for n in range(b * W, (b + 1) * W):
            table[n, full[b]:full[b] + counts[n]] = ids[at:at + int(counts[n])]
            at += int(counts[n])
            if n > b * W and prefix[b] % page:
                same.append((int(table[b * W, full[b]]), int(table[n, full[b]]), int(prefix[b] % page)))
    return table.to(torch.int32), prefix, lengths, same, total


def prepare(case, seed):
    r, kind = _Random(seed), case["kind"]
    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    if kind == "quant":
        N, W, K, hd, page = (case[n] for n in ("N", "width", "kv_heads", "head_dim", "page"))
        lengths = r.lengths(N, W, N > 1)
        table, pages = _table(r, lengths, page, (W + page - 1) // page)
        at = torch.arange(W).cuda()
        slots = table.long()[:, at // page] * page + at % page
        s["slots"] = torch.where(at < lengths.cuda()[:, None], slots, -1)
        s["k"], s["v"] = (r.normal(N, K, W, hd, dtype=dt) for _ in range(2))
        s["pages"] = [torch.zeros(pages, K, page, hd, device="cuda").to(EIGHT[case["eight"]]) for _ in range(2)]
        s["scales"] = [torch.ones(pages, K, page, device="cuda") for _ in range(2)]
    elif kind == "attn":
        N, H, K, hd, page = (case[n] for n in ("N", "heads", "kv_heads", "head_dim", "page"))
        lengths = r.lengths(N, case["length"], case["ragged"])
        s["table"], pages = _table(r, lengths, page, (case["length"] + page - 1) // page)
        s["lengths"] = lengths.to(torch.int32).cuda()
        s["q"] = F.normalize(r.normal(N, H, hd), dim=-1).to(dt)
        s["pages"], s["scales"] = _pages(r, pages, K, page, hd, dt, case["eight"])
    elif kind == "shared":
        H, K, hd, page = (case[n] for n in ("heads", "kv_heads", "head_dim", "page"))
        table, prefix, lengths, same, pages = _groups(r, case)
        s["table"], s["shared"], s["lengths"] = (t.to(torch.int32).cuda() for t in (table, prefix, lengths))
        s["q"] = F.normalize(r.normal(len(lengths), H, hd), dim=-1).to(dt)
        s["pages"], s["scales"] = _pages(r, pages, K, page, hd, dt, case["eight"])
        for a, b, rows in same:  # each request's copy of the prefix's last page
            for t in [*s["pages"], *(s["scales"] or ())]:
                t[b, :, :rows] = t[a, :, :rows]
    elif kind == "beam":
        B, W, V = case["groups"], case["width"], case["vocab"]
        s["logits"] = r.normal(B * W, V, std=2.5, dtype=dt)
        s["scores"] = r.normal(B, W, std=1.0, mean=-20.0)
    else:
        B, W, K, hd, page = (case[n] for n in ("groups", "width", "kv_heads", "head_dim", "page"))
        table, prefix, lengths, _, pages = _groups(r, case)
        # a page for each fork, and some
        spare = B * W * (case["suffix"] // page + 2)
        extra = torch.zeros(pages + spare, dtype=torch.int32)
        full = prefix // page
        for b in range(B):
            extra[table[b * W, :full[b]].long()] = W - 1
        first = torch.arange(B).repeat_interleave(W) * W
        s["parents"] = (first + torch.randint(0, W, (B * W,), generator=r.c)).to(torch.int32).cuda()
        stack = pages + r.order(spare)
        s["free_pages"] = torch.cat([stack, torch.zeros(pages, dtype=torch.long)]).to(torch.int32).cuda()
        s["free_count"] = torch.tensor([spare], dtype=torch.int32).cuda()
        s["table"], s["lengths"], s["extra"] = (t.to(torch.int32).cuda() for t in (table, lengths, extra))
        s["pages"] = [r.normal(pages + spare, K, page, hd, dtype=dt) for _ in range(2)]
        s["ring"] = r.normal(B * W, 5, 8 * K * hd, dtype=dt)
    return s


# ------------------------------------------------------------ the plain forms
def _quant(s):
    case = s["case"]
    page, eight, dt = case["page"], case["eight"], DTYPES[case["dtype"]]
    kept = s["slots"] >= 0
    slots = s["slots"][kept]
    back = []
    for rows, pages, scales in zip((s["k"], s["v"]), s["pages"], s["scales"]):
        x = rows.transpose(1, 2)[kept].float()
        scale = _scales(x, eight)
        pages.view(torch.int8)[slots // page, :, slots % page] = _to_eight(x, scale, eight).view(torch.int8)
        scales[slots // page, :, slots % page] = scale
        q = pages.view(torch.int8)[slots // page, :, slots % page].view(pages.dtype)
        out = torch.zeros_like(rows)
        out.transpose(1, 2)[kept] = (q.float() * scales[slots // page, :, slots % page][..., None]).to(dt)
        back.append(out)
    return {"k": back[0], "v": back[1], "k_scales": s["scales"][0], "v_scales": s["scales"][1]}


def _gathered(s, ids):
    """fp32 keys and values [n, K, S, hd] of page ids [n, columns]."""
    out = []
    for i, p in enumerate(s["pages"]):
        x = p.view(torch.int8)[ids].view(p.dtype).float() if p.element_size() == 1 else p[ids].float()
        if s["scales"]:
            x = x * s["scales"][i][ids][..., None]
        n, c, K, page, hd = x.shape
        out.append(x.transpose(1, 2).reshape(n, K, c * page, hd))
    return out


def _attend(s):
    q, table, lengths = s["q"], s["table"].long().clamp(min=0), s["lengths"].long()
    N, H, hd = q.shape
    _, K, page, _ = s["pages"][0].shape
    G, S = H // K, table.shape[1] * page
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // (K * S * hd))
    for a in range(0, N, step):  # as many requests at a time as a gigabyte of keys holds
        n = min(step, N - a)
        k, v = _gathered(s, table[a:a + step])
        past = (torch.arange(S, device=q.device) >= lengths[a:a + step, None])[:, None, None]
        x = q[a:a + step].float().view(n, K, G, hd) @ k.transpose(2, 3).contiguous() * hd ** -0.5
        x = x.masked_fill(past, -math.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        o = (e @ v) / e.sum(-1, keepdim=True)
        out[a:a + step] = o.view(n, H, hd).to(q.dtype)
    return out


def _attend_shared(s):
    """The prefix's scores of a group's requests in one product, those of what
    is behind it for each request."""
    case, q = s["case"], s["q"]
    table, shared, lengths = s["table"].long().clamp(min=0), s["shared"].long(), s["lengths"].long()
    N, H, hd = q.shape
    _, K, page, _ = s["pages"][0].shape
    B, W, G = case["groups"], case["width"], H // K
    out = torch.empty_like(q)
    first = (case["prefix"] + page - 1) // page
    behind = (case["suffix"] + page - 1) // page + 1
    step = max(1, (1 << 28) // (K * behind * page * hd))
    for b in range(B):
        rows = slice(b * W, (b + 1) * W)
        x = q[rows].float().view(W, K, G, hd).transpose(0, 1).reshape(K, W * G, hd) * hd ** -0.5
        k, v = (t[0] for t in _gathered(s, table[b * W:b * W + 1, :first]))
        seen = torch.arange(k.shape[1], device=q.device) < shared[b]
        x1 = (x @ k.transpose(1, 2).contiguous()).masked_fill(~seen, -math.inf).view(K, W, G, -1).transpose(0, 1)
        m1 = x1.amax(-1, keepdim=True)
        e1 = torch.exp(x1 - m1)
        o1 = (e1.transpose(0, 1).reshape(K, W * G, -1) @ v).view(K, W, G, hd).transpose(0, 1)
        for a in range(0, W, step):
            n = min(step, W - a)
            at = slice(b * W + a, b * W + a + n)
            cols = shared[b] // page + torch.arange(behind, device=q.device)
            ids = table[at][:, cols.clamp(max=table.shape[1] - 1)]
            k, v = _gathered(s, ids)
            t = (cols[:, None] * page + torch.arange(page, device=q.device)).flatten()
            seen = (t >= shared[b]) & (t < lengths[at, None])
            x2 = q[at].float().view(n, K, G, hd) @ k.transpose(2, 3).contiguous() * hd ** -0.5
            x2 = x2.masked_fill(~seen[:, None, None], -math.inf)
            m = torch.maximum(m1[a:a + n], x2.amax(-1, keepdim=True))
            e2, c = torch.exp(x2 - m), torch.exp(m1[a:a + n] - m)
            o = o1[a:a + n] * c + e2 @ v
            total = e1[a:a + n].sum(-1, keepdim=True) * c + e2.sum(-1, keepdim=True)
            out[at] = (o / total).reshape(n, H, hd).to(q.dtype)
    return out


def _beam(s):
    """In 64 bits: of two continuations of nearly equal score the order counts."""
    case = s["case"]
    B, W, V, n = case["groups"], case["width"], case["vocab"], case["count"]
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = x - x.exp().sum(-1, keepdim=True).log()
    x = (s["scores"].double().view(B * W, 1) + x).view(B, W * V)
    order = torch.sort(x, dim=1, descending=True, stable=True)  # the lowest index first among equals
    best = order.indices[:, :n]
    return {"scores": order.values[:, :n].float(), "beams": best // V, "tokens": best % V}


def _fork(s):
    case, table, page = s["case"], s["table"].long(), s["case"]["page"]
    N, P = table.shape
    dev = table.device
    parents, length, pages = s["parents"].long(), s["lengths"].long(), s["extra"].numel()
    row, col = torch.arange(N, device=dev), torch.arange(P, device=dev)
    have, full = (length + page - 1) // page, length // page
    kids = torch.zeros(N, dtype=torch.long, device=dev).scatter_add_(0, parents, torch.ones_like(parents))
    first = torch.full((N,), N, device=dev).scatter_reduce_(0, parents, row, "amin")
    held, whole, idle = col < have[:, None], col < full[:, None], (kids == 0)[:, None]
    # holders of each page, the entries that are none counted in one more
    gone = torch.where(whole, kids[:, None] - 1, torch.where(held & idle, -1, 0))
    entry = torch.where(held, table, pages)
    extra = F.pad(s["extra"].long(), (0, 1)).scatter_add_(0, entry.flatten(), gone.flatten())
    owner = torch.full((pages + 1,), N, device=dev)
    owner.scatter_reduce_(0, torch.where(idle, entry, pages).flatten(), row[:, None].expand(N, P).flatten(), "amin")
    back = held & idle & (extra[entry] < 0) & (owner[entry] == row[:, None])
    free = s["free_count"].long()
    to = free + back.flatten().cumsum(0) - 1
    stack = F.pad(s["free_pages"], (0, 1))
    stack.scatter_(0, torch.where(back.flatten(), to, s["free_pages"].numel()), entry.flatten().to(torch.int32))
    s["free_pages"].copy_(stack[:-1])
    extra = extra[:-1].clamp(min=0)
    free = free + back.sum()
    need = (first[parents] != row) & (have[parents] > full[parents])
    rank = need.long().cumsum(0) - 1
    granted = ~need | (rank < free)
    takes = need & granted
    last = full[parents].clamp(max=P - 1)
    copies = torch.where(takes, s["free_pages"].long()[(free - 1 - rank).clamp(min=0)], -1)
    sources = torch.where(takes, table[parents, last], -1)
    new = torch.where((col < have[parents, None]) & granted[:, None], table[parents], -1)
    new = torch.where(takes[:, None] & (col == last[:, None]), copies[:, None], new)
    refused = (~granted)[:, None] & (col < full[parents, None])
    extra = F.pad(extra, (0, 1)).scatter_add_(0, torch.where(refused, table[parents], pages).flatten(), -refused.long().flatten())
    s["extra"].copy_(extra[:-1])
    s["free_count"].copy_(free - takes.sum())
    s["table"].copy_(new)
    s["lengths"].copy_(torch.where(granted, length[parents], 0))
    for p in s["pages"]:
        p[copies[takes]] = p[sources[takes]]
    s["ring"].copy_(s["ring"][parents])
    return {n: s[n] for n in ("table", "lengths", "free_pages", "free_count", "extra", "pages", "ring")} | {"granted": granted}


# --------------------------------------------------------------- one pass
def _run_own(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "quant":
        from hydra_amd.attention import read_pages, store_pages
        store_pages(s["k"], s["v"], *s["pages"], s["slots"], scales=s["scales"])
        k, v = read_pages(*s["pages"], s["slots"], scales=s["scales"], dtype=s["k"].dtype)
        return {"k": k, "v": v, "k_scales": s["scales"][0], "v_scales": s["scales"][1]}
    if kind == "attn":
        from hydra_amd.attention import paged_attention
        return paged_attention(s["q"], *s["pages"], s["table"], s["lengths"], scales=s["scales"])
    if kind == "shared":
        from hydra_amd.attention import paged_attention
        return paged_attention(s["q"], *s["pages"], s["table"], s["lengths"], scales=s["scales"], shared=s["shared"])
    if kind == "beam":
        from hydra_amd.kernels import beam_select
        best = beam_select(s["logits"], s["scores"], case["count"])
        return {"scores": best.scores, "beams": best.beams, "tokens": best.tokens}
    from hydra_amd.attention import copy_pages, fork_pages, take_rows
    fork = fork_pages(s["parents"], s["lengths"], s["table"], s["free_pages"], s["free_count"], s["extra"], case["page"])
    copy_pages(*s["pages"], fork.sources, fork.copies)
    take_rows(s["ring"], fork.parents)
    return {n: s[n] for n in ("table", "lengths", "free_pages", "free_count", "extra", "pages", "ring")} | \
        {"granted": fork.granted}


_PLAIN = {"quant": _quant, "attn": _attend, "shared": _attend_shared, "beam": _beam, "fork": _fork}


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


# ------------------------------------------------------ what a pass needs
def work(case):
    kind = case["kind"]
    r = _Random(0)
    e = SIZE[case["dtype"]]
    if kind == "quant":
        n = int(r.lengths(case["N"], case["width"], case["N"] > 1).sum())
        rows, all_rows = n * case["kv_heads"], case["N"] * case["width"] * case["kv_heads"]
        # rows read, 8 bits and scales written and read, rows written back with zeros beside them
        return {"bytes": 2 * (rows * (e + 2) * case["head_dim"] + 8 * rows + e * all_rows * case["head_dim"]) +
                16 * case["N"] * case["width"], "flops": 8 * rows * case["head_dim"]}
    if kind in ("attn", "shared"):
        H, K, hd = case["heads"], case["kv_heads"], case["head_dim"]
        row = 2 * K * (hd + 4 if case["eight"] else e * hd)  # bytes of a position
        if kind == "attn":
            keys = read = int(r.lengths(case["N"], case["length"], case["ragged"]).sum())
            N = case["N"]
        else:
            B, W = case["groups"], case["width"]
            N, prefix = B * W, int(r.lengths(B, case["prefix"], B > 1).sum())
            behind = int(r.lengths(N, case["suffix"], True).sum())
            keys, read = W * prefix + behind, prefix + behind
        return {"bytes": read * row + 2 * e * N * H * hd, "flops": 4 * keys * H * hd}
    if kind == "beam":
        n = case["groups"] * case["width"] * case["vocab"]
        return {"bytes": e * n + 20 * case["groups"] * case["count"], "flops": 4 * n}
    N, page = case["groups"] * case["width"], case["page"]
    # tables, about a third of the rows with a page of each kind and a state to copy
    pages = 2 * N * ((case["prefix"] + case["suffix"]) // page + 1)
    moved = 2 * (N // 3) * e * case["kv_heads"] * case["head_dim"] * (2 * page + 40)
    return {"bytes": 4 * pages + moved, "flops": 4 * pages}


# ------------------------------------------------------- in 64 bits
def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "fork":  # whole numbers and copies
        return None
    if kind == "quant":
        out = []
        for name, scales in zip("kv", s["scales"]):
            x = s[name].double()
            top = x.abs().amax(-1)
            if case["eight"] == "int8":  # the scale is kept in fp32, and the row rounded against that
                scale = (top / 127).float().double().clamp(min=LEAST)
                q = torch.round(x / scale[..., None])
            else:
                scale = torch.exp2(torch.ceil(torch.log2(top / 448))).clamp(min=LEAST)
                y = x / scale[..., None]
                # steps of e4m3: 2^-9 below 2^-6, then 8 to each power of two
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                q = torch.round(y / step) * step
            kept = s["slots"] >= 0
            out.append((q * scale[..., None]) * kept[:, None, :, None])
            held = scales.double()
            slots = s["slots"][kept]
            held[slots // case["page"], :, slots % case["page"]] = scale.transpose(1, 2)[kept]
            out.append(held)
        return {"k": out[0], "v": out[2], "k_scales": out[1], "v_scales": out[3]}
    if kind in ("attn", "shared"):  # each request by itself
        outs = []
        K, page = case["kv_heads"], case["page"]
        for n in range(s["q"].shape[0]):
            S = int(s["lengths"][n])
            ids = s["table"][n, :(S + page - 1) // page].long()
            kv = []
            for i, p in enumerate(s["pages"]):
                x = (p.view(torch.int8)[ids].view(p.dtype).float() if p.element_size() == 1 else p[ids]).double()
                if s["scales"]:
                    x = x * s["scales"][i][ids].double()[..., None]
                kv.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :S])
            q = s["q"][n].double().view(K, -1, case["head_dim"])
            x = torch.matmul(q, kv[0].mT.contiguous()) / math.sqrt(case["head_dim"])
            outs.append(torch.matmul(torch.softmax(x, -1), kv[1]).flatten(0, 1))
        return torch.stack(outs)
    B, W, V = case["groups"], case["width"], case["vocab"]
    best = []
    for b in range(B):
        lp = torch.log_softmax(s["logits"][b * W:(b + 1) * W].double(), -1) + s["scores"][b].double()[:, None]
        best.append(torch.topk(lp.flatten(), case["count"]).values)
    return {"scores": torch.stack(best), "beams": None, "tokens": None}
