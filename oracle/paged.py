"""Oracle for the paged key-value cache: page plans, attention of one token
over pages.  Written from the definitions, one request at a time, in Python
integers and fp64.

Test infrastructure only: see oracle/__init__.py.
"""
from __future__ import annotations

import torch


def plan(lengths, new_tokens, table, free_pages, free_count, page_size, width, from_empty=False):
    """Lists in, lists out: (slots, lengths, seen, granted, free_count, table)."""
    table = [list(r) for r in table]
    P = len(table[0])
    stack = list(free_pages[:max(0, min(free_count, len(free_pages)))])
    slots, after, seen, granted = [], [], [], []
    asked, left = 0, len(stack)
    for i, (n, add) in enumerate(zip(lengths, new_tokens)):
        fits = n >= 0 and 0 <= add <= width and n + add <= P * page_size
        if from_empty and n != 0 and add != 0:
            fits = False
        have = -(-n // page_size) if fits else 0
        need = -(-(n + add) // page_size) - have if fits else 0
        asked += need
        ok = fits and (need == 0 or asked <= len(stack))
        row = [-1] * width
        if ok:
            for j in range(need):
                table[i][have + j] = stack[left - 1 - j]
            left -= need
            for j in range(add):
                page = table[i][(n + j) // page_size]
                row[j] = page * page_size + (n + j) % page_size if page >= 0 else -1
        slots.append(row)
        granted.append(ok)
        after.append(n + add if ok else n)
        seen.append(n + add if ok and add > 0 else 0)
    return slots, after, seen, granted, left, table


def release(done, lengths, table, free_pages, free_count, page_size, pages=None):
    """(lengths, table, free_pages, free_count) after the requests with `done`
    have given their pages back; entries that are no page (negative, or not
    below `pages`) do not come back."""
    lengths, table, free_pages = list(lengths), [list(r) for r in table], list(free_pages)
    top = max(0, min(free_count, len(free_pages)))
    for i, d in enumerate(done):
        if not d:
            continue
        for c in range(min(len(table[i]), max(0, -(-lengths[i] // page_size)))):
            if table[i][c] >= 0 and (pages is None or table[i][c] < pages) and top < len(free_pages):
                free_pages[top] = table[i][c]
                top += 1
            table[i][c] = -1
        lengths[i] = 0
    return lengths, table, free_pages, top


def attention(q, k_pages, v_pages, table, lengths, scale=None):
    """(out, weight): out [N, Hq, hd] fp64 of q over the pages, and
    sum_t p_t |v_t| beside it, which the bounds of its error are stated in.
    Keys on a page outside the pool are not seen; a request without a key gets
    zeros."""
    N, H, hd = q.shape
    pages, K, page, _ = k_pages.shape
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(N, H, hd, dtype=torch.float64)
    weight = torch.zeros(N, H, hd, dtype=torch.float64)
    for n in range(N):
        at = [(int(table[n, t // page]), t % page) for t in range(max(0, min(int(lengths[n]), table.shape[1] * page)))]
        at = [(p, r) for p, r in at if 0 <= p < pages]
        if not at:
            continue
        ids, rows = (torch.tensor(c) for c in zip(*at))
        for h in range(H):
            k = k_pages[ids, h // (H // K), rows].double()
            v = v_pages[ids, h // (H // K), rows].double()
            x = (k @ q[n, h].double()) * scale
            p = torch.softmax(x, 0)
            out[n, h] = p @ v
            weight[n, h] = p @ v.abs()
    return out, weight


def attention_bound(q, k_pages, weight, out, lengths, dtype, scale=None):
    """Largest error of an fp32 evaluation rounded once to dtype, elementwise.

    A score sums hd exact (16-bit) or rounded products: at most (hd + 2) u of
    sum |q k| scale <= |q| |k| scale =: s, u = 2^-24; the scaling and the
    reduction by the maximum add 4 u (s log2(e) + 1) each way.  exp2 is good to
    2 u.  A weight is thus off by a factor within 1 +- d, d = (hd + 16) u
    (2 s + 1); numerator and denominator both, and each sums at most `length`
    terms (u each) and a few joins: out is off by at most
    2 (d + (length + 64) u) sum p |v|, then half a step of dtype."""
    u = 2.0 ** -24
    hd = q.shape[-1]
    scale = hd ** -0.5 if scale is None else scale
    finite = torch.where(torch.isfinite(k_pages.double()), k_pages.double(), torch.zeros(()).double())
    s = float(q.double().norm(dim=-1).max() * finite.norm(dim=-1).max()) * abs(scale)
    d = (hd + 16) * u * (2 * s + 1)
    n = lengths.double().clamp(min=0).view(-1, 1, 1)
    return 2 * (d + (n + 64) * u) * weight * 1.01 + torch.finfo(dtype).eps / 2 * out.abs() * 1.01 + \
        torch.finfo(dtype).smallest_normal



def decode_bound(params, qkv, cfg, dtype):
    """(q, k) bounds, [Hq, hd] and [Hkv, hd], of the error of the last row's q
    and k of qkv [S, W] (fp64) when they are computed in fp32 and rounded once.

    With |.| through both convs: y1 sums ks hd products, y2 ks C, each at most
    u = 2^-24 a product and sum of the absolute values' result Y; a 16-bit
    conv2 takes y1 as two rounded terms, 2^-8 of 2^-8 (bf16; fp16 less): 2^-16
    of Y.  The mean sums at most Hq rows: (Hq + 4) u of its absolute value's.
    The norm then moves z / |z| by at most (dz + |z_i| |dz| / |z|) / |z|, its own
    sum and root by (hd + 8) u; the rotation mixes a pair's errors, 2 u more and
    the table's fp32."""
    u = 2.0 ** -24
    L, K, hd, ks = cfg.latent_dim, cfg.kv_dim, cfg.head_dim, cfg.conv_kernel_size
    S = qkv.shape[0]
    x = qkv.abs()[None]
    parts = {}
    for name, a, b, heads, w in (("q", 0, L, cfg.n_heads, "q_conv"), ("k", L, L + K, cfg.n_kv_heads, "k_conv")):
        C = b - a
        raw = qkv[:, a:b]
        if cfg.use_convs:
            w1, w2 = (params[f"{w}.conv{i}.weight"].double() for i in (1, 2))
            Y = _convs(x[..., a:b], w1.abs(), w2.abs(), heads)[0, -1]
            z = _convs(raw[None], w1, w2, heads)[0, -1]
            dz = (ks * (hd + C) + 8) * u * Y + (0 if dtype == torch.float32 else 2.0 ** -16) * Y
        else:
            z, dz = raw[-1], torch.zeros(C, dtype=torch.float64)
        parts[name] = [z.view(heads, hd), dz.view(heads, hd), raw[-1].view(heads, hd)]
    (zq, dq, q0), (zk, dk, k0) = parts["q"], parts["k"]
    if cfg.use_qk_mean:
        if cfg.n_groups == 1:
            means = [(0.5 * (q0 + k0), 0.5 * (q0.abs() + k0.abs()))] * 2
        else:
            means = [(0.5 * k0.mean(0, True), 0.5 * k0.abs().mean(0, True)),
                     (0.5 * q0.mean(0, True), 0.5 * q0.abs().mean(0, True))]
        zq, zk = zq + means[0][0], zk + means[1][0]
        dq, dk = (d + (cfg.n_heads + 4) * u * m[1] for d, m in zip((dq, dk), means))
    bounds = []
    for z, d, gain in ((zq, dq, 1.0), (zk, dk, float(params["key_temperature"].double()))):
        d = d + 4 * u * z.abs()
        if cfg.use_qk_norm:
            norm = z.norm(dim=-1, keepdim=True)
            d = (d + z.abs() * d.norm(dim=-1, keepdim=True) / norm) / norm * abs(gain)
            z = z / norm * gain
            d = d + (hd + 8) * u * z.abs()
        if cfg.use_rope:
            pair = lambda t: t.view(-1, hd // 2, 2).sum(-1, keepdim=True).expand(-1, -1, 2).reshape(-1, hd)  # noqa: E731
            d = pair(d) + 4 * u * pair(z.abs())
            z = pair(z.abs())
        # z: at least the result's size; half a step of dtype
        bounds.append(1.01 * d + torch.finfo(dtype).eps / 2 * (z.abs() + d) + torch.finfo(dtype).smallest_normal)
    return bounds


def _convs(x, w1, w2, groups):
    from .ccgqa import causal_conv_seq

    return causal_conv_seq(x, w1, w2, groups)




def dequantise(q, scales):
    """What rows of 8 bits and their scales stand for, fp64."""
    x = q.view(torch.int8).float() if q.dtype == torch.int8 else q.float()
    return x.double() * scales.double()[..., None]


def two_term_bound(weight, v, lengths, page_dtype, q_dtype):
    """What the attention over shared prefixes and 8-bit pages adds to
    attention_bound where its products are of 16-bit operands: a weight p (times its
    value's scale) is taken as hi + lo, hi off by half a step of the type, lo by half
    a step of that: 2^-16 of p in bf16 (8-bit pages, bf16), 2^-22 in fp16 (fp16
    pages), where what is left below fp16's least step, 2^-24, is lost by half: under
    a lift of 2^13 (or 2^15) that is 2^-25 2^-13 of a weight whose largest is 1, for
    each key.  (The lifted exponents, up to 16, round by 2^-21: 6 u of a weight, which
    are within the 16 u that attention_bound has beside a score's own.)"""
    if q_dtype == torch.float32:
        return torch.zeros_like(weight)
    if page_dtype == torch.float16:
        finite = torch.where(torch.isfinite(v.double()), v.double(), torch.zeros(()).double())
        return 2.0 ** -22 * weight + 2.0 ** -38 * lengths.double().clamp(min=0).view(-1, 1, 1) * float(finite.abs().max())
    return 2.0 ** -16 * weight


def quantise(x, page_dtype):
    """Rows x [..., hd] in 8 bits: (values fp64 [..., hd], scales fp32 [...]), from
    the definition; fp64 holds the quotients apart from the middles between two
    values (a quotient of two 24-bit numbers is off such a middle by 2^-25 of it
    or not at all)."""
    x = x.double()
    top = x.abs().amax(-1)
    least = torch.tensor(2.0 ** -126, dtype=torch.float64)
    if page_dtype == torch.int8:
        scales = torch.maximum((top / 127).float().double(), least)
        q = torch.round(x / scales[..., None])
    else:
        scales = torch.full_like(top, 2.0 ** -126)
        finite = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
        while bool((large := finite / scales > 448).any()):
            scales[large] *= 2
        y = x / scales[..., None]
        _, e = torch.frexp(y)  # y in [2^(e-1), 2^e): steps of 2^(e-4), of 2^-9 at least
        step = torch.ldexp(torch.ones_like(y), (e - 4).clamp(min=-9))
        q = torch.round(y / step) * step
    wrong = ~torch.isfinite(top)
    q[wrong] = 0.0
    scales[wrong] = float("nan")
    return q, scales.float()


def fork(parents, lengths, table, free_pages, free_count, extra, page_size):
    """Lists in, lists out: (lengths, table, free_pages, free_count, extra,
    sources, copies, taken, granted), by sets of holders."""
    N, P, pages = len(lengths), len(table[0]), len(extra)
    stack = list(free_pages)
    top = max(0, min(free_count, len(stack)))
    parents = [p if 0 <= p < N else -1 for p in parents]
    full = [max(0, min(n // page_size, P)) for n in lengths]
    held = [min(P, -(-n // page_size)) if n > 0 else 0 for n in lengths]
    kids = [[i for i in range(N) if parents[i] == j] for j in range(N)]
    count = {}  # holders of a page that is given up or shared
    for j in range(N):
        for c in range(held[j]):
            p = table[j][c]
            if 0 <= p < pages:
                count[p] = count.get(p, extra[p] + 1) + (len(kids[j]) - 1 if c < full[j] else -(not kids[j]))
    done = set()
    for j in range(N):
        for c in range(held[j]) if not kids[j] else ():
            p = table[j][c]
            if 0 <= p < pages and count[p] == 0 and p not in done:
                done.add(p)
                if top < len(stack):
                    stack[top] = p
                    top += 1
    free, rank = top, 0
    after, rows, sources, copies, taken, granted = [], [], [], [], [], []
    for i, j in enumerate(parents):
        row, length, source, copy, ok = [-1] * P, 0, -1, -1, True
        if j >= 0:
            last = full[j]
            if held[j] > last and kids[j][0] != i and 0 <= table[j][last] < pages:
                ok = rank < free
                if ok:
                    source, copy = table[j][last], stack[free - 1 - rank]
                    top -= 1
                rank += 1
            if ok:
                row[:held[j]] = table[j][:held[j]]
                length = lengths[j]
                if copy >= 0:
                    row[last] = copy
            else:
                for p in table[j][:last]:
                    if 0 <= p < pages:
                        count[p] -= 1
        after.append(length)
        rows.append(row)
        sources.append(source)
        copies.append(copy)
        taken.append(j if ok else -1)
        granted.append(ok)
    extra = [max(0, count[p] - 1) if p in count else extra[p] for p in range(pages)]
    return after, rows, stack, top, extra, sources, copies, taken, granted


__all__ = ["plan", "release", "attention", "attention_bound", "decode_bound", "dequantise", "two_term_bound",
           "quantise", "fork"]
