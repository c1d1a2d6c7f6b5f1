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


__all__ = ["plan", "release", "attention", "attention_bound", "decode_bound"]
