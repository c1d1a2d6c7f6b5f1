"""GPU tests of rows stored in pages of 8 bits and read back, against the oracle:
the same bits."""
from __future__ import annotations

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EIGHT = [torch.int8, torch.float8_e4m3fn]


def bits(t):
    """Comparable bits, every NaN alike."""
    if t.dtype == torch.float32:
        return torch.where(t.isnan(), 0x7fc00000, t.view(torch.int32))
    return t.view(torch.int8)


def nearest(x, dtype):
    """fp64 rounded to dtype at once (torch's own conversion goes through fp32), as fp64."""
    info = torch.finfo(dtype)
    _, e = torch.frexp(torch.nan_to_num(x))  # |x| in [2^(e-1), 2^e)
    _, least = torch.frexp(torch.tensor(info.smallest_normal, dtype=torch.float64))
    step = torch.ldexp(torch.ones_like(x), torch.maximum(e, least) - 1) * info.eps
    out = torch.round(x / step) * step
    return torch.where(out.abs() > info.max, torch.sign(out) * float("inf"), out)


def pool(pages, K, page, hd, eight, device):
    """Pages and scales that hold something else."""
    g = torch.Generator().manual_seed(9)
    make = lambda: torch.randint(0, 100, (pages, K, page, hd), generator=g, dtype=torch.int8).view(eight).to(device)  # noqa: E731
    return make(), make(), *(torch.rand(pages, K, page, generator=g).to(device) for _ in range(2))


def check(cuda, k, v, slots, page, eight, rows=None, pages=None, form=lambda n, t: t):
    """The stored bits, all others as they were, and what reads back."""
    from hydra_amd.attention import read_pages, store_pages

    _, K, S, hd = k.shape
    pages = pages or 8
    kp, vp, ks, vs = (form(n, t) for n, t in zip(("kp", "vp", "ks", "vs"), pool(pages, K, page, hd, eight, cuda)))
    want = [t.cpu().clone() for t in (kp, vp, ks, vs)]
    src = range(k.shape[0]) if rows is None else rows.tolist()
    for x, q8, s8 in ((k, want[0], want[2]), (v, want[1], want[3])):
        q, s = op.quantise(x, eight)
        q = q.to(torch.int8) if eight == torch.int8 else q.float().to(eight)
        for n, r in enumerate(src):
            if not 0 <= r < slots.shape[0]:
                continue
            for t, at in enumerate(slots[r].tolist()):
                if 0 <= at < pages * page:
                    q8.view(torch.int8)[at // page, :, at % page] = q.view(torch.int8)[n, :, t]
                    s8[at // page, :, at % page] = s[n, :, t]
    dev = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    store_pages(form("k", dev(k)), form("v", dev(v)), kp, vp, dev(slots), dev(rows), scales=(ks, vs))
    for name, got, exp in zip(("keys", "values", "key scales", "value scales"), (kp, vp, ks, vs), want):
        assert int((bits(got.cpu()) != bits(exp)).sum()) == 0, name
    for dtype in DTYPES:
        back = read_pages(kp, vp, dev(slots), dev(rows), scales=(ks, vs), dtype=dtype)
        for got, q8, s8 in zip(back, want[:2], want[2:]):
            exp = torch.zeros(got.shape, dtype=torch.float64)
            for n, r in enumerate(src):
                for t, at in enumerate(slots[r].tolist() if 0 <= r < slots.shape[0] else ()):
                    if 0 <= at < pages * page:
                        exp[n, :, t] = op.dequantise(q8[at // page, :, at % page].contiguous(), s8[at // page, :, at % page])
            # A product of an 8-bit and a 24-bit number has 32 bits.  It is rounded to dtype, and may be
            # rounded to fp32 before that: to one of two neighbours of dtype then, where it lies within
            # 2^-25 of it of their middle, and to the nearest of them elsewhere.  fp64 holds it exactly.
            got, once, twice = (torch.nan_to_num(x.double(), 7.5) for x in (got.cpu(), nearest(exp, dtype), exp.float().to(dtype)))
            wrong = (got != once) & (got != twice)
            assert not bool(wrong.any()), (got[wrong], once[wrong], twice[wrong])
    return kp, vp, ks, vs


@pytest.mark.parametrize("eight", EIGHT)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [1, 3, 8, 16, 20, 32, 33, 48, 64, 80, 128, 250, 256])
def test_head_dims(cuda, eight, dtype, hd):
    g = torch.Generator().manual_seed(hd)
    k, v = (torch.randn(2, 3, 19, hd, generator=g).to(dtype) for _ in range(2))
    slots = torch.randperm(8 * 16, generator=g)[:38].view(2, 19)
    slots[0, 3], slots[1, 7], slots[1, 0] = -1, 128, -2**62
    check(cuda, k, v, slots, 16, eight)


@pytest.mark.parametrize("eight", EIGHT)
@pytest.mark.parametrize("dtype", DTYPES)
def test_middles_and_extremes(cuda, eight, dtype):
    """Quotients in the middle of two values, rows of zeros, of the type's largest
    and least values, and with values of all sizes beside them."""
    g = torch.Generator().manual_seed(1)
    info = torch.finfo(dtype)
    rows = []
    for m in range(128, 256):  # every 8-bit significand as the largest, all halves and eighths of it beside it
        rows.append(torch.tensor([m, m / 2, -m / 2, m / 4, m / 8, 3 * m / 8, -5 * m / 8, 7 * m / 8] * 2))
    for e in range(16):
        rows.append(torch.arange(16).float() * 2.0 ** (e - 8))
    x = torch.stack(rows)
    x = torch.cat([x, torch.randn(64, 16, generator=g) * torch.exp2(torch.randint(-30, 30, (64, 16), generator=g).float())])
    x = x.to(dtype)
    extra = torch.zeros(12, 16, dtype=dtype)
    extra[1] = info.max
    extra[2, 0], extra[2, 1] = -info.max, 1
    extra[3] = info.smallest_normal
    extra[4, 5] = info.smallest_normal * info.eps  # the least subnormal
    extra[5] = info.smallest_normal * info.eps * torch.arange(16)
    extra[6, 3] = float("nan")
    extra[7, 15] = float("inf")
    extra[8, 0] = float("-inf")
    extra[9] = -0.0
    extra[10] = torch.where(torch.arange(16) % 2 == 0, 1.75, 1.7500001)
    extra[11] = 448
    x = torch.cat([x, extra])[None, None]
    S = x.shape[2]
    check(cuda, x, x.flip(2), torch.randperm(S, generator=g)[None], 16, eight, pages=-(-S // 16))


@pytest.mark.parametrize("eight", EIGHT)
def test_strides_and_rows(cuda, eight):
    """Rows taken from [N, S, K, hd], pages with gaps, scales of other strides, prompts in the rows of a plan."""
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(3, 2, 21, 32, generator=g).to(torch.bfloat16) for _ in range(2))
    slots = torch.randperm(8 * 32, generator=g)[:105].view(5, 21)

    def form(name, t):
        if name in ("k", "v"):
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if name in ("ks", "vs"):
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        wide = torch.zeros(*t.shape[:2], t.shape[2] * 2, t.shape[3] + 16, dtype=torch.int8, device=t.device)
        out = wide.view(t.dtype)[:, :, ::2, 16:]
        out.view(torch.int8).copy_(t.view(torch.int8))
        return out

    check(cuda, k, v, slots, 32, eight, rows=torch.tensor([4, 1, 9]), form=form)


def test_many_prompts(cuda):
    """More prompts than a grid has along an axis."""
    from hydra_amd.attention import read_pages, store_pages

    N = 70000
    g = torch.Generator().manual_seed(2)
    k = torch.randn(N, 1, 1, 16, generator=g)
    kp, vp, ks, vs = pool(N // 16 + 1, 1, 16, 16, torch.int8, cuda)
    slots = torch.randperm(N, generator=g)[:, None]
    store_pages(k.to(cuda), k.to(cuda), kp, vp, slots.to(cuda), scales=(ks, vs))
    back, _ = read_pages(kp, vp, slots.to(cuda), scales=(ks, vs), dtype=torch.float32)
    q, s = op.quantise(k, torch.int8)
    assert torch.equal(back.cpu(), (q * s.double()[..., None]).float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [3, 16, 64, 250])
def test_other_pages_are_read_as_they_are(cuda, dtype, hd):
    from hydra_amd.attention import read_pages

    g = torch.Generator().manual_seed(hd)
    kp, vp = (torch.randn(5, 2, 16, hd, generator=g).to(dtype).to(cuda) for _ in range(2))
    slots = torch.randint(-3, 90, (4, 9), generator=g).to(cuda)
    for got, p in zip(read_pages(kp, vp, slots), (kp, vp)):
        at = slots.clamp(0, 79)
        want = p[at // 16, :, at % 16].transpose(1, 2)
        assert torch.equal(got, torch.where(((slots >= 0) & (slots < 80))[:, None, :, None], want, 0))


def test_nothing_to_do(cuda):
    from hydra_amd.attention import read_pages, store_pages

    kp, vp, ks, vs = pool(2, 2, 16, 16, torch.int8, cuda)
    before = kp.clone()
    for n, s in ((0, 4), (3, 0)):
        slots = torch.zeros(n, s, dtype=torch.int64, device=cuda)
        store_pages(*(torch.ones(n, 2, s, 16, device=cuda) for _ in range(2)), kp, vp, slots, scales=(ks, vs))
        assert read_pages(kp, vp, slots, scales=(ks, vs), dtype=torch.float32)[0].shape == (n, 2, s, 16)
    assert torch.equal(kp, before)
