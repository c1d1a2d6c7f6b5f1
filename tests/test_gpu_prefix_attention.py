"""GPU tests of the attention of one token per request over pages of 8 bits and
over prefixes that groups of requests share, against the oracle in fp64; bounds
derived in oracle/paged.py."""
from __future__ import annotations

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EIGHT = [torch.int8, torch.float8_e4m3fn]


def eight_bits(x, dtype):
    """Rows x in 8 bits, with scales that their values fill (any scales do here)."""
    top = x.abs().amax(-1).clamp(min=1e-6)
    if dtype == torch.int8:
        scales = top / 127
        return (x / scales[..., None]).round().to(torch.int8), scales
    scales = top / 448
    return (x / scales[..., None]).clamp(-448, 448).to(dtype), scales


class Case:
    """q, pages, table (CPU) of groups of requests: lengths [groups][W], prefixes
    [groups].  Requests as long as their prefix hold its full pages in common
    and a copy of the rest; others pages of their own.  Rows that nobody may see
    hold NaN (in 8 bits their scales do); entries behind a request's pages are ids
    outside the pool."""

    def __init__(self, lengths, prefixes, H, K, hd, page, dtype, eight=None, seed=0, P=None, sharp=1.0):
        g = torch.Generator().manual_seed(seed)
        flat = [n for row in lengths for n in row]
        P = P or max(1, -(-max(flat) // page))
        count = sum(-(-n // page) for n in flat) + sum(-(-n // page) for n in prefixes) + 2
        ids = iter(torch.randperm(count, generator=g).tolist())
        kp, vp = (torch.full((count, K, page, hd), float("nan")) for _ in range(2))
        junk = torch.tensor([-1, count, 2**31 - 1, -2**31])
        table = junk[torch.randint(4, (len(flat), P), generator=g)]
        rand = lambda n, s: torch.randn(K, n, hd, generator=g) * s  # noqa: E731

        def put(page_id, first, k, v):
            kp[page_id, :, first:first + k.shape[1]] = k
            vp[page_id, :, first:first + k.shape[1]] = v

        n = 0
        for row, prefix in zip(lengths, prefixes):
            k0, v0 = rand(prefix, sharp), rand(prefix, 1.0)
            common = [next(ids) for _ in range(prefix // page)]
            for c, p in enumerate(common):
                put(p, 0, k0[:, c * page:(c + 1) * page], v0[:, c * page:(c + 1) * page])
            for length in row:
                mine = common if length >= prefix else []
                k, v = rand(length, sharp), rand(length, 1.0)
                if length >= prefix:
                    k[:, :prefix], v[:, :prefix] = k0, v0
                for c in range(-(-length // page)):
                    if c < len(mine):
                        table[n, c] = mine[c]
                        continue
                    table[n, c] = next(ids)
                    put(int(table[n, c]), 0, k[:, c * page:(c + 1) * page], v[:, c * page:(c + 1) * page])
                n += 1
        self.q = torch.randn(len(flat), H, hd, generator=g).to(dtype)
        self.table, self.lengths = table.to(torch.int32), torch.tensor(flat, dtype=torch.int32)
        self.shared = torch.tensor(prefixes, dtype=torch.int32)
        self.dtype, self.eight, self.scales = dtype, eight, None
        self.kp, self.vp = kp.to(dtype), vp.to(dtype)
        self.k64, self.v64 = self.kp, self.vp
        if eight is not None:
            unseen = kp[..., 0].isnan()
            self.scales = []
            for name in ("kp", "vp"):
                x, s = eight_bits(torch.nan_to_num(getattr(self, name).float()), eight)
                s[unseen] = float("nan")
                setattr(self, name, x)
                self.scales.append(s)
            self.k64, self.v64 = (op.dequantise(x, s) for x, s in zip((self.kp, self.vp), self.scales))

    def call(self, cuda, scale=None, out=None, shared=True, form=lambda name, t: t):
        from hydra_amd.attention import paged_attention

        q, kp, vp, table = (form(n, getattr(self, n).to(cuda)) for n in ("q", "kp", "vp", "table"))
        scales = None if self.scales is None else [form("scales", s.to(cuda)) for s in self.scales]
        return paged_attention(q, kp, vp, table, self.lengths.to(cuda), scale=scale, out=out, scales=scales,
                               shared=self.shared.to(cuda) if shared else None)

    def bound(self, scale=None):
        want, weight = op.attention(self.q, self.k64, self.v64, self.table, self.lengths, scale)
        bound = op.attention_bound(self.q, self.k64, weight, want, self.lengths, self.dtype, scale)
        return want, bound + op.two_term_bound(weight, self.v64, self.lengths,
                                               self.eight or self.dtype, self.dtype)

    def check(self, cuda, scale=None, **kw):
        want, bound = self.bound(scale)
        got = self.call(cuda, scale=scale, **kw)
        err = (got.cpu().double() - want).abs()
        assert got.shape == self.q.shape and got.dtype == self.dtype
        assert bool((err <= bound).all()), f"error {err.max():.3e}, {(err / bound).max():.2f} of the bound"
        return got


EDGES = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513]


@pytest.mark.parametrize("eight", EIGHT)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,hd,page", [(8, 2, 16, 16), (4, 1, 64, 64), (28, 4, 16, 32), (8, 8, 32, 16), (4, 1, 128, 128),
                                         (1, 1, 256, 16), (40, 2, 64, 16), (9, 1, 48, 256), (24, 2, 80, 32)])
def test_eight_bits(cuda, eight, dtype, H, K, hd, page):
    Case([[n] for n in EDGES], [0] * len(EDGES), H, K, hd, page, dtype, eight, seed=H + hd).check(cuda, shared=False)


@pytest.mark.parametrize("eight", EIGHT)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,H,K,hd,page", [([5000], 4, 1, 64, 64), ([1, 9000, 3, 0, 2500], 8, 2, 16, 16),
                                                 ([2777], 2, 1, 128, 128), ([1999, 1], 3, 1, 256, 4096)])
def test_eight_bits_of_long_contexts(cuda, eight, dtype, lengths, H, K, hd, page):
    Case([[n] for n in lengths], [0] * len(lengths), H, K, hd, page, dtype, eight, seed=sum(lengths)).check(cuda, shared=False)


@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,hd,page", [(8, 2, 16, 16), (4, 1, 64, 64), (28, 4, 32, 32), (4, 4, 128, 16), (3, 1, 256, 64)])
def test_shared_prefixes(cuda, eight, dtype, H, K, hd, page):
    """Prefixes that end inside a page and a 16, of nothing, longer than some
    of their requests; requests that end with the prefix."""
    lengths = [[33, 40, 161], [200, 200, 17], [5, 0, 1], [300, 260, 259], [0, 0, 0], [64, 65, 128], [15, 14, 16]]
    Case(lengths, [33, 200, 0, 260, 7, 64, 15], H, K, hd, page, dtype, eight, seed=hd).check(cuda)


@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W,H,K,hd,prefix", [(2, 4, 1, 64, 3000), (9, 8, 2, 64, 2048), (40, 8, 2, 16, 1111), (70, 8, 8, 32, 700),
                                             (33, 12, 2, 128, 600), (20, 16, 2, 256, 400)])
def test_rows_of_a_prefix(cuda, eight, dtype, W, H, K, hd, prefix):
    """Few rows (waves in turn) and many (rows of their own, more than one block)."""
    lengths = [[prefix + (i * 29) % 131 for i in range(W)], [prefix // 2 + i * (i % 2) for i in range(W)]]
    Case(lengths, [prefix, prefix // 2], H, K, hd, 32, dtype, eight, seed=W).check(cuda)
