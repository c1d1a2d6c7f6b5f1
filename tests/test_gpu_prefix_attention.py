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


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scale(cuda, dtype, eight, scale):
    """Also of groups whose rows go through each form."""
    Case([[90, 200, 83], [40, 45, 39]], [83, 39], 4, 2, 32, 16, dtype, eight, seed=3).check(cuda, scale=scale)
    Case([[300 + i for i in range(20)]], [300], 8, 2, 64, 64, dtype, eight, seed=4).check(cuda, scale=scale)


@pytest.mark.parametrize("sharp", [0.0, 30.0])
@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", DTYPES)
def test_flat_and_sharp_scores(cuda, dtype, eight, sharp):
    """Equal scores, and scores of hundreds: the running maximum, which moves late."""
    Case([[700 + 3 * i for i in range(24)]], [690], 8, 2, 64, 64, dtype, eight, seed=5, sharp=sharp).check(cuda)
    Case([[700, 130], [401, 420]], [130, 400], 4, 1, 64, 16, dtype, eight, seed=6, sharp=sharp).check(cuda)


@pytest.mark.parametrize("page", [16, 32, 64, 4096])
@pytest.mark.parametrize("hd", [32, 64, 128, 256, 48, 8])
def test_pages_of_all_sizes(cuda, page, hd):
    """A tile of the direct loads within a page and over several."""
    prefix = 1000
    Case([[prefix + (i * 7) % 90 for i in range(40)]], [prefix], 4, 1, hd, page, torch.bfloat16, seed=hd + page).check(cuda)


def test_growing_scores(cuda):
    """Keys whose scores grow along the context by more than the maximum lags behind
    in each tile, and by less."""
    for step in (0.05, 2.0):
        case = Case([[1500 + i for i in range(40)]], [1500], 4, 1, 64, 64, torch.bfloat16, seed=9)
        case.q[:] = 1.0
        grow = (torch.arange(1540) * step / 64).to(torch.bfloat16)
        for n in range(40):
            for t in range(int(case.lengths[n])):
                case.kp[int(case.table[n, t // 64]), 0, t % 64] = grow[t]
        case.k64 = case.kp
        case.check(cuda)


@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_and_entries_that_are_wrong(cuda, dtype, eight):
    """Lengths and prefixes outside the table's reach count to its ends; entries
    outside the pool are not seen, in prefixes and behind them; a request that sees
    nothing gets zeros."""
    case = Case([[64, 64, 64, 64], [64, 64, 64, 64]], [0, 32], 4, 2, 32, 16, dtype, eight, seed=4)
    case.lengths[:4] = torch.tensor([-3, 2**31 - 1, 64, 40])
    case.table[2] = torch.tensor([-1, 2**31 - 1, case.kp.shape[0], -2**31])
    case.table[3, 1] = -1
    case.shared[0] = -7
    case.table[4:, 1] = 2**30  # of the prefix, in every row
    case.table[6, 3] = -5
    case.table[7, 2:] = -1
    got = case.check(cuda)
    assert not got[0].any() and not got[2].any()
    case.shared[1] = 2**31 - 1  # counts to the end of the table: all 64
    for c in range(4):
        case.table[4:, c] = case.table[4, c]
    case.check(cuda)
    many = Case([[64] * 40], [48], 4, 1, 32, 16, dtype, eight, seed=5)
    many.table[:, 0], many.table[:, 2] = -1, many.kp.shape[0]
    many.check(cuda)
    many.table[:, 1] = 2**31 - 1
    many.lengths[:] = 48
    assert not many.check(cuda).any()


@pytest.mark.parametrize("eight", [None, *EIGHT])
def test_nan_reaches_who_sees_it(cuda, eight):
    """A NaN row of the prefix: all requests of the group that have it; one behind:
    its request alone; of a key: its heads' scores."""
    for W in (3, 20):
        case = Case([[100] * W, [100] * W], [70, 70], 4, 2, 32, 16, torch.bfloat16, eight, seed=8)
        clean = case.call(cuda)

        def spoil(x, s, page, head, row):
            if eight is None:
                x[page, head, row, 5] = float("nan")
            else:
                s[page, head, row] = float("nan")

        ks, vs = case.scales or (None, None)
        spoil(case.vp, vs, case.table[0, 2], 1, 3)
        spoil(case.kp, ks, case.table[W, 6], 0, 3)
        got = case.call(cuda)
        same = torch.ones_like(got, dtype=torch.bool)
        assert got[:W, 2:, 5].isnan().all() and got[W, :2].isnan().all()
        same[:W, 2:, 5 if eight is None else slice(None)] = False
        same[W, :2] = False
        assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_that_see_nothing_of_infinities(cuda, dtype):
    """Keys of -inf alone: zeros, as without them."""
    case = Case([[40] * 20, [40] * 20], [32, 32], 4, 2, 32, 16, dtype, seed=2)
    case.q[:] = case.q.abs() + 0.5
    case.kp[:] = float("-inf")
    assert not case.call(cuda).any()


@pytest.mark.parametrize("N,W", [(1023, 1), (1025, 1), (2100, 1), (1026, 2), (2050, 1025), (3000, 1500)])
@pytest.mark.parametrize("eight", [None, torch.int8])
def test_many_requests(cuda, N, W, eight):
    """More than one launch takes; groups of more than that."""
    if eight is None and W == 1:
        pytest.skip("no groups: the attention of pages of the queries' type")
    lengths = [[20 + (i * 37) % 70 if i % 9 else 5 for i in range(g * W, g * W + W)] for g in range(N // W)]
    Case(lengths, [20] * (N // W), 4, 2, 16, 16, torch.bfloat16, eight, seed=N, P=12).check(cuda, shared=W > 1)


@pytest.mark.parametrize("N", [63, 64, 65, 300])
def test_groups_with_and_without_a_prefix(cuda, N):
    """Plans of few requests in one wave and of many; groups of which nobody has the
    prefix, or which have none."""
    W = {63: 9, 64: 16, 65: 13, 300: 6}[N]
    lengths = [[(i * 61) % 170 + (400 if g % 3 == 0 else 0) for i in range(g * W, g * W + W)] for g in range(N // W)]
    Case(lengths, [[400, 0, 600][g % 3] for g in range(N // W)], 4, 2, 32, 16, torch.float16, seed=N, P=64).check(cuda)


@pytest.mark.parametrize("eight", [None, *EIGHT])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(cuda, dtype, eight):
    """Queries and pages of other strides, aligned and not; out with gaps, and q itself."""
    for W, step in ((3, 16), (30, 16), (3, 1), (30, 1)):
        case = Case([[50 + i for i in range(W)]], [47], 6, 2, 32, 16, dtype, eight, seed=W)

        def form(name, t, step=step):
            if name == "table":
                wide = torch.full((t.shape[0], t.shape[1] + 5), -1, dtype=t.dtype, device=t.device)
                wide[:, :t.shape[1]] = t
                return wide[:, :t.shape[1]]
            if name == "scales":
                return t.transpose(0, 1).contiguous().transpose(0, 1)
            raw = t.view(torch.int8) if t.element_size() == 1 else t
            wide = torch.zeros(*raw.shape[:-2], raw.shape[-2] * 2, raw.shape[-1] + step, dtype=raw.dtype, device=t.device)
            cut = wide[..., ::2, step:]
            cut.copy_(raw)
            return cut.view(t.dtype)

        case.check(cuda, form=form)
        out = torch.full((W, 6, 50), 9.0, dtype=dtype, device=cuda)
        case.check(cuda, out=out[:, :, 7:39])
        assert (out[:, :, :7] == 9).all() and (out[:, :, 39:] == 9).all()
        from hydra_amd.attention import paged_attention

        q = case.q.to(cuda)
        scales = None if case.scales is None else [s.to(cuda) for s in case.scales]
        want = case.call(cuda)
        got = paged_attention(q, case.kp.to(cuda), case.vp.to(cuda), case.table.to(cuda), case.lengths.to(cuda), out=q,
                              scales=scales, shared=case.shared.to(cuda))
        assert got is q and torch.equal(q, want)
        # transposed queries, and a request vector with a stride
        qt = case.q.to(cuda).transpose(1, 2).contiguous().transpose(1, 2)
        lengths = torch.stack([case.lengths, case.lengths], 1).to(cuda)[:, 0]
        got = paged_attention(qt, case.kp.to(cuda), case.vp.to(cuda), case.table.to(cuda), lengths, scales=scales,
                              shared=case.shared.to(cuda))
        assert torch.equal(got, want)


def test_same_bits(cuda):
    """No sum depends on which workgroup is first."""
    for W, eight in ((4, None), (40, None), (40, torch.int8)):
        case = Case([[2000 + 13 * i for i in range(W)]], [1990], 8, 2, 64, 64, torch.bfloat16, eight, seed=W)
        want = case.call(cuda)
        for _ in range(5):
            assert torch.equal(case.call(cuda), want)


def test_groups_of_one(cuda):
    """Every request a group of its own: the attention without groups."""
    from hydra_amd.attention import paged_attention

    case = Case([[40], [90], [3]], [32, 64, 3], 4, 2, 32, 16, torch.bfloat16, seed=1)
    args = [t.to(cuda) for t in (case.q, case.kp, case.vp, case.table, case.lengths)]
    assert torch.equal(case.call(cuda), paged_attention(*args))


def test_another_stream(cuda):
    case = Case([[700 + i for i in range(24)]], [690], 8, 2, 64, 64, torch.bfloat16, torch.int8, seed=5)
    want = case.call(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = case.call(cuda)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(cuda):
    from hydra_amd.attention import paged_attention

    case = Case([[40, 50], [33, 60]], [32, 16], 4, 2, 32, 16, torch.bfloat16, torch.int8, seed=1)
    q, kp, vp, table, lengths, shared = (t.to(cuda) for t in (case.q, case.kp, case.vp, case.table, case.lengths, case.shared))
    ks, vs = (s.to(cuda) for s in case.scales)
    kb, vb = (torch.zeros(kp.shape, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    call = lambda *a, **kw: paged_attention(*a, **kw)  # noqa: E731
    for error, text, args, kw in (
            (ValueError, "need scales", (q, kp, vp, table, lengths), {}),
            (ValueError, "need scales", (q, kp, vp, table, lengths), dict(shared=shared)),
            (ValueError, "scales are of pages of 8 bits", (q, kb, vb, table, lengths), dict(scales=(ks, vs))),
            (ValueError, "scales must be", (q, kp, vp, table, lengths), dict(scales=(ks.double(), vs))),
            (ValueError, "scales must be", (q, kp, vp, table, lengths), dict(scales=(ks, vs[:-1]))),
            (ValueError, "overlap", (q, kp, vp, table, lengths), dict(scales=(ks, vs[:1].expand(vs.shape)))),
            (ValueError, "no multiple of 3 groups", (q, kb, vb, table, lengths), dict(shared=lengths[:3])),
            (ValueError, "no multiple of 0 groups", (q, kb, vb, table, lengths), dict(shared=lengths[:0])),
            (ValueError, "shared must be a int32", (q, kb, vb, table, lengths), dict(shared=shared.long())),
            (ValueError, "share a dtype", (q.half(), kb, vb, table, lengths), dict(shared=shared)),
            (ValueError, "no multiple of 2 key heads", (q[:, :3], kb, vb, table, lengths), dict(shared=shared)),
            (ValueError, "out must be", (q, kb, vb, table, lengths), dict(shared=shared, out=q.float())),
            (ValueError, "lengths must be", (q, kb, vb, table, lengths[:3]), dict(shared=shared)),
            (TypeError, "dtype", (q.double(), kp, vp, table, lengths), dict(scales=(ks, vs))),
            (RuntimeError, "GPU tensors only", (q, kb, vb, table, lengths), dict(shared=shared.cpu())),
            (RuntimeError, "GPU tensors only", (q, kp, vp, table, lengths), dict(scales=(ks.cpu(), vs))),
            (RuntimeError, "no gradient", (q.clone().requires_grad_(), kb, vb, table, lengths), dict(shared=shared))):
        with pytest.raises(error, match=text):
            call(*args, **kw)


@pytest.mark.parametrize("form", ["shared few", "shared many", "shared many, pages of 16", "8 bits", "fp32"])
def test_pools_past_32_bits(cuda, form):
    """Pages more than 2^32 bytes into the pool, of every kernel that walks them."""
    from hydra_amd.attention import copy_pages, paged_attention, read_pages, store_pages

    page = 16 if "16" in form else 4096
    K, hd = 1, 256
    dtype = torch.float32 if form == "fp32" else torch.bfloat16
    e = 1 if form == "8 bits" else dtype.itemsize
    pages = (1 << 32) // (page * hd * e) + 40
    free, _ = torch.cuda.mem_get_info()
    if free < 3 * pages * page * hd * e:
        pytest.skip("too little memory")
    g = torch.Generator().manual_seed(1)
    W = 2 if form in ("shared few", "8 bits", "fp32") else 70
    n = 150
    P = -(-n // page)
    # each request its own page behind the prefix's; a small pool with the same rows to compare with
    case = Case([[n] * W], [n // 2 // page * page if page == 16 else n // 2], 1, K, hd, page, dtype,
                torch.int8 if form == "8 bits" else None, seed=2)
    used = case.kp.shape[0]
    far = torch.arange(pages - used, pages)
    table = torch.where((case.table >= 0) & (case.table < used), far[case.table.long().clamp(0, used - 1)].to(torch.int32), -1)
    kp, vp = (torch.empty((pages, K, page, hd), dtype=t.dtype, device=cuda) for t in (case.kp, case.vp))
    kp[-used:], vp[-used:] = case.kp.to(cuda), case.vp.to(cuda)
    scales = small = None
    if case.scales is not None:
        scales = [torch.empty((pages, K, page), device=cuda) for _ in range(2)]
        for s, c in zip(scales, case.scales):
            s[-used:] = c.to(cuda)
        small = [s.to(cuda) for s in case.scales]
    shared = None if form == "8 bits" else case.shared.to(cuda)
    q, lengths = case.q.to(cuda), case.lengths.to(cuda)
    want = paged_attention(q, case.kp.to(cuda), case.vp.to(cuda), case.table.to(cuda), lengths, scales=small, shared=shared)
    assert torch.equal(paged_attention(q, kp, vp, table.to(cuda), lengths, scales=scales, shared=shared), want)
    # rows written, read and copied there
    slots = ((pages - 1) * page + torch.tensor([[3, 9]])).to(cuda)
    rows = torch.randn(1, K, 2, hd, generator=g).to(torch.bfloat16 if scales else dtype).to(cuda)
    store_pages(rows, rows, kp, vp, slots, scales=scales)
    copy_pages(kp, vp, *(torch.tensor([p], dtype=torch.int32, device=cuda) for p in (pages - 1, pages - 2)), scales=scales)
    a, _ = read_pages(kp, vp, slots, scales=scales, dtype=dtype)
    b, _ = read_pages(kp, vp, slots - page, scales=scales, dtype=dtype)
    assert torch.equal(a, b)
    if scales is None:
        assert torch.equal(a, rows)
    else:
        x, s = op.quantise(rows.cpu(), torch.int8)
        assert (a.cpu().double() - x * s.double()[..., None]).abs().max() <= 2.0 ** -8 * rows.abs().max()
