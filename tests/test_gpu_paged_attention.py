"""GPU tests of the attention of one token per request over a paged cache,
against the oracle in fp64; bounds derived in oracle/paged.py."""
from __future__ import annotations

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(lengths, H, K, hd, page, dtype, seed, P=None, sharp=1.0, spare=3):
    """q, pages and table (CPU) for these lengths.  Rows that nobody may see
    hold NaN: pages not handed out, and what follows a request in its last
    page; entries behind a request's pages are ids outside the pool."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    P = P or max(1, max(counts))
    pages = sum(counts) + spare
    ids = torch.randperm(pages, generator=g)
    junk = torch.tensor([-1, pages, 2**31 - 1, -2**31])
    table = junk[torch.randint(4, (len(lengths), P), generator=g)]
    kp, vp = (torch.full((pages, K, page, hd), float("nan")) for _ in range(2))
    at = 0
    for i, n in enumerate(lengths):
        mine = ids[at:at + counts[i]]
        at += counts[i]
        table[i, :counts[i]] = mine
        for c, p in enumerate(mine.tolist()):
            rows = min(page, n - c * page)
            kp[p, :, :rows] = torch.randn(K, rows, hd, generator=g) * sharp
            vp[p, :, :rows] = torch.randn(K, rows, hd, generator=g)
    q = torch.randn(len(lengths), H, hd, generator=g)
    return q.to(dtype), kp.to(dtype), vp.to(dtype), table.to(torch.int32), torch.tensor(lengths, dtype=torch.int32)


def check(case, cuda, scale=None, form=lambda q, k, v, t: (q, k, v, t), out=None):
    from hydra_amd.attention import paged_attention

    q, kp, vp, table, lengths = case
    want, weight = op.attention(q, kp, vp, table, lengths, scale)
    bound = op.attention_bound(q, kp, weight, want, lengths, q.dtype, scale)
    dq, dk, dv, dt = form(q.to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda))
    got = paged_attention(dq, dk, dv, dt, lengths.to(cuda), scale=scale, out=out)
    err = (got.cpu().double() - want).abs()
    assert got.shape == q.shape and got.dtype == q.dtype
    assert bool((err <= bound).all()), f"error {err.max():.3e}, {(err / bound).max():.2f} of the bound"
    return got


EDGES = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,hd,page", [(8, 2, 16, 16), (4, 1, 64, 64), (28, 4, 16, 32), (8, 8, 32, 16), (4, 1, 128, 128),
                                         (6, 2, 32, 64), (1, 1, 256, 16), (16, 1, 64, 16), (9, 1, 48, 256), (2, 1, 8, 16),
                                         (24, 2, 80, 32)])
def test_lengths_and_layouts(cuda, dtype, H, K, hd, page):
    check(make(EDGES, H, K, hd, page, dtype, seed=H * 100 + hd), cuda)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [1, 3, 20, 33, 250])
def test_head_dims_that_no_vector_fits(cuda, dtype, hd):
    check(make([0, 1, 33, 200], 6, 2, hd, 16, dtype, seed=hd), cuda)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,H,K,hd,page", [
    ([5000], 4, 1, 64, 64), ([1, 9000, 3, 0, 2500], 8, 2, 16, 16), ([3001, 17], 8, 8, 32, 32), ([2777], 2, 1, 128, 128),
    ([1999, 1], 3, 1, 256, 4096),
])
def test_long_contexts_are_split(cuda, dtype, lengths, H, K, hd, page):
    check(make(lengths, H, K, hd, page, dtype, seed=sum(lengths)), cuda)


@pytest.mark.parametrize("sharp", [0.0, 30.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_flat_and_sharp_scores(cuda, dtype, sharp):
    """Equal scores, and scores of hundreds: the running maximum."""
    check(make([700, 130], 4, 1, 64, 64, dtype, seed=5, sharp=sharp), cuda)


@pytest.mark.parametrize("N", [300, 2100])
def test_many_requests(cuda, N):
    """A workgroup for each item, without a split."""
    lengths = [(i * 37) % 90 for i in range(N)]
    check(make(lengths, 8, 4, 16, 16, torch.bfloat16, seed=N, P=64), cuda)


@pytest.mark.parametrize("N", [63, 64, 65, 300, 1000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_requests_are_split(cuda, N, dtype):
    """Prefix sums of the requests' rounds in a wave's lanes (64 and fewer) and
    in LDS; runs of requests without keys, a long one among short ones."""
    lengths = [0 if i % 5 == 2 or 20 < i < 40 else (i * 61) % 170 for i in range(N)]
    lengths[N // 2] = 2500
    check(make(lengths, 4, 2, 32, 16, dtype, seed=N, P=160), cuda)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scale(cuda, scale):
    check(make([40, 600], 4, 2, 32, 32, torch.bfloat16, seed=3), cuda, scale=scale)


def test_tables_longer_than_any_request(cuda):
    """The capacity of the table, not the lengths, decides on the split."""
    case = make([3, 200, 0, 65], 4, 2, 64, 16, torch.bfloat16, seed=9, P=4096)
    check(case, cuda)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lengths_and_entries_that_are_wrong(cuda, dtype):
    """Lengths outside the table's reach count to its ends; entries outside
    the pool are not seen; a request that sees nothing gets zeros."""
    q, kp, vp, table, lengths = make([64, 64, 64, 64], 4, 2, 32, 16, dtype, seed=4)
    lengths = torch.tensor([-3, 2**31 - 1, 64, 40], dtype=torch.int32)
    table[2] = torch.tensor([-1, 2**31 - 1, kp.shape[0], -2**31])
    table[3, 1] = -1
    got = check((q, kp, vp, table, lengths), cuda)
    assert not got[0].any() and not got[2].any()


def test_infinities_and_nan_in_what_is_seen(cuda):
    """They reach the requests and heads that see them and no others."""
    from hydra_amd.attention import paged_attention

    q, kp, vp, table, lengths = make([100, 100, 100], 4, 2, 32, 16, torch.bfloat16, seed=8)
    clean = paged_attention(*(t.to(cuda) for t in (q, kp, vp, table, lengths)))
    vp[table[0, 2], 1, 3, 5] = float("nan")
    kp[table[1, 6], 0, 3, 0] = float("nan")
    got = paged_attention(*(t.to(cuda) for t in (q, kp, vp, table, lengths)))
    assert got[0, 2:, 5].isnan().all() and got[1, :2].isnan().all()
    same = torch.ones_like(got, dtype=torch.bool)
    same[0, 2:, 5] = same[1, :2] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(cuda, dtype):
    case = make([70, 0, 900], 6, 2, 32, 32, dtype, seed=11)
    other = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731  rows before heads
    shift = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    wide = lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]]  # noqa: E731
    check(case, cuda, form=lambda q, k, v, t: (q.transpose(0, 1).contiguous().transpose(0, 1), other(k), other(v), t))
    check(case, cuda, form=lambda q, k, v, t: (shift(q), shift(k), shift(v), t))
    check(case, cuda, form=lambda q, k, v, t: (wide(q), wide(k), wide(v), torch.cat([t, t], 1)[:, :t.shape[1]]))
    check(case, cuda, form=lambda q, k, v, t: (q.mT.contiguous().mT, k, v, t))
    buf = torch.full((6, 3, 40), 7.0, dtype=dtype, device=cuda)
    check(case, cuda, out=buf.transpose(0, 1)[..., 4:36])
    assert (buf[..., :4] == 7).all() and (buf[..., 36:] == 7).all()
    inside = case[0].to(cuda)
    got = check((inside.cpu(), *case[1:]), cuda, form=lambda q, k, v, t: (inside, k, v, t), out=inside)
    assert got.data_ptr() == inside.data_ptr()


def test_same_bits_again_and_on_another_stream(cuda):
    from hydra_amd.attention import paged_attention

    case = [t.to(cuda) for t in make([6000, 31, 0, 2000], 8, 2, 64, 64, torch.bfloat16, seed=1)]
    want = paged_attention(*case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = paged_attention(*case)
        b = paged_attention(*case)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


def test_captured_call_follows_the_lengths(cuda):
    """Replays read the lengths and tables of their time; eager work in
    between takes other scratch."""
    from hydra_amd.attention import paged_attention

    q, kp, vp, table, lengths = (t.to(cuda) for t in make([4000, 1500, 64], 4, 1, 64, 64, torch.bfloat16, seed=2))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        paged_attention(q, kp, vp, table, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(paged_attention(q, kp, vp, table, lengths))
    for step in ([4000, 1500, 64], [1, 0, 7], [3999, 64, 0], [100, 1400, 33]):
        lengths.copy_(torch.tensor(step, dtype=torch.int32))
        want = paged_attention(q, kp, vp, table, lengths)
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes (and 2^31 elements), its last pages in
    use."""
    from hydra_amd.attention import paged_attention

    page, K, hd = 4096, 8, 128
    pages = (1 << 32) // (page * K * hd * 2) + 260
    q, kp, vp, table, lengths = make([9000, 100], 8, K, hd, page, torch.bfloat16, seed=6, spare=0)
    small = paged_attention(*(t.to(cuda) for t in (q, kp, vp, table, lengths)))
    n = kp.shape[0]
    far = [torch.empty((pages, K, page, hd), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    for pool, t in zip(far, (kp, vp)):
        pool[pages - n:] = t.to(cuda)
    used = (table >= 0) & (table < n)
    moved = torch.where(used, table + pages - n, -1).to(torch.int32)
    assert far[0].numel() > 2**31
    got = paged_attention(q.to(cuda), *far, moved.to(cuda), lengths.to(cuda))
    assert torch.equal(got, small)


def test_refusals(cuda):
    from hydra_amd.attention import paged_attention

    q, kp, vp, table, lengths = (t.to(cuda) for t in make([20, 3], 4, 2, 16, 16, torch.bfloat16, seed=1))
    for args, text in (((q[0], kp, vp, table, lengths), "q must be"), ((q[..., :8], kp, vp, table, lengths), "q must be"),
                       ((q[:, :3], kp, vp, table, lengths), "multiple"), ((q.float(), kp, vp, table, lengths), "dtype"),
                       ((q, kp, vp.half(), table, lengths), "alike"), ((q, kp, vp, table[:1], lengths), "table"),
                       ((q, kp, vp, table, lengths.long()), "lengths"), ((q, kp, vp, table, lengths[:1]), "lengths"),
                       ((q, kp, vp, table[:, :0], lengths), "without pages"),
                       ((q, kp[:, :, :8], vp[:, :, :8], table, lengths), "power of two"),
                       ((q, kp, vp, table, lengths, None, q[:, :2]), "out must be"),
                       ((q, kp, vp, table, lengths, None, q[:1].expand(2, 4, 16)), "overlap"),
                       ((q, kp, vp, table, lengths, None, q.mT.contiguous().mT), "unit stride")):
        with pytest.raises(ValueError, match=text):
            paged_attention(*args)
    with pytest.raises(TypeError, match="dtype"):
        paged_attention(q.double(), kp.double(), vp.double(), table, lengths)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention(q.clone().requires_grad_(), kp, vp, table, lengths)
    with torch.no_grad():
        paged_attention(q.clone().requires_grad_(), kp, vp, table, lengths)
    assert paged_attention(q[:0], kp, vp, table[:0], lengths[:0]).shape == (0, 4, 16)
