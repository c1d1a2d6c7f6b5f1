"""CPU checks of the entry points for pages of 8 bits, shared prefixes, beams and
forks: what the host can see wrong is refused before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 4096  # an address that a refused call never uses


def st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def refused(text, call, **kw):
    with pytest.raises(ValueError, match=text):
        call(**kw)


def test_prefix_attention():
    from hydra_amd import _lib

    def call(groups=1, N=2, H=4, K=2, hd=16, P=4, page=16, pages=8, rs=4, q=FAKE, ks=FAKE, shared=FAKE, last=1, row=None,
             dtype=1, of=16, size=1 << 40, ws=FAKE):
        row = hd if row is None else row
        q3, p4, s3 = st(H * hd, hd, last), st(K * page * hd, page * hd, row, 1), st(K * page, page, 1)
        _lib.call("hydra_prefix_attn", q, FAKE, FAKE, ks, FAKE, FAKE, FAKE, rs, FAKE, shared, groups, N, H, K, hd, P, page,
                  pages, q3, p4, p4, s3, s3, st(H * hd, hd, 1), ctypes.c_float(1.0), dtype, of, ws, size, None)

    for kw, text in ((dict(H=3), "multiple of n_kv"), (dict(hd=257), "at most 256"), (dict(hd=0), "bad size"),
                     (dict(groups=-1), "bad size"), (dict(groups=2, N=3), "multiple of groups"), (dict(dtype=7), "unknown dtype"),
                     (dict(of=2), "of 8 bits"), (dict(of=3), "of 8 bits"), (dict(of=1, groups=0), "need groups"),
                     (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(pages=0), "number of pages"),
                     (dict(pages=1 << 31), "number of pages"), (dict(rs=3), "row stride"), (dict(q=None), "null"),
                     (dict(ks=None), "null"), (dict(shared=None), "null"), (dict(last=2), "unit stride"),
                     (dict(row=1 << 40), "too far apart"), (dict(row=1 << 62), "too far apart"), (dict(row=-1), "too far apart"),
                     (dict(P=1 << 27, rs=1 << 27), "too large"), (dict(N=1 << 40, groups=1 << 20), "too large"),
                     (dict(N=1 << 62, groups=0), "too large"), (dict(H=1 << 20, K=1 << 20), "too large"),
                     (dict(P=1 << 26, rs=1 << 26, H=1 << 12, K=1 << 12), "too large"),
                     (dict(size=0), "workspace"), (dict(ws=None), "workspace"), (dict(ws=8), "workspace")):
        refused(text, call, **kw)
    call(N=0, groups=0)  # nothing to do
    call(N=0, groups=3)


def test_prefix_attention_workspace():
    from hydra_amd import _lib

    need = ctypes.c_int64(0)
    ask = lambda *a: (_lib.call("hydra_prefix_attn_workspace", *a, ctypes.byref(need)), need.value)[1]  # noqa: E731
    assert ask(0, 1, 4, 1, 64, 8, 64, 1, 16) == 0          # a workgroup for the item
    assert ask(0, 1, 4, 1, 64, 512, 64, 1, 16) > 0         # its keys dealt out
    assert ask(0, 5000, 4, 1, 64, 512, 64, 1, 17) == 0     # requests enough
    assert ask(8, 32, 8, 2, 64, 32, 64, 1, 1) > 0
    assert ask(0, 0, 4, 1, 64, 8, 64, 1, 16) == 0
    with pytest.raises(ValueError, match="null"):
        _lib.call("hydra_prefix_attn_workspace", 1, 2, 4, 2, 16, 4, 16, 1, 1, None)


def rows8(entry, hd=16, N=1, K=1, S=4, pages=4, page=16, R=1, rows=None, dtype=1, of=16, k=FAKE, ks=FAKE, last=1, scale_last=1,
          row=None):
    from hydra_amd import _lib

    r4, p4, s3 = st(K * S * hd, S * hd, hd, last), st(K * page * hd, page * hd, hd if row is None else row, 1), st(K * page, page, scale_last)
    if entry == "hydra_page_store8":
        _lib.call(entry, k, FAKE, FAKE, FAKE, ks, FAKE, FAKE, R, rows, N, K, S, hd, pages, page, r4, r4, p4, p4, s3, s3, dtype, of, None)
    else:
        _lib.call(entry, FAKE, FAKE, ks, FAKE, k, FAKE, FAKE, R, rows, N, K, S, hd, pages, page, p4, p4, s3, s3, r4, r4, dtype, of, None)


@pytest.mark.parametrize("entry", ["hydra_page_store8", "hydra_page_read"])
def test_rows_of_eight_bits(entry):
    for kw, text in ((dict(hd=0), "bad size"), (dict(pages=0), "bad size"), (dict(R=0), "fewer rows"), (dict(page=48), "power of two"),
                     (dict(dtype=9), "unknown dtype"), (dict(of=18), "8 bits"), (dict(hd=257), "too large"), (dict(K=65536), "too large"),
                     (dict(N=1 << 31, R=1 << 31), "too large"), (dict(S=1 << 31), "too large"), (dict(k=None), "null"),
                     (dict(ks=None), "null"), (dict(last=2), "unit stride"), (dict(scale_last=2), "unit stride"),
                     (dict(row=-16), "too far apart"), (dict(row=1 << 33), "too far apart")):
        refused(text, lambda **k: rows8(entry, **k), **kw)
    rows8(entry, N=0)
    rows8(entry, S=0)
    if entry == "hydra_page_store8":
        refused("8 bits", lambda **k: rows8(entry, **k), of=1)


def test_forks_and_copies():
    from hydra_amd import _lib

    def fork(N=2, P=4, rs=4, page=16, pages=8, cap=8, parents=FAKE, ws=FAKE, size=1 << 40):
        _lib.call("hydra_page_fork", parents, FAKE, FAKE, rs, FAKE, cap, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, N, P, page, pages, ws,
                  size, None)

    for kw, text in ((dict(N=0), "bad size"), (dict(P=0), "bad size"), (dict(pages=0), "bad size"), (dict(N=8193), "8192"),
                     (dict(P=1 << 31, rs=1 << 31), "too large"), (dict(N=8192, P=1 << 19, rs=1 << 19), "too large"),
                     (dict(pages=1 << 31), "too large"), (dict(page=20), "power of two"), (dict(rs=3), "row stride"),
                     (dict(P=1 << 27, rs=1 << 27), "too large"), (dict(cap=-1), "too large"), (dict(parents=None), "null"),
                     (dict(ws=None), "workspace"), (dict(size=0), "workspace"), (dict(ws=2), "workspace")):
        refused(text, fork, **kw)

    def copy(N=1, K=1, hd=16, pages=4, page=16, e=2, kp=FAKE, ks=None, vs=None, last=1, row=None, scale_last=1):
        p4, s3 = st(K * page * hd, page * hd, hd if row is None else row, last), st(K * page, page, scale_last)
        _lib.call("hydra_page_copy", kp, FAKE, ks, vs, FAKE, FAKE, N, K, hd, pages, page, p4, p4, s3, s3, e, None)

    for kw, text in ((dict(N=-1), "bad size"), (dict(hd=0), "bad size"), (dict(page=17), "power of two"), (dict(e=3), "1, 2 or 4"),
                     (dict(K=65536), "too large"), (dict(hd=65536, K=4096), "too large"), (dict(pages=1 << 31), "too large"),
                     (dict(kp=None), "null"), (dict(ks=FAKE), "null"), (dict(vs=FAKE), "null"), (dict(last=2), "unit stride"),
                     (dict(ks=FAKE, vs=FAKE, scale_last=3), "unit stride"), (dict(row=1 << 32), "too far apart")):
        refused(text, copy, **kw)
    copy(N=0)

    def take(N=2, row=16, stride=16, x=FAKE):
        _lib.call("hydra_rows_take", x, stride, row, FAKE, N, None)

    for kw, text in ((dict(N=-1), "bad size"), (dict(N=8193), "8192"), (dict(row=-1), "bad size"), (dict(stride=8), "overlap"),
                     (dict(row=1 << 41, stride=1 << 41), "too large"), (dict(x=None), "null"), (dict(row=(1 << 40) - 1, stride=(1 << 40) - 1), "too large")):
        refused(text, take, **kw)
    take(N=1)
    take(row=0)


def test_beam_selection():
    from hydra_amd import _lib

    def call(B=1, W=2, V=100, n=4, rs=100, dtype=1, x=FAKE, ws=FAKE, size=1 << 40):
        _lib.call("hydra_beam_select", x, rs, FAKE, B, W, V, n, FAKE, FAKE, FAKE, FAKE, dtype, ws, size, None)

    for kw, text in ((dict(B=-1), "bad size"), (dict(W=0), "bad size"), (dict(V=0, rs=0), "bad size"), (dict(n=0), "bad size"),
                     (dict(W=1025), "1024 beams"), (dict(n=129), "128 continuations"), (dict(V=2, rs=2, n=5), "beams x vocabulary"),
                     (dict(V=1 << 31, rs=1 << 31), "2\\^31"), (dict(W=1024, V=1 << 22, rs=1 << 22), "2\\^31"), (dict(B=1 << 31), "too large"),
                     (dict(B=1 << 62), "too large"), (dict(dtype=5), "unknown dtype"), (dict(rs=99), "row stride"), (dict(x=None), "null"),
                     (dict(x=FAKE + 1), "aligned"), (dict(ws=None), "workspace"), (dict(ws=FAKE + 8), "workspace"), (dict(size=8), "workspace")):
        refused(text, call, **kw)
    call(B=0)


def test_python_entry_points_take_gpu_tensors_only():
    from hydra_amd.attention import PagePool, copy_pages, fork_pages, paged_attention, read_pages, store_pages, take_rows
    from hydra_amd.kernels import beam_select

    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    p = torch.zeros(4, 1, 16, 16, dtype=torch.int8)
    s, rows, slots = torch.ones(4, 1, 16), torch.zeros(1, 1, 3, 16), torch.zeros(1, 3, dtype=torch.long)
    for call in (lambda: store_pages(rows, rows, p, p, slots, scales=(s, s)), lambda: read_pages(p, p, slots, scales=(s, s), dtype=torch.float32),
                 lambda: paged_attention(rows[0].transpose(0, 1)[:2], p, p, t, i, scales=(s, s)),
                 lambda: paged_attention(rows[0].transpose(0, 1)[:2], p.float(), p.float(), t, i, shared=i[:1]),
                 lambda: fork_pages(i, i, t, i, i[:1], torch.zeros(9, dtype=torch.int32), 16), lambda: copy_pages(p, p, i, i, scales=(s, s)),
                 lambda: take_rows(rows[0, 0, :2], i), lambda: beam_select(torch.zeros(4, 9), torch.zeros(2, 2), 3)):
        with pytest.raises(RuntimeError, match="GPU tensors only"):
            call()
    with pytest.raises(ValueError, match="8192"):
        PagePool(8193, 64, 4, 16, device="cpu", sharing=True)
    with pytest.raises(RuntimeError, match="sharing=True"):
        PagePool(2, 64, 4, 16, device="cpu").fork(i)
