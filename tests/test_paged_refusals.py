"""CPU checks of the page and paged-attention entry points of the C ABI: what
the host can see wrong is refused before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 4096  # an address that a refused call never uses


def st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def plan(N=2, P=4, width=1, page=16, rs=4, cap=8, lengths_out=FAKE * 2, free_out=FAKE * 3):
    from hydra_amd import _lib

    _lib.call("hydra_page_plan", FAKE, FAKE, FAKE, rs, FAKE, cap, FAKE, FAKE, lengths_out, FAKE, FAKE, FAKE, free_out,
              N, P, width, page, 0, None)


@pytest.mark.parametrize("page", [0, 1, 8, 15, 24, 48, 8192, -16])
def test_page_size_is_a_power_of_two_in_range(page):
    from hydra_amd import _lib

    with pytest.raises(ValueError, match="power of two"):
        plan(page=page)
    with pytest.raises(ValueError, match="power of two"):
        _lib.call("hydra_page_release", FAKE, FAKE, FAKE, 4, FAKE, 8, FAKE, 2, 4, page, None)
    s = st(1, 1, 1, 1)
    with pytest.raises(ValueError, match="power of two"):
        _lib.call("hydra_page_store", FAKE, FAKE, FAKE, FAKE, FAKE, 1, None, 1, 1, 1, 16, 4, page, s, s, s, s, 1, None)
    need = ctypes.c_int64(0)
    with pytest.raises(ValueError, match="power of two"):
        _lib.call("hydra_paged_attn_workspace", 1, 1, 1, 16, 4, page, 1, ctypes.byref(need))


def test_plan_refusals():
    with pytest.raises(ValueError, match="bad size"):
        plan(N=0)
    with pytest.raises(ValueError, match="bad size"):
        plan(width=0)
    with pytest.raises(ValueError, match="row stride"):
        plan(rs=3)
    with pytest.raises(ValueError, match="too large"):
        plan(N=1 << 20, P=1 << 12, rs=1 << 12)
    with pytest.raises(ValueError, match="too large"):
        plan(P=1 << 28, rs=1 << 28)
    with pytest.raises(ValueError, match="null"):
        plan(lengths_out=None)
    with pytest.raises(ValueError, match="one workgroup"):
        plan(N=300, lengths_out=FAKE)
    with pytest.raises(ValueError, match="one workgroup"):
        plan(N=2, width=4097, free_out=FAKE)


def test_in_place_rule():
    from hydra_amd import _lib

    ask = lambda n, w: _lib.query("hydra_page_plan_in_place", n, w)  # noqa: E731
    assert ask(1, 1) == ask(256, 1) == ask(256, 16) == ask(1, 4096) == ask(2, 2048) == 1
    assert ask(257, 1) == ask(256, 17) == ask(1, 4097) == ask(0, 1) == ask(1, 0) == 0


def test_paged_attention_refusals():
    from hydra_amd import _lib

    def call(N=1, H=4, K=2, hd=16, P=4, page=16, pages=8, rs=4, q=FAKE, last=1, dtype=1, size=1 << 40, ws=FAKE):
        q3, p4 = st(H * hd, hd, last), st(K * page * hd, page * hd, hd, 1)
        _lib.call("hydra_paged_attn", q, FAKE, FAKE, FAKE, FAKE, rs, FAKE, N, H, K, hd, P, page, pages, q3, p4, p4,
                  st(H * hd, hd, 1), ctypes.c_float(1.0), dtype, ws, size, None)

    for kw, text in ((dict(H=3), "multiple"), (dict(hd=257), "at most 256"), (dict(hd=0), "bad size"),
                     (dict(dtype=7), "unknown dtype"), (dict(pages=0), "number of pages"),
                     (dict(N=2, rs=3), "row stride"), (dict(q=None), "null"), (dict(last=2), "unit stride"),
                     (dict(P=1 << 27, rs=1 << 27), "too large"), (dict(P=4096, rs=4096, size=0), "workspace"),
                     (dict(P=4096, rs=4096, ws=None), "workspace"), (dict(P=4096, rs=4096, ws=8), "workspace")):
        with pytest.raises(ValueError, match=text):
            call(**kw)
    call(N=0)  # nothing to do


def test_python_entry_points_take_gpu_tensors_only():
    from hydra_amd.attention import PagePool, paged_attention, plan_pages, release_pages, store_pages

    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    kv = torch.zeros(4, 1, 16, 16)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        plan_pages(i, i, t, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        release_pages(i.bool(), i, t, i, i[:1], 16)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        store_pages(kv, kv, kv, kv, torch.zeros(4, 16, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        paged_attention(kv[:2, :, 0], kv, kv, t, i)
    for kw in (dict(requests=0), dict(max_length=0), dict(pages=0), dict(page_size=24)):
        with pytest.raises(ValueError, match="PagePool"):
            PagePool(**{**dict(requests=2, max_length=64, pages=4, page_size=16, device="cpu"), **kw})


def test_sizes_whose_products_overflow():
    from hydra_amd import _lib

    huge = 1 << 32
    s = st(1, 1, 1, 1)
    with pytest.raises(ValueError, match="too large"):
        plan(N=huge, P=huge, rs=huge)
    with pytest.raises(ValueError, match="too large"):
        plan(N=16, P=1 << 60, rs=1 << 60)
    with pytest.raises(ValueError, match="too large"):
        _lib.call("hydra_page_release", FAKE, FAKE, FAKE, huge, FAKE, 8, FAKE, huge, huge, 16, None)
    with pytest.raises(ValueError, match="too large"):
        _lib.call("hydra_page_store", FAKE, FAKE, FAKE, FAKE, FAKE, 1, None, 1, 1, 1, 16, 1 << 60, 16, s, s, s, s, 1, None)
    far = st(1, 1, 1 << 40, 1)
    with pytest.raises(ValueError, match="too far apart"):
        _lib.call("hydra_page_store", FAKE, FAKE, FAKE, FAKE, FAKE, 1, None, 1, 1, 1, 16, 4, 16, s, s, far, s, 1, None)
    with pytest.raises(ValueError, match="too large"):
        _lib.call("hydra_page_store", FAKE, FAKE, FAKE, FAKE, FAKE, 1, None, 1, 1, (1 << 31) - 1, 16, 4, 16, s, s, s, s, 1,
                  None)


def test_decode_prep_refusals():
    from hydra_amd import _lib
    from hydra_amd.attention.backends.ccgqa.ops import CCGQA_CONVS, CCGQA_QK_NORM, CCGQA_ROPE

    def call(N=1, Hq=4, Hkv=2, hd=16, ks=3, flags=CCGQA_CONVS, R=5, rs=128, pages=4, page=16, w=FAKE, temp=FAKE,
             cos=FAKE, last=1, dtype=1, q=FAKE):
        p = st(1, 1, 1, last)
        _lib.call("hydra_ccgqa_decode_prep", FAKE, rs, FAKE, R, FAKE, FAKE, w, w, w, w, temp, cos, cos, hd // 2, 64, q,
                  FAKE, FAKE, p, p, pages, page, N, Hq, Hkv, hd, ks, flags, dtype, FAKE, 1 << 40, None)

    for kw, text in ((dict(Hkv=3), "multiple"), (dict(hd=15), "even"), (dict(hd=0), "bad size"), (dict(R=4), "looks back"),
                     (dict(ks=5), "looks back"), (dict(ks=17), "taps"), (dict(page=8), "power of two"),
                     (dict(flags=1 << 20), "unknown flag"), (dict(N=2, rs=127), "row stride"), (dict(N=65536), "too large"),
                     (dict(pages=1 << 60), "too large"), (dict(dtype=9), "unknown dtype"), (dict(w=None), "four weights"),
                     (dict(flags=CCGQA_QK_NORM, temp=None), "temperature"), (dict(flags=CCGQA_ROPE, cos=None), "cos"),
                     (dict(last=2), "unit stride"), (dict(q=None), "null"),
                     (dict(flags=CCGQA_CONVS | _lib.CCGQA_W_TILED, dtype=0), "16-bit")):
        with pytest.raises(ValueError, match=text):
            call(**kw)
    call(N=0)  # nothing to do

    def fill(M=1, S=4, W=8, N=2, R=5, keep=4, rows=None, dtype=1, qkv=FAKE):
        _lib.call("hydra_ccgqa_ring_fill", qkv, S * W, W, FAKE, rows, FAKE, M, S, W, N, R, keep, 1, dtype, None)

    for kw, text in ((dict(keep=6), "more rows"), (dict(M=3), "more prompts"), (dict(S=0), "bad size"), (dict(N=0), "bad size"),
                     (dict(M=65536, N=65536), "too large"), (dict(dtype=5), "unknown dtype"), (dict(qkv=None), "null")):
        with pytest.raises(ValueError, match=text):
            fill(**kw)
    fill(M=0)


def test_token_logprobs_refusals():
    from hydra_amd import _lib

    def call(rows=2, V=100, rs=100, top=4, T=1.0, dtype=1, x=FAKE, ids=FAKE):
        _lib.call("hydra_token_logprobs", x, rows, V, rs, FAKE, T, top, FAKE, FAKE, None, FAKE, ids, dtype, None)

    def grad(rows=2, V=100, rs=100, top=4, T=1.0, dtype=1, x=FAKE, ids=FAKE):
        _lib.call("hydra_token_logprobs_bwd", x, rows, V, rs, FAKE, T, top, FAKE, FAKE, ids, FAKE, FAKE, FAKE, FAKE, dtype,
                  None)

    for kw, text in ((dict(V=0), "bad size"), (dict(rows=-1), "bad size"), (dict(V=1 << 30), "too large"),
                     (dict(rows=1 << 31), "too large"), (dict(rs=-1), "negative"), (dict(top=65), "top_k"),
                     (dict(V=3), "top_k"), (dict(T=0.0), "temperature"), (dict(T=float("nan")), "temperature"),
                     (dict(dtype=4), "unknown dtype"), (dict(x=None), "null"), (dict(ids=None), "null"),
                     (dict(x=FAKE + 1), "misaligned")):
        for entry in (call, grad):
            with pytest.raises(ValueError, match=text):
                entry(**kw)
    call(rows=0)
    grad(rows=0)


def test_layers_that_have_no_cache():
    """What the one-token kernels do not take is refused before a prompt enters."""
    from hydra_amd.attention import CCGQAAttention, PagePool

    pool = PagePool(2, 64, 4, 16, device="cpu")
    for kw, text in ((dict(dim=4096, n_heads=64, n_kv_heads=2, conv_kernel_size=5), "5 taps of 4096"),
                     (dict(dim=6144, n_heads=128, n_kv_heads=2), "3 taps of 6144"),
                     (dict(dim=1024, n_heads=2, n_kv_heads=1), "up to 256"),
                     (dict(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=63), "RoPE cache")):
        with torch.device("meta"):
            m = CCGQAAttention(compression_factor=1, **{**dict(max_seq_len=64), **kw})
        with pytest.raises(ValueError, match=text):
            m.new_cache(pool)
    with torch.device("meta"):
        m = CCGQAAttention(dim=256, n_heads=4, n_kv_heads=2, max_seq_len=64)
    with pytest.raises(RuntimeError, match="the pool is on cpu"):
        m.new_cache(pool)
