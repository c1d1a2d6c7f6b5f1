"""GPU tests of one-token CCGQA: the prep of a token from the rows before it
against the oracle's whole sequence in fp64 (bounds derived in
oracle/paged.py), the ring of prompts, and layers and blocks that decode."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from conftest import max_rel_err
from oracle import blocks as ob
from oracle import ccgqa as oc
from oracle import paged as op

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
PLAIN = dict(use_convs=False)
CONFIGS = {
    "debug": dict(dim=512, n_heads=8, n_kv_heads=2),
    "hd64": dict(dim=1024, n_heads=4, n_kv_heads=1),
    "hd128": dict(dim=1024, n_heads=2, n_kv_heads=1),
    "mha": dict(dim=512, n_heads=4, n_kv_heads=4),
    "seven": dict(dim=1792, n_heads=28, n_kv_heads=4),
    "hd48": dict(dim=768, n_heads=4, n_kv_heads=2),       # no matrix-core form
    "hd6": dict(dim=96, n_heads=4, n_kv_heads=2),
    "taps5": dict(dim=256, n_heads=4, n_kv_heads=2, conv_kernel_size=5),
    "taps1": dict(dim=256, n_heads=4, n_kv_heads=2, conv_kernel_size=1),
    "noconv": dict(dim=256, n_heads=4, n_kv_heads=2, **PLAIN),
    "bare": dict(dim=256, n_heads=4, n_kv_heads=2, use_rope=False, use_qk_norm=False, use_qk_mean=False,
                 use_value_shift=False, **PLAIN),
    "norope": dict(dim=256, n_heads=4, n_kv_heads=2, use_rope=False),
    "nonorm": dict(dim=256, n_heads=4, n_kv_heads=2, use_qk_norm=False),
    "nomean": dict(dim=256, n_heads=4, n_kv_heads=1, use_qk_mean=False, use_value_shift=False),
}


def flags_of(cfg):
    from hydra_amd.attention.backends.ccgqa.ops import prep_flags

    return prep_flags(cfg.use_convs, cfg.use_qk_mean, cfg.use_value_shift, cfg.use_qk_norm, cfg.use_rope)


def weights_of(params, cfg, cuda, dtype):
    if not cfg.use_convs:
        return ()
    return tuple(params[n].to(cuda, dtype) for n in ("q_conv.conv1.weight", "q_conv.conv2.weight",
                                                     "k_conv.conv1.weight", "k_conv.conv2.weight"))


def case(cfg, positions, dtype, seed, R=None):
    """Rows of requests up to their positions, the ring they leave (NaN where
    no row of theirs may be read) and parameters, all rounded to dtype."""
    from hydra_amd.attention.backends.ccgqa.ops import decode_reach

    g = torch.Generator().manual_seed(seed)
    params = {k: v.to(dtype) for k, v in oc.init_params(cfg, g, std=0.1).items()}
    W = cfg.latent_dim + 2 * cfg.kv_dim
    reach = decode_reach(flags_of(cfg), cfg.conv_kernel_size)
    R = R or reach + 1
    rows = [torch.randn(p + 1, W, generator=g).to(dtype) for p in positions]
    ring = torch.full((len(positions), R, W), float("nan"), dtype=dtype)
    for n, p in enumerate(positions):
        for b in range(1, min(reach, p) + 1):
            ring[n, (p - b) % R] = rows[n][p - b]
    return params, rows, ring


def run(cuda, cfg, dtype, params, rows, ring, positions, slots, pages, page, tiled=False, table=None, **kw):
    from hydra_amd._lib import CCGQA_W_TILED
    from hydra_amd.attention.backends.ccgqa.ops import ccgqa_decode_prep
    from oracle.fused_ops import rope_cache

    cos, sin = rope_cache(cfg.head_dim, table or max(positions) + 1)
    kp, vp = (torch.full((pages, cfg.n_kv_heads, page, cfg.head_dim), 7.0, dtype=dtype, device=cuda) for _ in range(2))
    ring = ring.to(cuda)
    q = ccgqa_decode_prep(
        torch.stack([r[-1] for r in rows]).to(cuda), ring, torch.tensor(positions, dtype=torch.int32, device=cuda),
        torch.tensor(slots, device=cuda), kp, vp, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim,
        flags_of(cfg) | (CCGQA_W_TILED if tiled else 0), *weights_of(params, cfg, cuda, dtype),
        temperature=params["key_temperature"].to(cuda) if cfg.use_qk_norm else None,
        cos=cos.to(cuda) if cfg.use_rope else None, sin=sin.to(cuda) if cfg.use_rope else None,
        conv_ks=cfg.conv_kernel_size, **kw)
    return q.cpu(), kp.cpu(), vp.cpu(), ring.cpu(), (cos.double(), sin.double())


def check(cfg, dtype, params, rows, ring, positions, slots, page, got):
    q, kp, vp, kept, (cos, sin) = got
    R = ring.shape[1]
    p64 = {k: v.double() for k, v in params.items()}
    for n, (p, slot) in enumerate(zip(positions, slots)):
        want = oc.prep(p64, rows[n].double()[None], cfg, cos[:p + 1], sin[:p + 1])
        bq, bk = op.decode_bound(params, rows[n].double(), cfg, dtype)
        k, v = kp[slot // page, :, slot % page].double(), vp[slot // page, :, slot % page].double()
        for name, a, b, bound in (("q", q[n].double(), want[0][0, :, -1], bq), ("k", k, want[1][0, :, -1], bk)):
            err = (a - b).abs()
            assert bool((err <= bound).all()), f"{name} of request {n}: {err.max():.3e}, {(err / bound).max():.2f}"
        assert torch.equal(v, want[2][0, :, -1])
        ring[n, p % R] = rows[n][-1]
    assert torch.equal(kept.nan_to_num(nan=123.0), ring.nan_to_num(nan=123.0))
    free = torch.ones(kp.shape[0], kp.shape[2], dtype=torch.bool)
    for slot in slots:
        free[slot // page, slot % page] = False
    assert (kp.transpose(1, 2)[free] == 7).all() and (vp.transpose(1, 2)[free] == 7).all()


POSITIONS = [0, 1, 2, 3, 4, 5, 8, 17, 0, 29, 4, 2, 11, 1, 3, 40, 6]  # one past a tile of 16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", list(CONFIGS))
def test_prep_of_one_token(cuda, name, dtype):
    cfg = oc.CCGQAConfig(**CONFIGS[name])
    page = 16
    slots = [(7 * n + 3) % 19 * page + (5 * n) % page for n in range(len(POSITIONS))]
    params, rows, ring = case(cfg, POSITIONS, dtype, seed=len(name))
    got = run(cuda, cfg, dtype, params, rows, ring, POSITIONS, slots, 19, page)
    check(cfg, dtype, params, rows, ring, POSITIONS, slots, page, got)


@pytest.mark.parametrize("name", ["debug", "hd64", "hd128", "mha", "seven"])
@pytest.mark.parametrize("N", [1, 16, 33])
def test_tiled_weights_and_longer_rings(cuda, name, N):
    from hydra_amd.attention.backends.ccgqa.ops import tiled_weights_ok

    cfg = oc.CCGQAConfig(**CONFIGS[name])
    assert tiled_weights_ok(cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, torch.bfloat16)
    positions = [(5 * n) % 23 for n in range(N)]
    slots = [n * 64 + 63 for n in range(N)]
    params, rows, ring = case(cfg, positions, torch.bfloat16, seed=N, R=9)
    got = run(cuda, cfg, torch.bfloat16, params, rows, ring, positions, slots, N, 64, tiled=True)
    check(cfg, torch.bfloat16, params, rows, ring, positions, slots, 64, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_workgroups_than_units(cuda, dtype):
    """Heads times tiles of 16 requests past 256: workgroups of fewer waves."""
    cfg, N = oc.CCGQAConfig(**CONFIGS["seven"]), 133
    assert (cfg.n_heads + cfg.n_kv_heads) * -(-N // 16) > torch.cuda.get_device_properties(0).multi_processor_count
    positions = [n % 7 for n in range(N)]
    slots = [n * 16 + n % 16 for n in range(N)]
    params, rows, ring = case(cfg, positions, dtype, seed=3)
    got = run(cuda, cfg, dtype, params, rows, ring, positions, slots, N, 16)
    check(cfg, dtype, params, rows, ring, positions, slots, 16, got)


@pytest.mark.parametrize("name", ["debug", "hd48"])
def test_idle_requests_change_nothing(cuda, name):
    """No slot, one outside the pool, a position below 0 or past the rotation's
    table: zeros for q, and nothing else; their neighbours as ever."""
    cfg, dtype, page = oc.CCGQAConfig(**CONFIGS[name]), torch.bfloat16, 16
    positions = [3, 4, 5, 6, 7]
    slots = [5, -1, 3 * page, 20, 33]
    asked = [3, 4, 5, -1, 40]
    params, rows, ring = case(cfg, positions, dtype, seed=2)
    q, kp, vp, kept, tables = run(cuda, cfg, dtype, params, rows, ring, asked, slots, 3, page, table=40)
    assert not q[1:].any() and torch.equal(kept[1:].nan_to_num(nan=9.), ring[1:].nan_to_num(nan=9.))
    check(cfg, dtype, params, rows[:1], ring[:1], positions[:1], slots[:1], page, (q[:1], kp, vp, kept[:1], tables))


@pytest.mark.parametrize("name", ["hd128", "hd48"])
def test_pages_past_32_bits(cuda, name):
    """A slot in the last page of a pool of more than 2^32 bytes is written like
    one of a small pool."""
    from hydra_amd.attention.backends.ccgqa.ops import ccgqa_decode_prep
    from oracle.fused_ops import rope_cache

    cfg, dtype, page = oc.CCGQAConfig(**CONFIGS[name]), torch.bfloat16, 4096
    params, rows, ring = case(cfg, [9], dtype, seed=4)
    cos, sin = (t.to(cuda) for t in rope_cache(cfg.head_dim, 16))
    many = (1 << 32) // (page * cfg.kv_dim * 2) + 2
    outs = []
    for pages in (2, many):
        kp, vp = (torch.zeros(pages, cfg.n_kv_heads, page, cfg.head_dim, dtype=dtype, device=cuda) for _ in range(2))
        q = ccgqa_decode_prep(rows[0][-1:].to(cuda), ring.to(cuda), torch.tensor([9], dtype=torch.int32, device=cuda),
                              torch.tensor([pages * page - 5], device=cuda), kp, vp, cfg.n_heads, cfg.n_kv_heads,
                              cfg.head_dim, flags_of(cfg), *weights_of(params, cfg, cuda, dtype),
                              temperature=params["key_temperature"].to(cuda), cos=cos, sin=sin)
        outs.append((q, kp[-1].clone(), vp[-1].clone()))
        assert kp[-1, :, -5].any() and not kp[:-1].any() and not vp[:-1].any()
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_bf16_tables_and_strided_rows(cuda):
    from hydra_amd.attention.backends.ccgqa.ops import ccgqa_decode_prep
    from oracle.fused_ops import rope_cache

    cfg, dtype = oc.CCGQAConfig(**CONFIGS["hd64"]), torch.bfloat16
    positions, slots = [3, 9, 20], [1, 17, 40]
    params, rows, ring = case(cfg, positions, dtype, seed=3)
    cos, sin = (t[0, 0].to(dtype) for t in rope_cache(cfg.head_dim, 32))
    new = torch.stack([r[-1] for r in rows]).to(cuda)
    outs = []
    for wide, tab in ((new, (cos.float(), sin.float())), (torch.cat([new, new], 1)[:, :new.shape[1]], (cos, sin)),
                      (new.t().contiguous().t(), (cos[None, None], sin[None, None]))):
        kp, vp = (torch.zeros(3, 16, 1, 64, dtype=dtype, device=cuda).transpose(1, 2) for _ in range(2))
        kept = ring.to(cuda)
        q = ccgqa_decode_prep(wide, kept, torch.tensor(positions, dtype=torch.int32, device=cuda),
                              torch.tensor(slots, device=cuda).view(3, 1), kp, vp, 4, 1, 64, flags_of(cfg),
                              *weights_of(params, cfg, cuda, dtype), temperature=params["key_temperature"].to(cuda),
                              cos=tab[0].to(cuda), sin=tab[1].to(cuda))
        outs.append((q, kp, vp, kept.nan_to_num(nan=5.0)))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ring_fill(cuda, dtype):
    from hydra_amd.attention.backends.ccgqa.ops import ccgqa_ring_fill

    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(5, 11, 48, generator=g).to(dtype)
    lengths, rows = [1, 12, 11, 3, 0, 7, 2], [4, 0, 6, 2, 1]
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    for order in (None, rows):
        ring = torch.full((7, 6, 48), 3.0, dtype=dtype)
        got = ring.to(cuda)
        ccgqa_ring_fill(qkv.to(cuda), got, lens, 4, None if order is None else torch.tensor(order, device=cuda))
        for m in range(5):
            r = m if order is None else order[m]
            n = lengths[r]
            for s in range(max(0, n - 4), n if n <= 11 else 0):
                ring[r, s % 6] = qkv[m, s]
        assert torch.equal(got.cpu(), ring)
    ccgqa_ring_fill(qkv.to(cuda), got, lens, 4, torch.tensor([-1, 7, 2**40, -2**40, 7], device=cuda), clear=True)
    assert torch.equal(got.cpu(), ring)
    # the rows past a prompt's end, in place, of requests alone and also without a row to keep
    for keep in (4, 0):
        for order in (None, rows, [7, 0, -1, 2, 1]):
            x = qkv.clone()
            wide = torch.full((5, 11, 50), 2.0, dtype=dtype, device=cuda)
            wide[..., 1:49] = qkv.to(cuda)
            ccgqa_ring_fill(wide[..., 1:49], got.clone(), lens, keep,
                            None if order is None else torch.tensor(order, device=cuda), clear=True)
            for m in range(5):
                r = m if order is None else order[m]
                if 0 <= r < 7 and 0 < lengths[r] <= 11:
                    x[m, lengths[r]:] = 0
            assert torch.equal(wide[..., 1:49].cpu(), x) and (wide[..., ::49] == 2).all()
    with pytest.raises(ValueError, match="overlap"):
        ccgqa_ring_fill(qkv.to(cuda)[:1].expand(5, 11, 48), got, lens, 4, clear=True)


def layer(cuda, cfg, dtype, seed, max_seq_len=256):
    from hydra_amd.attention import CCGQAAttention

    kw = dataclasses.asdict(cfg)
    kw.pop("output_scale")
    kw["max_seq_len"] = max_seq_len
    m = CCGQAAttention(**kw)
    params = {k: v.to(dtype).float() for k, v in oc.init_params(cfg, torch.Generator().manual_seed(seed), std=0.05).items()}
    m.load_state_dict(params)
    return m.to(cuda, dtype).eval(), params


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2e-2), (torch.float16, 2e-2)])
@pytest.mark.parametrize("name", ["debug", "hd64", "seven", "hd48", "taps5", "noconv", "bare"])
def test_layer_prefill_and_decode(cuda, name, dtype, tol):
    """Prompts of unequal length, then tokens one by one (one request idle now
    and then, one that starts from nothing), against the oracle's forward of the
    whole sequences (the tolerances of the layer's forward)."""
    from hydra_amd.attention import PagePool

    cfg = oc.CCGQAConfig(**CONFIGS[name])
    m, params = layer(cuda, cfg, dtype, seed=1)
    N, steps = 5, 20
    pool = PagePool(N, 96, 30, 16, device=cuda)
    cache = m.new_cache(pool)
    prompts = [1, 17, 0, 40, 6]
    g = torch.Generator().manual_seed(2)
    x = torch.randn(N, 80, cfg.dim, generator=g).to(dtype).float()
    want = oc.forward(params, x, cfg)
    at = list(prompts)
    plan = pool.plan(torch.tensor(prompts, dtype=torch.int32, device=cuda), width=40, from_empty=True)
    out = m.prefill(x[:, :40].to(cuda, dtype), cache, plan)
    for n, p in enumerate(prompts):
        if p:
            assert max_rel_err(out[n, :p], want[n, :p]) < tol
    for step in range(steps):
        new = [0 if (step + n) % 7 == 3 else 1 for n in range(N)]
        plan = pool.plan(torch.tensor(new, dtype=torch.int32, device=cuda))
        rows = torch.stack([x[n, at[n]] for n in range(N)]).to(cuda, dtype)
        out = m.decode(rows[:, None] if step % 2 else rows, cache, plan).view(N, -1)
        for n in range(N):
            if new[n]:
                err = (out[n].cpu().double() - want[n, at[n]].double()).abs().max() / want[n].double().abs().max()
                assert err < tol, (step, n, float(err))
                at[n] += 1
            else:
                assert not out[n].any()
    assert pool.lengths.tolist() == at


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["debug", "hd64", "mha", "hd48", "noconv"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_padding_stays_out_whatever_it_holds(cuda, name, dtype, bad):
    from hydra_amd.attention import PagePool

    cfg = oc.CCGQAConfig(**CONFIGS[name])
    m, _ = layer(cuda, cfg, dtype, seed=1)
    prompts, S = [50, 64, 1, 33, 0], 64
    x = torch.randn(5, S, cfg.dim, generator=torch.Generator().manual_seed(8)).to(cuda, dtype)
    new = torch.tensor(prompts, dtype=torch.int32, device=cuda)
    outs = []
    for fill in (0.0, bad):
        pool = PagePool(5, 96, 30, 16, device=cuda)
        cache = m.new_cache(pool)
        for n, p in enumerate(prompts):
            x[n, p:] = fill
        out = m.prefill(x, cache, pool.plan(new, width=S, from_empty=True))
        step = m.decode(x[:, 0], cache, pool.plan((new > 0).int()))
        assert not step[4].any()  # idle, its row of x padding
        outs.append(([out[n, :p].clone() for n, p in enumerate(prompts)], step[:4], cache.ring[:4], cache.k_pages,
                     cache.v_pages))
    for a, b in zip(outs[0][0], outs[1][0]):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(outs[0][1:], outs[1][1:]))
    assert all(t.isfinite().all() for t in (*outs[1][0], *outs[1][1:]))


def test_prompts_join_a_running_batch(cuda):
    """Requests end, give their pages back and others take their rows while
    the rest decode; a request for which no page is left is refused and leaves
    the others alone."""
    from hydra_amd.attention import PagePool

    cfg, dtype = oc.CCGQAConfig(**CONFIGS["debug"]), torch.float32
    m, params = layer(cuda, cfg, dtype, seed=4)
    pool = PagePool(3, 64, 5, 16, device=cuda)
    cache = m.new_cache(pool)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    x = torch.randn(4, 64, cfg.dim, generator=torch.Generator().manual_seed(3))
    want = oc.forward(params, x, cfg)
    plan = pool.plan(i32(20, 30, 0), width=30, from_empty=True)
    out = m.prefill(x[:3, :30].to(cuda), cache, plan)
    assert max_rel_err(out[0, :20], want[0, :20]) < 1e-5 and max_rel_err(out[1, :30], want[1, :30]) < 1e-5
    plan = pool.plan(i32(0, 0, 33), width=33, from_empty=True)  # three pages, one left
    assert plan.granted.tolist() == [True, True, False] and pool.free_count.tolist() == [1]
    m.prefill(x[2:3, :33].to(cuda), cache, plan, rows=torch.tensor([2], device=cuda))
    pool.release(torch.tensor([True, False, False], device=cuda))
    plan = pool.plan(i32(0, 0, 33), width=33, from_empty=True)
    assert plan.granted.all()
    out = m.prefill(x[2:3, :33].to(cuda), cache, plan, rows=torch.tensor([2], device=cuda))
    assert max_rel_err(out[0], want[2, :33]) < 1e-5
    plan = pool.plan(i32(5, 0, 0), width=5, from_empty=True)  # no page left
    assert plan.granted.tolist() == [False, True, True]
    before = [t.clone() for t in (cache.k_pages, cache.v_pages, cache.ring)]
    m.prefill(x[:3, :5].to(cuda), cache, plan, rows=torch.tensor([0, -1, 3], device=cuda))  # refused, no requests
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k_pages, cache.v_pages, cache.ring)))
    for step in range(2):
        plan = pool.plan(i32(1, 1, 1))
        out = m.decode(torch.stack([x[3, 0], x[1, 30 + step], x[2, 33 + step]]).to(cuda), cache, plan)
        assert plan.granted.tolist() == [False, True, True] and not out[0].any()
        assert max_rel_err(out[1], want[1, 30 + step]) < 1e-5 and max_rel_err(out[2], want[2, 33 + step]) < 1e-5


def test_decode_step_captured(cuda):
    """A captured step (plan, layer) replayed with eager work in between
    equals the eager steps, replay by replay."""
    from hydra_amd.attention import PagePool

    cfg, dtype = oc.CCGQAConfig(**CONFIGS["hd64"]), torch.bfloat16
    m, _ = layer(cuda, cfg, dtype, seed=6)
    N = 3
    state = []
    for _ in range(2):
        pool = PagePool(N, 128, 24, 16, device=cuda)
        state.append((pool, m.new_cache(pool)))
    (pool, cache), (epool, ecache) = state
    x = torch.randn(N, 100, cfg.dim, generator=torch.Generator().manual_seed(5)).to(cuda, dtype)
    lens = torch.tensor([30, 4, 17], dtype=torch.int32, device=cuda)
    for p, c in state:
        m.prefill(x[:, :30], c, p.plan(lens, width=30, from_empty=True))
    token, one = torch.zeros(N, cfg.dim, dtype=dtype, device=cuda), torch.ones(N, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a step without tokens: warms up, changes nothing
        m.decode(token, cache, pool.plan(torch.zeros_like(one)))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.decode(token, cache, pool.plan(one))
    for step in range(40):
        token.copy_(x[:, 30 + step])
        graph.replay()
        want = m.decode(x[:, 30 + step].contiguous(), ecache, epool.plan(one))
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
    assert pool.lengths.tolist() == [70, 44, 57]


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2)])
def test_block_generates(cuda, dtype, tol):
    """Two HydraBlocks over one pool, prompts and eight tokens, against the
    oracle's blocks on the whole sequences."""
    from hydra_amd.attention import PagePool
    from hydra_amd.model.framework import HydraBlock

    torch.manual_seed(0)
    dim, N = 256, 3
    made = [HydraBlock(dim, n_heads=4, n_kv_heads=2, max_seq_len=128).to(dtype).float() for _ in range(2)]
    refs = [{k: v.detach().clone() for k, v in b.state_dict().items()} for b in made]
    cfg = oc.CCGQAConfig(dim=dim, n_heads=4, n_kv_heads=2, max_seq_len=128)
    x = torch.randn(N, 40, dim, generator=torch.Generator().manual_seed(1)).to(dtype).float()
    want = x
    for ref in refs:
        want = ob.hydra_block(ref, want, cfg)
    blocks = [b.to(cuda, dtype).eval() for b in made]
    pool = PagePool(N, 64, 12, 16, device=cuda)
    caches = [b.new_cache(pool) for b in blocks]
    lens = [20, 3, 11]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    plan = pool.plan(i32(lens), width=20, from_empty=True)
    h = x[:, :20].to(cuda, dtype)
    for b, c in zip(blocks, caches):
        h = b.prefill(h, c, plan)
    top = want.abs().max()
    for n, p in enumerate(lens):
        assert (h[n, :p].float().cpu() - want[n, :p]).abs().max() / top < tol
    for step in range(8):
        plan = pool.plan(i32([1] * N))
        h = torch.stack([x[n, lens[n] + step] for n in range(N)]).to(cuda, dtype)
        for b, c in zip(blocks, caches):
            h = b.decode(h, c, plan)
        ref = torch.stack([want[n, lens[n] + step] for n in range(N)])
        assert (h.float().cpu() - ref).abs().max() / top < tol, step


def test_refusals(cuda):
    from hydra_amd.attention import PagePool
    from hydra_amd.attention.backends.ccgqa.ops import ccgqa_decode_prep, ccgqa_ring_fill

    cfg, dtype = oc.CCGQAConfig(**CONFIGS["debug"]), torch.bfloat16
    m, params = layer(cuda, cfg, dtype, seed=1, max_seq_len=64)
    pool = PagePool(2, 64, 8, 16, device=cuda)
    cache = m.new_cache(pool)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    x = torch.zeros(2, 8, cfg.dim, dtype=dtype, device=cuda)
    wide = pool.plan(i32(0, 0), width=8)
    empty = pool.plan(i32(0, 0), width=8, from_empty=True)
    one = pool.plan(i32(0, 0))
    with pytest.raises(ValueError, match="from_empty"):
        m.prefill(x, cache, wide)
    with pytest.raises(ValueError, match="width 8"):
        m.prefill(x, cache, pool.plan(i32(0, 0), width=9, from_empty=True))
    with pytest.raises(ValueError, match="say which"):
        m.prefill(x[:1], cache, empty)
    with pytest.raises(ValueError, match="rows must be"):
        m.prefill(x, cache, empty, rows=i32(0, 1))
    with pytest.raises(ValueError, match="width 1"):
        m.decode(x[:, 0], cache, wide)
    for bad in (x[:1, 0], x[:, :2], x[:, 0].view(2, 2, -1)):
        with pytest.raises(ValueError, match="x must be"):
            m.decode(bad, cache, one)
    with pytest.raises(ValueError, match="the cache"):
        m.decode(x[:, 0].float(), cache, one)
    with pytest.raises(ValueError, match="RoPE cache"):
        m.new_cache(PagePool(2, 65, 8, 16, device=cuda))
    other, _ = layer(cuda, oc.CCGQAConfig(**CONFIGS["hd64"]), dtype, seed=1)
    with pytest.raises(ValueError, match="another layer"):
        other.decode(torch.zeros(2, 1024, dtype=dtype, device=cuda), cache, one)
    with pytest.raises(ValueError, match="a plan of"):
        m.decode(x[:, 0], cache, PagePool(3, 64, 8, 16, device=cuda).plan(i32(0, 0, 0)))
    w = weights_of(params, cfg, cuda, dtype)
    rope = dict(cos=m.cos_cached, sin=m.sin_cached)
    rows = torch.zeros(2, cfg.latent_dim + 2 * cfg.kv_dim, dtype=dtype, device=cuda)
    good = dict(qkv=rows, ring=cache.ring, positions=one.positions, slots=one.slots, k_pages=cache.k_pages,
                v_pages=cache.v_pages, n_heads=8, n_kv_heads=2, head_dim=16, flags=flags_of(cfg), wq1=w[0], wq2=w[1],
                wk1=w[2], wk2=w[3], temperature=m.key_temperature, **rope)
    ccgqa_decode_prep(**good)
    for change, text in ((dict(qkv=rows[:, :8]), "qkv must be"), (dict(ring=cache.ring[:, :4].contiguous()), "more than 4"),
                         (dict(ring=cache.ring[:, :, :8]), "ring must be"), (dict(ring=cache.ring[:1]), "ring must hold"),
                         (dict(positions=one.positions.long()), "positions"), (dict(slots=one.slots.int()), "slots"),
                         (dict(slots=one.slots[:1]), "slots"), (dict(k_pages=cache.k_pages[:, :1], v_pages=cache.v_pages[:, :1]), "pages must be"),
                         (dict(temperature=None), "temperature"), (dict(wq1=w[1]), "weight shape"),
                         (dict(cos=m.cos_cached[..., :4], sin=m.sin_cached[..., :4]), "columns"),
                         (dict(conv_ks=5), "more than 8"), (dict(n_heads=7), "qkv must be")):
        with pytest.raises(ValueError, match=text):
            ccgqa_decode_prep(**{**good, **change})
    for key in ("qkv", "ring", "k_pages"):
        with pytest.raises(RuntimeError, match="no gradient"):
            ccgqa_decode_prep(**{**good, key: good[key].clone().requires_grad_()})
    with pytest.raises(RuntimeError, match="no gradient"):
        ccgqa_ring_fill(x[:, :, :1].expand(2, 8, cache.ring.shape[2]).clone().requires_grad_(), cache.ring, one.seen, 4)
    none = m.prefill(x[:0], cache, empty, rows=torch.zeros(0, dtype=torch.long, device=cuda))
    assert none.shape == (0, 8, cfg.dim)
