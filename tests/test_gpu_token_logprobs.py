"""GPU tests of token_logprobs against the oracle in fp64 (bounds derived in
oracle/logprobs.py): values, alternatives with ties, gradients against the
formula and against differences, and what masks leave."""
from __future__ import annotations

import pytest
import torch

from oracle import logprobs as ol

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = float("inf")


def make(rows, V, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * std).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g)
    return x, t, g


def check(x, t, cuda, top_k, T, form=lambda x: x):
    from hydra_amd.kernels import token_logprobs

    got = token_logprobs(form(x.to(cuda)), t.to(cuda), top_k=top_k, temperature=T)
    want = ol.forward(x, t, top_k, T)
    bound = ol.bounds(x, t, want[3], T)
    assert torch.equal(got.top_tokens.cpu(), want[3])
    for name, a, b, c in zip(("logprobs", "entropy", "top_logprobs"), got, want, bound):
        assert a.dtype == torch.float32 and a.shape == b.shape
        err = (a.cpu().double() - b).abs()
        assert bool((err <= c).all()), f"{name}: {err.max():.3e}, {(err / c).max():.2f} of the bound"
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,top_k", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 64, 64), (3, 100, 5), (2, 1000, 64), (9, 4099, 20), (2, 8192, 8),
    (4, 16000, 1), (3, 32000, 20), (5, 50257, 20), (2, 65536, 64), (2, 131080, 5), (1, 300001, 20),
])
def test_values_and_alternatives(cuda, dtype, rows, V, top_k):
    x, t, _ = make(rows, V, dtype, seed=V + top_k)
    for k, T in ((top_k, 1.0), (0, 0.7)):
        check(x, t, cuda, k, T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_shapes(cuda, dtype):
    from hydra_amd.kernels import token_logprobs

    x, t, _ = make(6, 1003, dtype, seed=1)
    want = check(x, t, cuda, 5, 1.0)
    for form in (lambda x: torch.cat([x, x], 1)[:, :1003], lambda x: torch.cat([x[:, :1], x], 1)[:, 1:],
                 lambda x: x.t().contiguous().t(), lambda x: torch.cat([x.new_zeros(3), x.reshape(-1)])[3:].view(6, 1003)):
        # sums go by 16-byte pieces of memory, so where a row starts orders them
        assert torch.equal(check(x, t, cuda, 5, 1.0, form).top_tokens, want.top_tokens)
    got = token_logprobs(x.to(cuda).view(2, 3, 1003), t.to(cuda).view(2, 3), top_k=5)
    assert got.logprobs.shape == (2, 3) and got.top_tokens.shape == (2, 3, 5)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    one = token_logprobs(x[0].to(cuda), t[0].to(cuda), top_k=5)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, want.top_tokens[0])
    none = token_logprobs(x[:0].to(cuda), t[:0].to(cuda), top_k=2)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 2)
    check(x[:1].repeat(4, 1), t[:4], cuda, 1, 1.0, form=lambda x: x[:1].expand(4, -1))


def test_strides_of_tokens(cuda):
    """A column of a wider tensor, every second of a vector, one for all rows, a
    transposed batch: the tokens' own strides, forward and backward."""
    from hydra_amd.kernels import token_logprobs

    x, t, g = make(6, 300, torch.float32, seed=4)
    wide = torch.randint(0, 300, (2, 3, 2), generator=g)
    wide[..., 1] = t.view(2, 3)
    spread = torch.full((11,), 7)
    spread[::2] = t
    for rows, tokens in ((x.view(2, 3, 300), wide.to(cuda)[..., 1]), (x, spread.to(cuda)[::2]),
                         (x, torch.tensor([5], device=cuda).expand(6)),
                         (x.view(2, 3, 300), t.view(2, 3).t().contiguous().to(cuda).t())):
        leaf, flat = rows.to(cuda).requires_grad_(), x.to(cuda).requires_grad_()
        same = tokens.cpu().contiguous().view(-1).to(cuda)
        got, want = token_logprobs(leaf, tokens, top_k=3), token_logprobs(flat, same, top_k=3)
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
        got.logprobs.sum().backward()
        want.logprobs.sum().backward()
        assert torch.equal(leaf.grad.view(6, 300), flat.grad)
        with torch.no_grad():
            assert torch.equal(token_logprobs(leaf, tokens).logprobs.view(-1), want.logprobs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 5000, 50257])
def test_equal_logits_take_the_lowest_index(cuda, dtype, V):
    """Rows of one value, of few values, of zeros of both signs, and with more
    equal largest values than the list of candidates holds."""
    g = torch.Generator().manual_seed(V)
    x = torch.stack([torch.full((V,), 1.5), torch.randint(0, 3, (V,), generator=g).float(),
                     torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0),
                     torch.randint(0, 40, (V,), generator=g).float(), (torch.arange(V) >= V // 2).float()]).to(dtype)
    t = torch.randint(0, V, (5,), generator=g)
    for k in (1, 7, min(V, 64)):
        check(x, t, cuda, k, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_masked_logits(cuda, dtype, low):
    """Few allowed tokens (fewer than the alternatives asked for), one, and a
    row that allows none."""
    low = -INF if low == "-inf" else torch.finfo(dtype).min
    V = 9001
    x, t, g = make(6, V, dtype, seed=3)
    keep = torch.zeros(6, V, dtype=torch.bool)
    for r, n in enumerate((V - 1, 300, 12, 3, 1, 0)):
        keep[r, torch.randperm(V, generator=g)[:n]] = True
    t = torch.where(keep.any(1), keep.float().argmax(1), t)
    x = torch.where(keep, x, torch.tensor(low, dtype=dtype))
    from hydra_amd.kernels import token_logprobs

    got = token_logprobs(x.to(cuda), t.to(cuda), top_k=20)
    want = ol.forward(x, t, 20)
    assert torch.equal(got.top_tokens.cpu(), want[3])
    full = slice(0, 6) if low != -INF else slice(0, 5)
    bound = ol.bounds(x[full], t[full], want[3][full], 1.0)
    for a, b, c in zip(got, want, bound):
        a, b = a.cpu().double(), b
        assert torch.equal(torch.isinf(a), torch.isinf(b))
        err = torch.where(torch.isinf(b), 0.0, a - b).abs()[full]
        # a masked entry's log probability is as large as the mask: 4 u of it
        assert bool((err <= c + 4 * ol.U * torch.where(torch.isinf(b), 0.0, b.abs())[full]).all())
    if low == -INF:
        assert got.logprobs[5] == -INF and got.entropy[5] == 0 and (got.top_logprobs[5] == -INF).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinities(cuda, dtype):
    """As log_softmax: NaN throughout, and in their row alone; NaN leads the
    alternatives."""
    from hydra_amd.kernels import token_logprobs

    x, t, _ = make(4, 3001, dtype, seed=5)
    x[1, 77], x[1, 3000], x[2, 5] = float("nan"), float("nan"), INF
    got = token_logprobs(x.to(cuda).requires_grad_(), t.to(cuda), top_k=4)
    for v in got[:3]:
        assert v[1].isnan().all() and v[2].isnan().all() and not v[0].isnan().any() and not v[3].isnan().any()
    assert got.top_tokens[1, :2].tolist() == [77, 3000] and got.top_tokens[2, 0] == 5
    assert torch.equal(got.top_tokens.cpu(), ol.forward(x, t, 4)[3])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,top_k,T", [(1, 1, 1, 1.0), (3, 5, 0, 1.0), (4, 37, 37, 0.5), (5, 4099, 3, 1.0),
                                            (2, 32000, 0, 0.7), (3, 50257, 20, 1.3), (2, 140000, 2, 1.0)])
def test_gradient_of_the_formula(cuda, dtype, rows, V, top_k, T):
    from hydra_amd.kernels import token_logprobs

    x, t, g = make(rows, V, dtype, seed=V)
    if rows > 2:
        t[1] = -100
        t[2] = V
    gl, gh, gt = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, top_k, generator=g)
    for form in (lambda x: x, lambda x: torch.cat([x, x], 1)[:, :V], lambda x: torch.cat([x[:, :1], x], 1)[:, 1:]):
        leaf = form(x.to(cuda)).detach().requires_grad_()
        out = token_logprobs(leaf, t.to(cuda), top_k=top_k, temperature=T)
        assert not out.top_tokens.requires_grad
        if rows > 2:
            assert out.logprobs[1] == 0 and out.logprobs[2] == 0
        loss = (out.logprobs * gl.to(cuda)).sum() + (out.entropy * gh.to(cuda)).sum() + (out.top_logprobs * gt.to(cuda)).sum()
        loss.backward()
        ids = out.top_tokens.cpu()
        want = ol.backward(x, t, gl, gh, gt if top_k else None, ids, T)
        bound = ol.bounds(x, t, ids, T, gl, gh, gt if top_k else None)[3]
        bound = 1.01 * bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + torch.finfo(dtype).smallest_normal
        assert leaf.grad.dtype == dtype and leaf.grad.shape == x.shape
        err = (leaf.grad.cpu().double() - want).abs()
        assert bool((err <= bound).all()), f"{err.max():.3e}, {(err / bound).max():.2f} of the bound"


@pytest.mark.parametrize("which", ["logprobs", "entropy", "top_logprobs"])
def test_gradient_of_each_output_alone_against_differences(cuda, which):
    """Directional differences of the fp64 oracle, and grads that are None."""
    from hydra_amd.kernels import token_logprobs

    x, t, g = make(3, 600, torch.float32, seed=12, std=1.0)
    w = torch.randn((3, 4) if which == "top_logprobs" else (3,), generator=g)
    leaf = x.to(cuda).requires_grad_()
    out = token_logprobs(leaf, t.to(cuda), top_k=4, temperature=0.8)
    (getattr(out, which) * w.to(cuda)).sum().backward()
    d = torch.randn(3, 600, generator=g).double()
    index = ("logprobs", "entropy", "top_logprobs").index(which)
    h = 1e-5

    def value(z):  # the alternatives stay those of x
        lp = torch.log_softmax(z / 0.8, 1)
        outs = (lp.gather(1, t[:, None])[:, 0], -(lp.exp() * lp).sum(1), lp.gather(1, out.top_tokens.cpu()))
        return (outs[index] * w.double()).sum()

    slope = (value(x.double() + h * d) - value(x.double() - h * d)) / (2 * h)
    # differences: h^2 of the third derivative, below 1e-8; the gradient's own
    # terms are good to 1e-6 of their absolute sum
    got = (leaf.grad.cpu().double() * d).sum()
    assert abs(got - slope) <= 1e-6 * (leaf.grad.cpu().double() * d).abs().sum() + 1e-7


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_gradient_of_masked_rows(cuda, dtype, low):
    """No gradient at masked logits, none at all (and no NaN) in a row of -inf."""
    from hydra_amd.kernels import token_logprobs

    x, t, g = make(3, 2000, dtype, seed=7)
    x[0, ::2] = x[1, 1:] = x[2] = -INF if low == "-inf" else torch.finfo(dtype).min
    t[0], t[1] = 1, 0
    leaf = x.to(cuda).requires_grad_()
    out = token_logprobs(leaf, t.to(cuda), top_k=3)
    (out.logprobs[:2].sum() + out.entropy.sum() + out.top_logprobs[:1].sum()).backward()
    grad = leaf.grad.cpu()
    assert grad.isfinite().all()
    assert not grad[0, ::2].any() and grad[0, 1::2].any()
    if low == "-inf":
        assert not grad[2].any()


def test_broadcast_logits_share_their_gradient(cuda):
    from hydra_amd.kernels import token_logprobs

    x, _, _ = make(1, 500, torch.float32, seed=2)
    t = torch.tensor([3, 3, 9, -100], device=cuda)
    one, many = x.to(cuda).requires_grad_(), x.to(cuda).repeat(4, 1).requires_grad_()
    for leaf, rows in ((one, one.expand(4, -1)), (many, many)):
        token_logprobs(rows, t).logprobs.sum().backward()
    assert torch.allclose(one.grad, many.grad.sum(0, keepdim=True), rtol=1e-6, atol=1e-7)


def test_captured_training_step(cuda):
    """Forward and backward captured, replayed with new inputs and eager work
    in between, while an eager graph of other leaves lives."""
    from hydra_amd.kernels import token_logprobs

    x, t, g = make(50, 4099, torch.bfloat16, seed=9)
    gl = torch.randn(50, generator=g).to(cuda)
    leaf, tok = x.to(cuda).requires_grad_(), t.to(cuda)
    alive = token_logprobs(x.to(cuda).requires_grad_(), tok, top_k=5)

    def step(z):
        out = token_logprobs(z, tok, top_k=5, temperature=0.9)
        return (out.logprobs.detach(), out.top_tokens, *torch.autograd.grad([out.logprobs, out.entropy], [z], [gl, gl]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(leaf)
    for i in range(4):
        with torch.no_grad():
            leaf.copy_(torch.roll(x, i, 1).to(cuda) * (1 + i))
        want = step(leaf)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    alive.logprobs.sum().backward()


def test_same_bits_on_two_streams(cuda):
    from hydra_amd.kernels import token_logprobs

    x, t, _ = make(300, 50257, torch.bfloat16, seed=4)
    x, t = x.to(cuda), t.to(cuda)
    want = token_logprobs(x, t, top_k=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            a = token_logprobs(x, t, top_k=20)
        b = token_logprobs(x, t, top_k=20)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) and torch.equal(r, q) for p, q, r in zip(a, want, b))


def test_rows_past_32_bits(cuda):
    """More than 2^31 logits: the last rows' values and gradient."""
    from hydra_amd.kernels import token_logprobs

    rows, V = 43000, 50257
    assert rows * V > 2**31
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=cuda)
    tail, t, _ = make(2, V, torch.bfloat16, seed=1)
    x[-2:] = tail.to(cuda)
    tokens = torch.full((rows,), 7, device=cuda)
    tokens[-2:] = t.to(cuda)
    x.requires_grad_()
    out = token_logprobs(x, tokens, top_k=3)
    small = tail.to(cuda).requires_grad_()
    ref = token_logprobs(small, t.to(cuda), top_k=3)
    assert torch.equal(out.logprobs[-2:], ref.logprobs) and torch.equal(out.top_tokens[-2:], ref.top_tokens)
    assert out.top_tokens[0].tolist() == [0, 1, 2]
    (grad,) = torch.autograd.grad(out.logprobs.sum(), x)
    (want,) = torch.autograd.grad(ref.logprobs.sum(), small)
    assert torch.equal(grad[-2:], want)


def test_refusals(cuda):
    from hydra_amd.kernels import token_logprobs

    x, t = torch.zeros(2, 30, device=cuda), torch.zeros(2, dtype=torch.long, device=cuda)
    for args, kw, text in (((x, t[:1]), {}, "do not match"), ((x, t.int()), {}, "int64"), ((x, t), dict(top_k=31), "top_k"),
                           ((x, t), dict(top_k=-1), "top_k"), ((x.repeat(1, 9), t), dict(top_k=65), "top_k"),
                           ((x, t), dict(temperature=0.0), "temperature"), ((x, t), dict(temperature=-1.0), "temperature"),
                           ((x, t), dict(temperature=INF), "temperature"), ((x, t), dict(temperature=float("nan")), "temperature"),
                           ((x, t), dict(temperature=1e-45), "temperature"), ((x[:, :0], t), {}, "bad size")):
        with pytest.raises(ValueError, match=text):
            token_logprobs(*args, **kw)
    with pytest.raises(TypeError, match="dtype"):
        token_logprobs(x.double(), t)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        token_logprobs(x.cpu(), t.cpu())
    leaf = x.clone().requires_grad_()
    (grad,) = torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
