"""GPU tests of row-wise operators on tensors whose dimensions of one element
have strides of their own (one decoding step, time first), and on no rows."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


FORMS = {
    "time first": lambda g: torch.randn(1, 5, 300, generator=g).transpose(0, 1),
    "one sequence": lambda g: torch.randn(5, 1, 300, generator=g).transpose(0, 1),
    "one column": lambda g: torch.randn(1, 6, generator=g).t(),
    "ones": lambda g: torch.randn(2, 1, 3, 1, 40, generator=g).permute(1, 0, 3, 2, 4),
    "none": lambda g: torch.randn(3, 0, 40, generator=g).transpose(0, 1),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", list(FORMS))
def test_token_logprobs(cuda, name, dtype):
    """The same bits as of a tensor laid out afresh, forward and backward."""
    from hydra_amd.kernels import token_logprobs

    g = torch.Generator().manual_seed(1)
    t = FORMS[name](g).to(dtype)
    view = torch.empty_strided(t.shape, t.stride(), dtype=dtype, device=cuda)
    view.copy_(t)
    plain = torch.empty(t.shape, dtype=dtype, device=cuda).copy_(t)
    tokens = torch.randint(0, t.shape[-1], t.shape[:-1], generator=g).to(cuda)
    k = min(3, t.shape[-1])
    outs = []
    for x in (view, plain):
        x.requires_grad_()
        with torch.no_grad():
            alone = token_logprobs(x, tokens, top_k=k)
        out = token_logprobs(x, tokens, top_k=k)
        for a, b in zip(alone, out):
            assert torch.equal(a, b)
        grad, = torch.autograd.grad([out.logprobs.sum() + 0.3 * out.entropy.sum() + 0.1 * out.top_logprobs.sum()], [x])
        assert grad.shape == x.shape
        outs.append((*out, grad))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    if t.numel():
        want = torch.log_softmax(t.double(), -1).gather(-1, tokens.cpu()[..., None])[..., 0]
        # one fp32 sum of 300 terms and a logarithm
        assert (outs[0][0].detach().cpu().double() - want).abs().max() < 1e-5


@pytest.mark.parametrize("name", list(FORMS))
def test_swiglu_and_rms_norm(cuda, name):
    from hydra_amd.kernels import fused_rms_norm, fused_swiglu

    g = torch.Generator().manual_seed(2)
    t = FORMS[name](g)
    views = []
    for _ in range(2):
        v = torch.empty_strided(t.shape, t.stride(), device=cuda)
        views.append(v.copy_(torch.randn(t.shape, generator=g)).requires_grad_())
    plain = [torch.empty(t.shape, device=cuda).copy_(v.detach()).requires_grad_() for v in views]
    weight = torch.randn(t.shape[-1], generator=g).to(cuda)
    for op in (lambda a, b: fused_swiglu(a, b), lambda a, b: fused_rms_norm(a, weight) + 0 * b):
        outs = []
        for pair in (views, plain):
            y = op(*pair)
            outs.append((y, *torch.autograd.grad(y.square().sum(), pair)))
        for a, b in zip(*outs):
            assert a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("shape", [(0, 40), (3, 0, 40)])
def test_rms_norm_of_no_rows(cuda, shape):
    """A batch without rows has an empty gradient and the weight's is zero."""
    from hydra_amd.kernels import fused_rms_norm

    x = torch.zeros(shape, device=cuda, requires_grad=True)
    weight = torch.ones(40, device=cuda, requires_grad=True)
    y = fused_rms_norm(x, weight)
    gx, gw = torch.autograd.grad(y.sum(), [x, weight])
    assert y.shape == gx.shape == shape and gw.shape == (40,) and not gw.any()
