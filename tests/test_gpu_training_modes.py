"""The operators around the scores under torch's transforms: batched by vmap as
one by one, refused where there is no derivative."""

from __future__ import annotations

import pytest
import torch

import maxsim_amd

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:There is a performance drop")]


def test_vmap():
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(3, 4, 5, 64, generator=gen, device="cuda")
    w = torch.randn(64, generator=gen, device="cuda", requires_grad=True)
    lengths = torch.randint(0, 6, (3, 4), generator=gen, device="cuda", dtype=torch.int32)
    got = torch.vmap(maxsim_amd.normalize_embeddings)(x, lengths)
    want = torch.stack([maxsim_amd.normalize_embeddings(a, b) for a, b in zip(x, lengths)])
    assert torch.equal(got, want)
    got = torch.vmap(lambda t: maxsim_amd.layer_norm(t, w), in_dims=1, out_dims=1)(x)
    want = torch.stack([maxsim_amd.layer_norm(t, w) for t in x.unbind(1)], 1)
    assert torch.equal(got, want)
    down = torch.randn(x.shape, generator=gen, device="cuda")
    a, b = (torch.autograd.grad(y, w, down)[0] for y in (got, want))
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-4)


def test_batched_gradients():
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(4, 5, 64, generator=gen, device="cuda", requires_grad=True)
    y = maxsim_amd.normalize_embeddings(x)
    down = torch.randn(3, 4, 5, 64, generator=gen, device="cuda")
    got, = torch.autograd.grad(y, x, down, is_grads_batched=True, retain_graph=True)
    want = [torch.autograd.grad(y, x, d, retain_graph=True)[0] for d in down]
    assert torch.equal(got, torch.stack(want))


def test_transforms_without_a_derivative_raise():
    x, w = torch.randn(4, 64, device="cuda"), torch.randn(64, device="cuda")
    for f in (lambda t: maxsim_amd.layer_norm(t, w), maxsim_amd.normalize_embeddings):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x)
        with pytest.raises(NotImplementedError, match="forward mode"):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(RuntimeError, match="no derivative"):
            torch.autograd.functional.hvp(lambda t: f(t).square().sum(), x, x)
