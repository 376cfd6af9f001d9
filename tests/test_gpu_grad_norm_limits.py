"""The gradients' norm and clipping at the ends of what their arguments may be:
limits and eps of zero, gradients of zeros."""

from __future__ import annotations

import math

import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._helpers import DTYPES

pytestmark = pytest.mark.gpu

SIZES = [[1], [5, 0, 300], [40001, 7], [3_000_000]]  # one launch, several, large shares


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("max_norm,eps", [(0.0, 0.0), (0.0, 1e-6), (1.0, 0.0), (math.inf, 0.0)])
def test_gradients_of_zeros_stay_zeros(max_norm, eps, sizes, dtype):
    # with eps = 0 the factor's quotient is 0 / 0 or x / 0
    grads = [torch.zeros(n, dtype=dtype, device="cuda") for n in sizes]
    norm, factor = maxsim_amd.clip_factor(grads, max_norm, eps=eps)
    assert float(norm) == 0.0 and float(factor) == oracle.clip_factor(0.0, max_norm, eps)
    assert float(maxsim_amd.clip_grad_norm(grads, max_norm, eps=eps)) == 0.0
    assert all(bool((g == 0).all()) for g in grads)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_a_limit_of_zero_clears(dtype):
    for eps in (0.0, 1e-6):
        grads = [torch.ones(300, dtype=dtype, device="cuda"), torch.zeros(9, dtype=dtype, device="cuda")]
        assert float(maxsim_amd.clip_factor(grads, 0.0, eps=eps)[1]) == 0.0
        maxsim_amd.clip_grad_norm(grads, 0.0, eps=eps)
        assert not any(bool(g.any()) for g in grads)


def test_a_step_on_gradients_of_zeros():
    p = torch.ones(100, device="cuda")
    m, v, g = (torch.zeros_like(p) for _ in range(3))
    _, factor = maxsim_amd.clip_factor([g], 0.0, eps=0.0)
    maxsim_amd.adamw_step([p], [g], [m], [v], step=1, weight_decay=0.0, grad_scale=factor)
    assert bool((p == 1).all()) and not m.any() and not v.any()


def test_no_gradients_have_a_norm_on_the_device():
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    try:
        norm, factor = maxsim_amd.clip_factor([], 1.0)
        results = [norm, maxsim_amd.grad_norm([]), maxsim_amd.clip_grad_norm((), 1.0), factor]
    finally:
        torch.set_default_dtype(before)
    for t, want in zip(results, (0.0, 0.0, 0.0, 1.0)):
        assert t.is_cuda and t.dtype == torch.float32 and t.shape == () and float(t) == want


def test_the_optimizer_without_gradients_has_its_norm_on_the_device():
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    opt = maxsim_amd.AdamW([p], max_norm=1.0)
    opt.step()
    assert opt.grad_norm.is_cuda and opt.grad_norm.dtype == torch.float32
    assert float(opt.grad_norm) == 0.0 and bool((p == 1).all())
    p.grad = torch.full_like(p, 2.0)
    opt.step()
    kept, p.grad = p.detach().clone(), None
    opt.step()  # the norm is the last step's, not the one before
    assert float(opt.grad_norm) == 0.0 and torch.equal(p, kept)
