"""The gradients' norm, the factor and clipping under torch's transforms: refused
where a derivative or a batch would be dropped, and nothing clipped then."""

from __future__ import annotations

import pytest
import torch

import maxsim_amd

from ._training_helpers import rand

pytestmark = pytest.mark.gpu


def _grads(seed):
    gen = torch.Generator().manual_seed(seed)
    return [rand(gen, 40, 7), rand(gen, 70001, dtype=torch.bfloat16), rand(gen, 3, 4, 5)]


def test_tangents_are_refused_before_anything_is_written():
    grads = _grads(0)
    before = [g.clone() for g in grads]
    for at, f in enumerate((lambda t: maxsim_amd.grad_norm([t, *grads]),
                            lambda t: maxsim_amd.clip_factor([*grads, t], 0.01)[1],
                            lambda t: maxsim_amd.clip_grad_norm([*grads, t], 0.01))):
        x = rand(torch.Generator().manual_seed(at), 33)
        kept = x.clone()
        with pytest.raises(NotImplementedError, match="forward mode"):
            torch.func.jvp(f, (x,), (x,))
        assert torch.equal(x, kept)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))


def test_batches_are_refused():
    x = rand(torch.Generator().manual_seed(3), 3, 50)
    for f in (lambda t: maxsim_amd.grad_norm([t]), lambda t: maxsim_amd.clip_grad_norm([t], 1.0)):
        with pytest.raises(RuntimeError, match="[Bb]atching rule"):
            torch.vmap(f)(x)


def test_gradients_with_a_graph():
    # documented: the norm is a constant, the clipped values are what is read
    p = rand(torch.Generator().manual_seed(4), 50).requires_grad_(True)
    (g,) = torch.autograd.grad(p.square().sum(), p, create_graph=True)
    want = maxsim_amd.clip_factor([g.detach().clone()], 0.5)
    norm, factor = maxsim_amd.clip_factor([g], 0.5)
    assert not norm.requires_grad and not factor.requires_grad
    assert torch.equal(norm, want[0]) and torch.equal(factor, want[1])
    kept = g.detach().clone()
    assert torch.equal(maxsim_amd.clip_grad_norm([g], 0.5), norm)
    assert torch.equal(g.detach(), kept * factor)


@pytest.mark.parametrize("dynamic", [None, True])
def test_compiled(dynamic):
    torch._dynamo.reset()
    compiled = lambda f: torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=dynamic)

    def clip(a, b, c):
        return maxsim_amd.clip_grad_norm([a, b, c], 0.5), a * 2  # reads what was clipped

    def step(p, g, m, v, at):
        norm, factor = maxsim_amd.clip_factor([g], 0.5)
        maxsim_amd.adamw_step([p], [g], [m], [v], step=at, grad_scale=factor)
        return norm, factor

    fast, fast_step = compiled(clip), compiled(step)
    for seed in (5, 6):
        x, y = _grads(seed), _grads(seed)
        assert all(torch.equal(a, b) for a, b in zip(fast(*x), clip(*y)))
        assert all(torch.equal(a, b) for a, b in zip(x, y))
        x, y = ([rand(torch.Generator().manual_seed(seed), 500 + seed) for _ in range(2)] +
                [torch.zeros(500 + seed, device="cuda") for _ in range(2)] +
                [torch.ones(1, dtype=torch.int64, device="cuda")] for _ in range(2))
        assert all(torch.equal(a, b) for a, b in zip(fast_step(*x), step(*y)))
        assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_parameters_are_not_clipped_in_place_of_gradients():
    # torch.nn.utils.clip_grad_norm_ takes parameters: the same call here would
    # have scaled the weights themselves
    p = torch.nn.Parameter(rand(torch.Generator().manual_seed(7), 50))
    q = torch.nn.Parameter(rand(torch.Generator().manual_seed(8), 70, dtype=torch.bfloat16))
    kept = [p.detach().clone(), q.detach().clone()]
    for call in (lambda: maxsim_amd.clip_grad_norm([p, q], 1e-3),
                 lambda: maxsim_amd.clip_grad_norm([kept[0].clone(), q], 1e-3),
                 lambda: maxsim_amd.clip_grad_norm(p, 1e-3)):
        with pytest.raises(RuntimeError, match="leaf that requires grad"):
            call()
    assert torch.equal(p.detach(), kept[0]) and torch.equal(q.detach(), kept[1])
    (p.sum() + q.sum()).backward()
    grads = [p.grad, q.grad]  # what is meant
    maxsim_amd.clip_grad_norm(grads, 1e-3)
    assert float(maxsim_amd.grad_norm(grads)) < 1.1e-3
    with torch.no_grad():
        maxsim_amd.clip_grad_norm([p], 0.5)
    assert float(maxsim_amd.grad_norm([p])) <= 0.5 * (1 + 2.0 ** -22)
    # their norm is nothing that writes
    assert float(maxsim_amd.grad_norm([q])) > 0
