"""The gradients' norm, the factor and clipping outside plain calls (CPU only: fake
tensors go through their autograd entry and launch nothing)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses import FakeTensorMode

import maxsim_amd


@pytest.fixture(autouse=True)
def _fake():
    with FakeTensorMode():
        yield


def _new(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _others():
    return [_new(5), _new(7, 3, dtype=torch.bfloat16)]


FUNCTIONS = {
    "grad_norm": lambda t: maxsim_amd.grad_norm(t),
    "grad_norm of a list": lambda t: maxsim_amd.grad_norm([*_others(), t]),
    "clip_factor": lambda t: maxsim_amd.clip_factor([t, *_others()], 1.0)[1],
    "clip_factor, last": lambda t: maxsim_amd.clip_factor([*_others(), t], 1.0)[0],
    "clip_grad_norm": lambda t: maxsim_amd.clip_grad_norm([t, *_others()], 1.0),
    "clip_grad_norm, last": lambda t: maxsim_amd.clip_grad_norm([*_others(), t], 1.0),
}


@pytest.mark.parametrize("name", FUNCTIONS)
def test_forward_mode_raises(name):
    # a tangent that is dropped would count as 0
    f = FUNCTIONS[name]
    with forward_ad.dual_level():
        primal = _new(4, 6)
        dual = forward_ad.make_dual(primal, _new(4, 6))
        with pytest.raises(NotImplementedError, match="forward mode"):
            f(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            f(dual)
        with forward_ad._set_fwd_grad_enabled(False):
            assert forward_ad.unpack_dual(f(dual)).tangent is None  # not asked for
        assert forward_ad.unpack_dual(f(primal)).tangent is None  # without a tangent as ever


@pytest.mark.parametrize("name", FUNCTIONS)
def test_func_jvp_raises(name):
    with pytest.raises(RuntimeError):
        torch.func.jvp(FUNCTIONS[name], (_new(4, 6),), (_new(4, 6),))


@pytest.mark.parametrize("name", FUNCTIONS)
def test_nothing_is_recorded(name):
    # documented: constants to what is computed from them
    leaf = _new(4, 6).requires_grad_(True)
    assert not FUNCTIONS[name](leaf * 2).requires_grad
