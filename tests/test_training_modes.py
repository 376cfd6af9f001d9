"""What the operators around the scores do outside plain reverse mode (CPU only:
fake tensors go through their autograd entry and launch nothing)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses import FakeTensorMode

import maxsim_amd
from maxsim_amd._ops import ops


@pytest.fixture(autouse=True)
def _fake():
    with FakeTensorMode():
        yield


def _rows(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


# name -> (function of the tensor that carries the tangent, that tensor's shape)
FUNCTIONS = {
    "layer_norm x": (lambda t: maxsim_amd.layer_norm(t, _rows(64), _rows(64)), (4, 64)),
    "layer_norm weight": (lambda t: maxsim_amd.layer_norm(_rows(4, 64), t), (64,)),
    "layer_norm bias": (lambda t: maxsim_amd.layer_norm(_rows(4, 64), None, t), (64,)),
    "normalize_embeddings": (maxsim_amd.normalize_embeddings, (4, 5, 64)),
    "normalize_embeddings with lengths": (
        lambda t: maxsim_amd.normalize_embeddings(t, _rows(4, dtype=torch.int32)), (4, 5, 64)),
    "pack_normalized_documents": (
        lambda t: ops.maxsim_pack_normalized(t, _rows(4, dtype=torch.int32),
                                             _rows(5, dtype=torch.int32), 7, 1e-12), (4, 5, 64)),
}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", FUNCTIONS)
def test_forward_mode_raises(name, requires_grad):
    # a tangent that is dropped would count as 0
    f, shape = FUNCTIONS[name]
    with forward_ad.dual_level():
        primal = _rows(*shape).requires_grad_(requires_grad)
        dual = forward_ad.make_dual(primal, _rows(*shape))
        with pytest.raises(NotImplementedError, match="forward mode"):
            f(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            f(dual)
        with forward_ad._set_fwd_grad_enabled(False):
            assert forward_ad.unpack_dual(f(dual)).tangent is None  # not asked for
        assert forward_ad.unpack_dual(f(primal)).tangent is None  # without a tangent as ever


@pytest.mark.parametrize("name", FUNCTIONS)
def test_func_jvp_raises(name):
    f, shape = FUNCTIONS[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (_rows(*shape),), (_rows(*shape),))
