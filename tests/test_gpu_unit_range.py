"""maxsim_amd.normalize_embeddings and pack_normalized_documents where the
squares of a row leave fp32: rows longer than 1.8e19, and rows shorter than
1e-19 beside an eps that is shorter still."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._training_helpers import f64, rand
from .test_gpu_unit_rows import _check, _check_pack

pytestmark = pytest.mark.gpu

WIDE = [torch.float32, torch.bfloat16]  # fp16 holds no such numbers
FLT_MIN = 2.0 ** -126
DIMS = [1, 3, 77, 128, 300, 768, 2560, 16384]  # groups of 8 lanes to a workgroup of 1024


def _rows(gen, n, length, dim, dtype, sizes):
    """Rows of the sizes in turn: powers of two, so that they stay exact."""
    x = torch.randn(n, length, dim, generator=gen).clamp(-3, 3).to(dtype)
    size = torch.tensor(sizes, dtype=torch.float64)[torch.arange(n * length) % len(sizes)]
    return (x.double() * size.view(n, length, 1)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", WIDE, ids=str)
@pytest.mark.parametrize("dim", DIMS)
def test_long_rows(dim, dtype):
    # up to a few times below the largest number, ordinary rows between them
    gen = torch.Generator().manual_seed(dim)
    x = _rows(gen, 3, 5, dim, dtype, [1.0, 2.0 ** 60, 2.0 ** 70, 2.0 ** 100, 1.0, 2.0 ** 126, 2.0 ** 64])
    assert x.isfinite().all()
    # gradients of every size: dx is theirs over the row's length
    for scale in (1.0, 2.0 ** 40, 2.0 ** -20):
        dy = rand(gen, 3, 5, dim, dtype=dtype, scale=scale)
        _check(x, None, dy)
        lengths = torch.tensor([5, 0, 3], device="cuda")
        _check(x, lengths, dy)
        _check_pack(x, lengths, dy)


@pytest.mark.parametrize("dtype", WIDE, ids=str)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("eps", [1e-30, FLT_MIN, 1e-20])
def test_short_rows_and_a_shorter_eps(dim, dtype, eps):
    gen = torch.Generator().manual_seed(dim)
    x = _rows(gen, 3, 5, dim, dtype, [1.0, 2.0 ** -60, 2.0 ** -70, 2.0 ** -80, 0.0, 2.0 ** -95,
                                      2.0 ** -115])
    x[2, 4] = 2.0 ** -127  # subnormal
    # gradients that leave dx below the largest number
    size = x.float().abs().amax(-1, keepdim=True).clamp_min(eps).clamp_max(2.0 ** -30)
    dy = (rand(gen, 3, 5, dim) * size).to(dtype)
    _check(x, None, dy, eps=eps)
    lengths = torch.tensor([5, 0, 4], device="cuda")
    _check(x, lengths, dy, eps=eps)
    _check_pack(x, lengths, dy, eps=eps)


@pytest.mark.parametrize("dtype", WIDE, ids=str)
def test_zero_rows_at_the_smallest_eps(dtype):
    x = torch.zeros(2, 3, 128, dtype=dtype, device="cuda")
    x[0, 1] = 1
    leaf = x.clone().requires_grad_(True)
    y = maxsim_amd.normalize_embeddings(leaf, eps=FLT_MIN)
    assert torch.equal(y[0, 0], x[0, 0]) and torch.equal(y[1], x[1])
    dy = torch.full_like(x, 2.0 ** -100)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert (dx[1] == 2.0 ** 26).all() and (dx[0, 2] == 2.0 ** 26).all()


@pytest.mark.parametrize("dim", [8, 64, 128, 384, 768, 4096])
def test_neighbours_of_long_rows_keep_their_bits(dim):
    gen = torch.Generator().manual_seed(dim)
    x, dy = rand(gen, 4, 33, dim, dtype=torch.bfloat16), rand(gen, 4, 33, dim, dtype=torch.bfloat16)
    lengths = torch.tensor([33, 20, 0, 7], device="cuda")
    for ln in (None, lengths):
        clean, clean_dx = _check(x, ln, dy)
        z = x.clone()
        z[:, ::5] *= 2.0 ** 100
        z[1, 3], z[1, 6, 0] = float("inf"), float("nan")
        leaf = z.requires_grad_(True)
        y = maxsim_amd.normalize_embeddings(leaf, ln)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        keep = torch.ones(4, 33, dtype=torch.bool, device="cuda")
        keep[:, ::5] = keep[1, 3] = keep[1, 6] = False
        assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])
        # scaling a row by a power of two scales nothing in y
        long = torch.zeros_like(keep)
        long[:, ::5] = True
        assert torch.equal(y[long], clean[long])
        assert y[1, 3].isnan().all() and y[1, 6].isnan().all()


def test_a_small_eps_without_short_rows_changes_nothing():
    gen = torch.Generator().manual_seed(1)
    x, dy = rand(gen, 3, 50, 128), rand(gen, 3, 50, 128)
    a, b = _check(x, None, dy), _check(x, None, dy, eps=FLT_MIN)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_large_gradients_of_ordinary_rows():
    # <x, dy> past fp32, dx far below its largest number
    gen = torch.Generator().manual_seed(2)
    x = _rows(gen, 2, 5, 128, torch.float32, [2.0 ** 50])
    dy = rand(gen, 2, 5, 128, scale=2.0 ** 90)
    _check(x, None, dy)


def test_refuses_an_eps_below_the_normal_numbers():
    x = torch.zeros(2, 3, 64, device="cuda")
    lengths = torch.tensor([3, 1], device="cuda")
    for eps in (1e-39, 1e-46, 1e-300, 0.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            maxsim_amd.normalize_embeddings(x, eps=eps)
        with pytest.raises(ValueError, match="eps"):
            maxsim_amd.pack_normalized_documents(x, lengths, eps=eps)


def test_oracle_divides_by_the_length():
    # the reference here is float64: its squares stay in range
    x = np.array([[[3e38, 0.0, 4e37]]])
    assert np.allclose((oracle.unit_rows(x, None, 1e-12) ** 2).sum(), 1.0)
    assert f64(torch.tensor([2.0 ** 127])).tolist() == [2.0 ** 127]


def test_more_than_two_to_the_31_rows():
    # [rows, dim] is one axis of rows, as long as memory has room for
    rows = 2 ** 31 + 5
    x = torch.ones(rows, 1, dtype=torch.float16, device="cuda")
    tail = torch.tensor([-3.0, 0.0, 5.0, 2.0 ** -20, -1.0], device="cuda").half()[:, None]
    x[-5:] = tail
    leaf = x.requires_grad_(True)
    y = maxsim_amd.normalize_embeddings(leaf)
    assert y.shape == x.shape and torch.equal(y[-5:].detach(), tail.sign())
    assert bool((y[:-5] == 1).all())
    del y
    y = maxsim_amd.normalize_embeddings(leaf, eps=0.5)  # below it the gradient is dy / eps
    (dx,) = torch.autograd.grad(y, leaf, torch.ones((1, 1), dtype=torch.float16,
                                                    device="cuda").expand(rows, 1))
    assert dx[-5:, 0].tolist() == [0.0, 2.0, 0.0, 2.0, 0.0] and bool((dx[:-5] == 0).all())
