"""maxsim_amd.layer_norm against the float64 oracle: every shape of the row
kernels, types, layouts, rows that are not finite, and its refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._helpers import DTYPES, one_element_off
from ._training_helpers import assert_within, f64, rand

pytestmark = pytest.mark.gpu


def _grads(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in (x, w, b)]
    y = maxsim_amd.layer_norm(*args, eps=eps)
    return y.detach(), torch.autograd.grad(y, leaves, dy)


def _check(x, w, b, dy, eps=1e-5):
    """Forward and every gradient, against the formulas."""
    y, grads = _grads(x, w, b, dy, eps)
    dim = x.shape[-1]
    xn, dn = f64(x).reshape(-1, dim), f64(dy).reshape(-1, dim)
    wn, bn = (None if t is None else f64(t) for t in (w, b))
    want = oracle.layer_norm(xn, wn, bn, eps)[0]
    assert y.dtype == x.dtype and y.shape == x.shape
    assert_within(y.reshape(-1, dim), want, oracle.layer_norm_error(xn, wn, bn, eps), "y")
    dx, dw, db = oracle.layer_norm_backward(dn, xn, wn, eps)
    ex, ew, eb = oracle.layer_norm_backward_error(dn, xn, wn, eps)
    assert_within(grads[0].reshape(-1, dim), dx, ex, "dx")
    rest = list(grads[1:])
    for t, g, e, name in ((w, dw, ew, "dw"), (b, db, eb, "db")):
        if t is not None:
            got = rest.pop(0)
            assert got.dtype == t.dtype
            assert_within(got, g, e, name)
    return y, grads


# one width at least for each shape of the kernels, whole and cut chunks
WIDTHS = [1, 2, 7, 8, 60, 64, 77, 128, 129, 250, 256, 300, 301, 384, 389, 500, 512, 768, 770, 1024,
          1500, 1536, 2048, 2500, 2560, 4096, 4099, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", WIDTHS)
def test_widths(dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    rows = 37 if dim <= 1024 else 5
    x = rand(gen, rows, dim, dtype=dtype) * 2 + 0.5
    _check(x, rand(gen, dim, dtype=dtype), rand(gen, dim, dtype=dtype),
           rand(gen, rows, dim, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim", [77, 768, 2560, 16384])
def test_weights_in_32_bits(dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    _check(rand(gen, 9, dim, dtype=dtype), rand(gen, dim), rand(gen, dim),
           rand(gen, 9, dim, dtype=dtype))


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 33, 257, 1031, 20011])
@pytest.mark.parametrize("dim", [96, 768])
def test_rows(rows, dim):
    # fewer rows than a workgroup holds up to several turns of every one
    gen = torch.Generator().manual_seed(rows)
    _check(rand(gen, rows, dim, dtype=torch.bfloat16), rand(gen, dim), rand(gen, dim),
           rand(gen, rows, dim, dtype=torch.bfloat16))


@pytest.mark.parametrize("dim", [301, 2560])
def test_many_turns_of_wide_and_odd_rows(dim):
    gen = torch.Generator().manual_seed(dim)
    _check(rand(gen, 4099, dim), rand(gen, dim), rand(gen, dim), rand(gen, 4099, dim))


@pytest.mark.parametrize("given", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(given):
    gen = torch.Generator().manual_seed(3)
    w = rand(gen, 300, dtype=torch.bfloat16) if given[0] else None
    b = rand(gen, 300, dtype=torch.bfloat16) if given[1] else None
    _check(rand(gen, 19, 300, dtype=torch.bfloat16), w, b, rand(gen, 19, 300, dtype=torch.bfloat16))


def test_layouts():
    gen = torch.Generator().manual_seed(4)
    w, b = rand(gen, 100), rand(gen, 100)
    full = rand(gen, 6, 9, 108, dtype=torch.bfloat16)
    dy = rand(gen, 6, 9, 100, dtype=torch.bfloat16)
    _check(full[..., :100], w, b, dy)                       # rows further apart
    _check(full[:, 1:, 3:103], w, b, dy[:, 1:])             # not one run of rows
    _check(full[..., :100].transpose(0, 1), w, b, dy.transpose(0, 1))
    _check(one_element_off(full[..., :100].contiguous()), one_element_off(w), one_element_off(b),
           one_element_off(dy))
    _check(full[..., :100], w, b, dy[0, 0].expand(6, 9, 100))     # one gradient row for all
    _check(full[..., :100], w, b, dy[..., :1].expand(6, 9, 100))  # one value for a row
    _check(full[0, 0, :100].expand(7, 100), w, b, dy.reshape(-1, 100)[:7])
    _check(full[0, 0, :100], w, b, dy[0, 0])                # a single row, 1-D
    _check(rand(gen, 100, 40, dtype=torch.bfloat16).t(), w, b, dy.reshape(-1, 100)[:40])


def test_large_mean_keeps_the_small_differences():
    # a difference of mean squares would lose all of the variance
    gen = torch.Generator().manual_seed(5)
    x = rand(gen, 13, 768) + 4096.0
    _check(x, rand(gen, 768), rand(gen, 768), rand(gen, 13, 768))


def test_constant_rows_give_the_bias():
    x = torch.full((3, 512), 7.25, device="cuda")
    b = torch.randn(512, device="cuda")
    y, (dx, dw, db) = _grads(x, torch.ones(512, device="cuda"), b, torch.ones_like(x))
    assert (y == b).all() and (dw == 0).all() and (db == 3).all()
    assert (dx.abs() <= 1e-4).all()  # (1 - mean of 1) / sqrt(eps)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [96, 4099])
def test_a_row_that_is_not_finite_stays_alone(bad, dim):
    gen = torch.Generator().manual_seed(6)
    x = rand(gen, 21, dim, dtype=torch.bfloat16)
    w, b, dy = rand(gen, dim), rand(gen, dim), rand(gen, 21, dim, dtype=torch.bfloat16)
    clean, (clean_dx, _, clean_db) = _grads(x, w, b, dy)
    x2 = x.clone()
    x2[5, dim - 1] = bad
    y, (dx, dw, db) = _grads(x2, w, b, dy)
    keep = torch.arange(21, device="cuda") != 5
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])
    assert y[5].isnan().all() and dx[5].isnan().all()
    assert dw.isnan().all() and torch.equal(db, clean_db)


def test_empty():
    w = torch.randn(64, device="cuda", requires_grad=True)
    x = torch.randn(0, 3, 64, device="cuda", requires_grad=True)
    y = maxsim_amd.layer_norm(x, w, w)
    assert y.shape == (0, 3, 64)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and (dw == 0).all()


def test_only_what_is_asked_for():
    gen = torch.Generator().manual_seed(7)
    x, dy = rand(gen, 31, 384), rand(gen, 31, 384)
    w, b = rand(gen, 384), rand(gen, 384)
    _, (dx, dw, db) = _grads(x, w, b, dy)
    for wanted in ([0], [1], [2], [0, 2], [1, 2]):
        args = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(maxsim_amd.layer_norm(*args), [args[i] for i in wanted], dy)
        for i, g in zip(wanted, got):
            assert torch.equal(g, (dx, dw, db)[i])
    # all require one, one is asked for
    args = [t.detach().requires_grad_(True) for t in (x, w, b)]
    (g,) = torch.autograd.grad(maxsim_amd.layer_norm(*args), args[2], dy)
    assert torch.equal(g, db)
    assert not maxsim_amd.layer_norm(x, w, b).requires_grad
    with torch.no_grad():
        assert torch.equal(maxsim_amd.layer_norm(*args), maxsim_amd.layer_norm(x, w, b))


def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(8)
    x, w, b, dy = rand(gen, 7, 200), rand(gen, 200), rand(gen, 200), rand(gen, 7, 200)
    _, grads = _grads(x, w, b, dy)
    host = [f64(t) for t in (x, w, b)]
    for i, g in enumerate(grads):
        v = np.random.RandomState(i).randn(*host[i].shape)
        h = 1e-5
        f = [(oracle.layer_norm(*[a + s * h * v if j == i else a for j, a in enumerate(host)],
                                1e-5)[0] * f64(dy)).sum() for s in (1, -1)]
        # fp32 gradients: their own rounding, summed over the direction
        size = float(np.abs(f64(g) * v).sum())
        assert abs((f64(g) * v).sum() - (f[0] - f[1]) / (2 * h)) <= 1e-5 * size


def test_same_bits_every_time():
    gen = torch.Generator().manual_seed(9)
    x, dy = rand(gen, 30011, 96, dtype=torch.bfloat16), rand(gen, 30011, 96, dtype=torch.bfloat16)
    w, b = rand(gen, 96), rand(gen, 96)
    y, grads = _grads(x, w, b, dy)
    for _ in range(3):
        y2, grads2 = _grads(x, w, b, dy)
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(grads, grads2))


def test_rows_past_two_to_the_31_elements():
    rows, dim = 2 ** 31 // 16384 + 3, 16384
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(10)
    tail = rand(gen, 3, dim, dtype=torch.bfloat16)
    x[-3:] = tail
    w, b, dy = rand(gen, dim), rand(gen, dim), rand(gen, 3, dim, dtype=torch.bfloat16)
    d = torch.zeros_like(x)
    d[-3:] = dy
    y, (dx, dw, _) = _grads(x, w, b, d)
    y3, (dx3, _, _) = _grads(tail, w, b, dy)
    assert torch.equal(y[-3:], y3) and torch.equal(dx[-3:], dx3)
    assert torch.equal(y[0], b.to(torch.bfloat16)) and (dx[:-3] == 0).all()
    dwn = oracle.layer_norm_backward(f64(dy), f64(tail), f64(w), 1e-5)[1]
    assert_within(dw, dwn, oracle.layer_norm_backward_error(f64(dy), f64(tail), f64(w), 1e-5)[1])


def test_on_another_stream_and_in_a_graph():
    gen = torch.Generator().manual_seed(11)
    x = rand(gen, 64, 768, dtype=torch.bfloat16).requires_grad_(True)
    w, b = rand(gen, 768).requires_grad_(True), rand(gen, 768).requires_grad_(True)
    dy = rand(gen, 64, 768, dtype=torch.bfloat16)

    def step():
        y = maxsim_amd.layer_norm(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(rand(torch.Generator().manual_seed(20 + k), 64, 768, dtype=torch.bfloat16))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_compiles():
    gen = torch.Generator().manual_seed(12)
    x = rand(gen, 6, 5, 96, dtype=torch.bfloat16).requires_grad_(True)
    w, b = rand(gen, 96).requires_grad_(True), rand(gen, 96).requires_grad_(True)

    def f(x, w, b):
        return maxsim_amd.layer_norm(x * 2, w, b).float().square().sum()

    want = torch.autograd.grad(f(x, w, b), (x, w, b))
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x, w, b),
                              (x, w, b))
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    w = torch.randn(64, device="cuda")
    cases = [
        (RuntimeError, "HIP", lambda: maxsim_amd.layer_norm(x.cpu(), w)),
        (TypeError, "x must be", lambda: maxsim_amd.layer_norm(x.double(), w)),
        (TypeError, "weight must be", lambda: maxsim_amd.layer_norm(x, w.int())),
        (TypeError, "weight must be", lambda: maxsim_amd.layer_norm(x, w.half())),
        (TypeError, "same dtype", lambda: maxsim_amd.layer_norm(x.half(), w.half(), w)),
        (ValueError, "weight must have shape", lambda: maxsim_amd.layer_norm(x, w[:63])),
        (ValueError, "bias must have shape", lambda: maxsim_amd.layer_norm(x, w, w[None])),
        (ValueError, "eps", lambda: maxsim_amd.layer_norm(x, w, eps=-1e-5)),
        (ValueError, "eps", lambda: maxsim_amd.layer_norm(x, w, eps=float("nan"))),
        (ValueError, "dim must be > 0", lambda: maxsim_amd.layer_norm(x[:, :0])),
        (ValueError, "1 dimension", lambda: maxsim_amd.layer_norm(x[0, 0])),
        (RuntimeError, "same device", lambda: maxsim_amd.layer_norm(x, w.cpu())),
        (RuntimeError, "16384", lambda: maxsim_amd.layer_norm(torch.zeros(1, 16385, device="cuda"))),
    ]
    for error, text, f in cases:
        with pytest.raises(error, match=text):
            f()


@pytest.mark.parametrize("of", ["x", "weight", "bias"])
def test_a_second_derivative_raises(of):
    leaves = {"x": torch.randn(5, 64, device="cuda", requires_grad=True),
              "weight": torch.ones(64, device="cuda", requires_grad=True),
              "bias": torch.zeros(64, device="cuda", requires_grad=True)}
    y = maxsim_amd.layer_norm(*leaves.values())
    once, = torch.autograd.grad(y.square().sum(), leaves[of], retain_graph=True)
    grad, = torch.autograd.grad(y.square().sum(), leaves[of], create_graph=True)
    assert torch.equal(once, grad)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(grad.square().sum(), leaves["x"])
