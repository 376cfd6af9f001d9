"""maxsim_amd.normalize_embeddings and pack_normalized_documents against the
float64 oracle: shapes, types, lengths, padding that holds anything, layouts,
and their refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import maxsim_amd
from oracle import training_oracle as oracle

from ._helpers import DTYPES, one_element_off
from ._training_helpers import U32, assert_within, f64, rand

pytestmark = pytest.mark.gpu

EPS = 1e-12


def _np3(x):
    return f64(x).reshape((-1, x.shape[-2], x.shape[-1]) if x.dim() >= 2 else (1, 1, -1))


def _check(x, lengths, dy, eps=EPS):
    leaf = x.detach().requires_grad_(True)
    y = maxsim_amd.normalize_embeddings(leaf, lengths, eps=eps)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert y.shape == x.shape and y.dtype == x.dtype and dx.dtype == x.dtype
    ln = None if lengths is None else lengths.cpu().numpy()
    xn, dn = _np3(x), _np3(dy)
    want = oracle.unit_rows(xn, ln, eps)
    # n additions in a chain and a tree, a root and a quotient
    assert_within(y.detach().reshape(want.shape), want, 60 * U32 * np.abs(want), "y")
    assert_within(dx.reshape(want.shape), oracle.unit_rows_backward(dn, xn, ln, eps),
                  oracle.unit_rows_backward_error(dn, xn, ln, eps), "dx")
    return y.detach(), dx


def _check_pack(x, lengths, dy_padded, eps=EPS):
    """dy_padded [N, L, D]: its real rows are what comes down."""
    ln = np.clip(lengths.cpu().numpy(), 0, x.shape[1])
    real = oracle.real_tokens(x.shape, ln)
    leaf = x.detach().requires_grad_(True)
    docs, offsets = maxsim_amd.pack_normalized_documents(leaf, lengths, eps=eps)
    assert docs.dtype == x.dtype and offsets.dtype == torch.int32
    assert offsets.tolist() == [0, *np.cumsum(ln).tolist()]
    assert docs.shape == (int(ln.sum()), x.shape[2])
    want = oracle.unit_rows(f64(x), ln, eps)[real]
    assert_within(docs.detach(), want, 60 * U32 * np.abs(want), "documents")
    dy = dy_padded[torch.from_numpy(real).to(x.device)]
    (dx,) = torch.autograd.grad(docs, leaf, dy)
    assert_within(dx, oracle.unit_rows_backward(f64(dy_padded), f64(x), ln, eps),
                  oracle.unit_rows_backward_error(f64(dy_padded), f64(x), ln, eps), "dx")
    return docs.detach(), offsets


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [1, 3, 8, 64, 77, 96, 128, 130, 256, 300, 384, 500, 768, 1030, 2560,
                                 4099, 8192, 16384])
def test_widths(dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    x = rand(gen, 3, 5, dim, dtype=dtype, scale=3.0)
    dy = rand(gen, 3, 5, dim, dtype=dtype)
    _check(x, None, dy)
    lengths = torch.tensor([5, 0, 2], dtype=torch.int32, device="cuda")
    _check(x, lengths, dy)
    _check_pack(x, lengths, dy)


@pytest.mark.parametrize("n,length", [(1, 1), (1, 700), (700, 1), (37, 61), (3000, 40)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_sequences(n, length, index):
    gen = torch.Generator().manual_seed(n)
    x = rand(gen, n, length, 128, dtype=torch.bfloat16)
    dy = rand(gen, n, length, 128, dtype=torch.bfloat16)
    lengths = torch.randint(0, length + 1, (n,), generator=gen).to(index).cuda()
    _check(x, lengths, dy)
    _check_pack(x, lengths, dy)


def test_every_length_from_none_to_all():
    gen = torch.Generator().manual_seed(1)
    x, dy = rand(gen, 34, 33, 96, dtype=torch.float16), rand(gen, 34, 33, 96, dtype=torch.float16)
    lengths = torch.arange(34, device="cuda")
    _check(x, lengths, dy)
    _check_pack(x, lengths, dy)
    _check_pack(x, torch.zeros_like(lengths), dy)  # no row at all


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_padding_may_hold_anything(bad):
    gen = torch.Generator().manual_seed(2)
    x, dy = rand(gen, 5, 7, 128, dtype=torch.bfloat16), rand(gen, 5, 7, 128, dtype=torch.bfloat16)
    lengths = torch.tensor([7, 3, 0, 1, 6], device="cuda")
    pad = torch.arange(7, device="cuda") >= lengths[:, None]
    want = _check(x, lengths, dy), _check_pack(x, lengths, dy)
    x2, dy2 = x.clone(), dy.clone()
    x2[pad], dy2[pad] = bad, bad
    leaf = x2.requires_grad_(True)
    y = maxsim_amd.normalize_embeddings(leaf, lengths)
    (dx,) = torch.autograd.grad(y, leaf, dy2)
    assert torch.equal(y, want[0][0]) and torch.equal(dx, want[0][1])
    docs, _ = maxsim_amd.pack_normalized_documents(leaf, lengths)
    assert torch.equal(docs, want[1][0])
    (dx,) = torch.autograd.grad(docs, leaf, dy[~pad])
    assert torch.equal(dx, want[0][1])


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_lengths_out_of_range_are_clamped(index):
    gen = torch.Generator().manual_seed(3)
    x, dy = rand(gen, 6, 9, 64), rand(gen, 6, 9, 64)
    far = 2 ** 31 - 1 if index == torch.int32 else 2 ** 32 + 1  # wraps to 1 where it is cut short
    lengths = torch.tensor([far, -1, -far, 9, 10, 4], dtype=index, device="cuda")
    _check(x, lengths, dy)
    _check_pack(x, lengths, dy)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_short_and_zero_rows(dtype):
    # below eps a row is divided by eps, and its gradient has no second part
    gen = torch.Generator().manual_seed(4)
    x, dy = rand(gen, 2, 4, 128, dtype=dtype), rand(gen, 2, 4, 128, dtype=dtype)
    x[0, 1] = 0
    x[1, 2] *= 2.0 ** -12
    _check(x, None, dy, eps=0.25)
    y = maxsim_amd.normalize_embeddings(x)
    assert (y[0, 1] == 0).all()


def test_rows_that_are_not_finite_stay_alone():
    gen = torch.Generator().manual_seed(5)
    x, dy = rand(gen, 6, 128, dtype=torch.bfloat16), rand(gen, 6, 128, dtype=torch.bfloat16)
    clean, clean_dx = _check(x, None, dy)
    x[1, 5], x[4, 127] = float("nan"), float("inf")
    leaf = x.requires_grad_(True)
    y = maxsim_amd.normalize_embeddings(leaf)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])
    # as the quotient: inf / inf is NaN, a number / inf is 0
    assert y[1].isnan().all() and y[4, 127].isnan() and (y[4, :127] == 0).all()
    assert dx[1].isnan().all()


def test_layouts():
    gen = torch.Generator().manual_seed(6)
    full = rand(gen, 5, 9, 136, dtype=torch.bfloat16)
    dy = rand(gen, 5, 9, 128, dtype=torch.bfloat16)
    lengths = torch.tensor([8, 0, 3, 1, 5], device="cuda")
    for x, d in ((full[..., 8:], dy), (full[:, 1:, :128], dy[:, 1:]),
                 (full[..., :128].transpose(0, 1), dy.transpose(0, 1)),
                 (one_element_off(dy), one_element_off(full[..., :128].contiguous())),
                 (full[..., :128], dy[0, 0].expand(5, 9, 128)),
                 (full[..., :128], dy[..., :1].expand(5, 9, 128)),
                 (full[0, 0, :128].expand(5, 9, 128), dy)):
        _check(x, None, d)
        if x.shape[0] == 5:
            _check(x, lengths, d)
            _check_pack(x, lengths, d)
    _check(full[0, :, :128], None, dy[0])
    _check(full[0, 0, :128], None, dy[0, 0])
    _check(full.view(5, 3, 3, 136)[..., :128], None, dy.view(5, 3, 3, 128))
    # a gradient of a sum: one value for everything
    leaf = full[..., :128].contiguous().requires_grad_(True)
    docs, _ = maxsim_amd.pack_normalized_documents(leaf, lengths)
    docs.float().sum().backward()
    want = oracle.unit_rows_backward(np.ones((5, 9, 128)), f64(leaf), lengths.cpu().numpy(), EPS)
    assert_within(leaf.grad, want, oracle.unit_rows_backward_error(
        np.ones((5, 9, 128)), f64(leaf), lengths.cpu().numpy(), EPS))


def test_empty():
    for shape in ((0, 4, 64), (3, 0, 64), (0, 64)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        y = maxsim_amd.normalize_embeddings(x)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape
    docs, off = maxsim_amd.pack_normalized_documents(
        torch.randn(0, 4, 64, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert docs.shape == (0, 64) and off.tolist() == [0]


def test_rows_past_two_to_the_31_elements():
    n, length, dim = 2 ** 31 // (128 * 1024) + 1, 1024, 128
    x = torch.zeros(n, length, dim, dtype=torch.float16, device="cuda")
    gen = torch.Generator().manual_seed(7)
    tail = rand(gen, 1, length, dim, dtype=torch.float16)
    x[-1:] = tail
    lengths = torch.full((n,), length, dtype=torch.int32, device="cuda")
    lengths[0], lengths[-1] = 3, 1000
    y = maxsim_amd.normalize_embeddings(x, lengths)
    want = maxsim_amd.normalize_embeddings(tail, lengths[-1:])
    assert torch.equal(y[-1:], want) and (y[:-1] == 0).all()
    docs, off = maxsim_amd.pack_normalized_documents(x, lengths)
    assert int(off[-1]) == docs.shape[0] and torch.equal(docs[-1000:], want[0, :1000])


def test_feeds_the_contrastive_step():
    """Packed and normalised in one pass or in torch's steps: the same loss and
    gradients up to the rounding of the embeddings."""
    gen = torch.Generator().manual_seed(8)
    d = rand(gen, 6, 20, 64, scale=2.0)
    q = rand(gen, 6, 8, 64, scale=2.0)
    lengths = torch.tensor([20, 3, 1, 11, 7, 19], device="cuda")

    def loss(normalize):
        dl, ql = d.clone().requires_grad_(True), q.clone().requires_grad_(True)
        if normalize:
            docs, off = maxsim_amd.pack_normalized_documents(dl, lengths)
            qn = maxsim_amd.normalize_embeddings(ql)
        else:
            real = torch.arange(20, device="cuda") < lengths[:, None]
            docs, qn = F.normalize(dl, dim=-1)[real], F.normalize(ql, dim=-1)
            off = F.pad(lengths.cumsum(0), (1, 0)).to(torch.int32)
        value = maxsim_amd.score_contrastive_cross_entropy(qn, docs, off)
        value.backward()
        return value.detach(), dl.grad, ql.grad

    for a, b in zip(loss(True), loss(False)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)


def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(9)
    x, dy = rand(gen, 3, 5, 50), rand(gen, 3, 5, 50)
    lengths = torch.tensor([5, 2, 4], device="cuda")
    leaf = x.requires_grad_(True)
    (dx,) = torch.autograd.grad(maxsim_amd.normalize_embeddings(leaf, lengths), leaf, dy)
    v, h, ln = np.random.RandomState(0).randn(3, 5, 50), 1e-5, lengths.cpu().numpy()
    f = [(oracle.unit_rows(f64(x) + s * h * v, ln, EPS) * f64(dy)).sum() for s in (1, -1)]
    size = float(np.abs(f64(dx) * v).sum())
    assert abs((f64(dx) * v).sum() - (f[0] - f[1]) / (2 * h)) <= 1e-5 * size


def test_in_a_graph():
    gen = torch.Generator().manual_seed(10)
    x = rand(gen, 9, 12, 128, dtype=torch.bfloat16).requires_grad_(True)
    dy = rand(gen, 9, 12, 128, dtype=torch.bfloat16)
    lengths = torch.randint(0, 13, (9,), generator=gen).to(torch.int32).cuda()

    def step():
        y = maxsim_amd.normalize_embeddings(x, lengths)
        return (y.detach(), *torch.autograd.grad(y, x, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        lengths.copy_(torch.randint(0, 13, (9,), generator=gen))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_compiles():
    gen = torch.Generator().manual_seed(11)
    x = rand(gen, 4, 6, 128).requires_grad_(True)
    lengths = torch.tensor([6, 0, 2, 5], dtype=torch.int32, device="cuda")

    def f(x):
        return (maxsim_amd.normalize_embeddings(x * 3, lengths) * x).square().sum()

    want = torch.autograd.grad(f(x), x)
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x), x)
    assert torch.equal(want[0], got[0])


def test_packing_under_compile():
    gen = torch.Generator().manual_seed(12)
    x = rand(gen, 4, 6, 128).requires_grad_(True)
    lengths = torch.tensor([6, 0, 2, 5], device="cuda")

    def f(x):
        docs, offsets = maxsim_amd.pack_normalized_documents(x * 3, lengths)
        return (docs * docs[:1]).sum() + offsets.sum()

    want = torch.autograd.grad(f(x), x)
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager")(x), x)
    assert torch.equal(want[0], got[0])


def test_refusals():
    x = torch.randn(4, 5, 64, device="cuda")
    ln = torch.tensor([1, 2, 3, 4], device="cuda")
    norm, pack = maxsim_amd.normalize_embeddings, maxsim_amd.pack_normalized_documents
    cases = [
        (RuntimeError, "HIP", lambda: norm(x.cpu())),
        (TypeError, "x must be", lambda: norm(x.double())),
        (TypeError, "lengths must be", lambda: norm(x, ln.float())),
        (ValueError, "lengths must have shape", lambda: norm(x, ln[:3])),
        (ValueError, "3-D", lambda: norm(x[0], ln)),
        (ValueError, "eps", lambda: norm(x, eps=0.0)),
        (ValueError, "dim must be > 0", lambda: norm(x[..., :0])),
        (RuntimeError, "same device", lambda: norm(x, ln.cpu())),
        (RuntimeError, "16384", lambda: norm(torch.zeros(1, 16385, device="cuda"))),
        (RuntimeError, "HIP", lambda: pack(x.cpu(), ln.cpu())),
        (ValueError, "3-D", lambda: pack(x[0], ln)),
        (ValueError, "doc_lengths must have shape", lambda: pack(x, ln[:2])),
        (TypeError, "lengths must be", lambda: pack(x, ln.float())),
        (ValueError, "eps", lambda: pack(x, ln, eps=-1.0)),
    ]
    for error, text, f in cases:
        with pytest.raises(error, match=text):
            f()


@pytest.mark.parametrize("packed", [False, True])
def test_a_second_derivative_raises(packed):
    x = torch.randn(4, 6, 64, device="cuda", requires_grad=True)
    lengths = torch.tensor([1, 6, 0, 3], device="cuda")
    y = (maxsim_amd.pack_normalized_documents(x, lengths)[0] if packed
         else maxsim_amd.normalize_embeddings(x, lengths))
    down = torch.randn_like(y)
    once, = torch.autograd.grad(y, x, down, retain_graph=True)
    grad, = torch.autograd.grad(y, x, down, create_graph=True)
    assert torch.equal(once, grad)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(grad.square().sum(), x)
