"""maxsim_amd.embed_tokens against the float64 oracle: every shape of its
kernels, types, layouts, ids that are none, runs of equal ids around every
boundary of the sums, and its refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._helpers import DTYPES, one_element_off
from ._training_helpers import assert_within, f64, rand

pytestmark = pytest.mark.gpu

KINDS = [(torch.float32, torch.float32), (torch.float16, torch.float16),
         (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16),
         (torch.float32, torch.bfloat16)]  # weight, result


def _ids(gen, vocab, *shape, dtype=torch.int64):
    """Some rows often, most seldom."""
    u = torch.rand(shape, generator=gen, dtype=torch.float64)
    return (vocab ** u).long().sub(1).clamp_(0, vocab - 1).to(dtype).cuda()


def _check(weight, ids, lengths=None, scale=1.0, padding=None, dtype=None, dy=None, gen=None):
    """Forward and gradient against the formulas; returns both."""
    vocab, dim = weight.shape
    out = dtype or weight.dtype
    leaf = weight.detach().requires_grad_(True)
    y = maxsim_amd.embed_tokens(leaf, ids, lengths, scale=scale, padding_idx=padding, dtype=dtype)
    assert y.dtype == out and y.shape == (*ids.shape, dim)
    plain = maxsim_amd.embed_tokens(weight.detach(), ids, lengths, scale=scale, dtype=dtype)
    assert torch.equal(plain.nan_to_num(-7.0), y.detach().nan_to_num(-7.0))
    flat = ids.cpu().numpy().reshape(ids.shape if lengths is not None else (1, -1))
    lens = None if lengths is None else lengths.cpu().numpy()
    want = oracle.embed(f64(weight), flat, lens, float(np.float32(scale))).reshape(-1, dim)
    got = y.detach().reshape(-1, dim)
    none = np.isnan(want).any(1)
    assert np.array_equal(np.isnan(f64(got)).all(1), none)
    assert_within(got[torch.from_numpy(~none).cuda()], want[~none], 0.0, "y")
    if dy is None:
        dy = rand(gen or torch.Generator().manual_seed(5), *ids.shape, dim, dtype=out)
    (dw,) = torch.autograd.grad(y, leaf, dy)
    assert dw.dtype == weight.dtype and dw.shape == weight.shape
    rows = oracle.embed_rows(vocab, flat, lens, padding)
    exact, bound = _gradient(dy.reshape(-1, dim), rows, vocab, float(np.float32(scale)))
    assert_within(dw, exact, bound, "dweight")
    return y.detach(), dw


def _gradient(dy, rows, vocab, scale):
    """oracle.embed_backward; large ones with its sums on the device, in 64 bits."""
    if dy.numel() < 1 << 20:
        return oracle.embed_backward(f64(dy), rows, vocab, scale)
    real = torch.from_numpy(rows >= 0).cuda()
    at, d = torch.from_numpy(rows).cuda()[real], dy[real].double()
    if vocab <= 64:  # few rows: atomics would wait for each other
        sums = [torch.stack([x[at == v].sum(0) for v in range(vocab)]) for x in (d, d.abs())]
    else:
        sums = [torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device="cuda").index_add_(0, at, x)
                for x in (d, d.abs())]
    count = np.bincount(rows[rows >= 0], minlength=vocab)[:, None]
    return f64(sums[0]) * scale, abs(scale) * (count + 2) * 2.0 ** -24 * f64(sums[1])


WIDTHS = [1, 2, 3, 7, 8, 60, 64, 77, 128, 129, 250, 256, 300, 301, 384, 389, 500, 512, 768, 770, 1024,
          1500, 1536, 2048, 2500, 2560, 4096, 4099, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("dim", WIDTHS)
def test_widths(dim, kind):
    # one launch in LDS, and the sort of many
    gen = torch.Generator().manual_seed(dim)
    weight = rand(gen, 37, dim, dtype=kind[0])
    _check(weight, _ids(gen, 37, 700 if dim <= 1024 else 90), dtype=kind[1], gen=gen)
    _check(weight, _ids(gen, 37, 4097), dtype=kind[1], gen=gen)


@pytest.mark.parametrize("vocab", [1, 2, 3, 127, 128, 255, 256, 257, 512, 513, 1000, 32000, 131072,
                                   131073, 300007])
def test_tables(vocab):
    gen = torch.Generator().manual_seed(vocab)
    weight = rand(gen, vocab, 24, dtype=torch.bfloat16)
    for tokens in (100, 3001, 4097, 20000):
        _check(weight, _ids(gen, vocab, tokens), gen=gen)


@pytest.mark.parametrize("tokens", [300, 4096, 5000])
@pytest.mark.parametrize("bits", [16, 17, 24, 25, 26, 28, 29])
def test_tables_of_many_rows(bits, tokens):
    # one to four passes of the sorts, and what the one in LDS has no bits for
    gen = torch.Generator().manual_seed(bits)
    vocab = 2 ** bits - (bits % 2) * 77
    weight = torch.zeros(vocab, 1, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    ids = torch.randint(0, vocab, (tokens,), generator=gen).cuda()
    ids[:100], ids[100:200], ids[200] = ids[250], vocab - 1, 0
    dy = rand(gen, tokens, 1, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(maxsim_amd.embed_tokens(weight, ids), weight, dy)
    unique, inverse = torch.unique(ids, return_inverse=True)
    want, bound = oracle.embed_backward(f64(dy), inverse.cpu().numpy(), len(unique), 1.0)
    assert_within(dw[unique], want, bound)
    dw[unique] = 0
    assert int(torch.count_nonzero(dw)) == 0


@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 4093,
                                    4095, 4096, 4097, 16384, 16385, 131072, 131073, 262144, 262145,
                                    600001])
def test_numbers_of_tokens(tokens):
    gen = torch.Generator().manual_seed(tokens)
    weight = rand(gen, 501, 16)
    _check(weight, _ids(gen, 501, tokens), scale=0.5, gen=gen)


@pytest.mark.parametrize("dim", [8, 100, 300, 600, 2100])
@pytest.mark.parametrize("tokens", [2000, 4096, 8 * 2048, 40 * 2048 + 11, 128 * 2048, 300000])
def test_runs_around_the_boundaries(tokens, dim):
    # runs of one row around the windows' 8 to 128 tokens and around the 64 that
    # are finished by one group, longer and shorter ones, in every position
    if tokens * dim > 1 << 26:
        dim = 8
    rng = np.random.default_rng(tokens)
    runs, left = [], tokens
    while left > 0:
        runs.append(min(left, int(rng.choice([1, 2, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 40, 41, 62, 63, 64,
                                              65, 66, 67, 127, 128, 129, 130, 200, 1000]))))
        left -= runs[-1]
    rows = rng.permutation(len(runs))
    ids = torch.from_numpy(rng.permutation(np.repeat(rows, runs))).cuda()
    gen = torch.Generator().manual_seed(1)
    _check(rand(gen, len(runs), dim, dtype=torch.float16), ids, gen=gen)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("dim", [5, 77, 768, 2560])
def test_one_row_for_all(kind, dim):
    gen = torch.Generator().manual_seed(dim)
    weight = rand(gen, 700, dim, dtype=kind[0])
    for tokens in (3, 1000, 4096, 70001 if dim < 100 else 9001):
        ids = torch.full((tokens,), 300, device="cuda")
        _check(weight, ids, dtype=kind[1], gen=gen)


def test_rows_of_one_bucket():
    # all rows alike in their low bits: one workgroup has them all where the
    # tokens are few, and one digit where they are many
    gen = torch.Generator().manual_seed(3)
    vocab = 200000
    for tokens in (4096, 20011):
        ids = torch.randint(0, vocab // 512, (tokens,), generator=gen) * 512 + 17
        _check(rand(gen, vocab, 8), ids.cuda(), gen=gen)


@pytest.mark.parametrize("vocab,tokens", [(1, 296), (1, 297), (2, 336), (2, 337), (6, 496), (6, 497),
                                          (44, 2016), (44, 2017), (45, 2048), (45, 2049),
                                          (96, 4096), (96, 4097), (500, 20480), (500, 20481)])
@pytest.mark.parametrize("dim", [64, 512, 1024, 1025, 2048, 2049])
def test_where_the_launches_change(vocab, tokens, dim):
    gen = torch.Generator().manual_seed(tokens)
    for dtype in (torch.bfloat16, torch.float32):
        _check(rand(gen, vocab, dim, dtype=dtype), _ids(gen, vocab, tokens), gen=gen)


@pytest.mark.parametrize("vocab,tokens,dim", [(2, 300001, 64), (3, 70000, 72), (40, 131073, 8),
                                              (1, 100000, 300)])
def test_long_runs(vocab, tokens, dim):
    gen = torch.Generator().manual_seed(tokens)
    _check(rand(gen, vocab, dim, dtype=torch.bfloat16), _ids(gen, vocab, tokens), gen=gen)


@pytest.mark.parametrize("dim", [300, 304, 320, 1030])
def test_results_past_the_caches(dim):
    # more than 96 MiB, in rows that are whole lines and that are not
    gen = torch.Generator().manual_seed(dim)
    tokens = (100 << 20) // (2 * dim) + 3
    weight = rand(gen, 1000, dim, dtype=torch.float16)
    ids = _ids(gen, 1000, tokens)
    lens = torch.tensor([tokens - 70], device="cuda")
    y = maxsim_amd.embed_tokens(weight, ids[None], lens, scale=0.5)[0]
    assert torch.equal(y[:-70], weight[ids[:-70]] * 0.5) and not y[-70:].any()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=str)
@pytest.mark.parametrize("lengths", [[0, 0, 0], [5, 0, 9], [9, 9, 9], [1, 200, -4], [0, 9, 1]])
def test_lengths(lengths, dtype):
    gen = torch.Generator().manual_seed(2)
    ids = _ids(gen, 50, 3, 9, dtype=dtype)
    lens = torch.tensor(lengths, dtype=dtype, device="cuda")
    for i, k in enumerate(lengths):
        ids[i, max(k, 0):] = 10 ** 9  # never looked at
    y, _ = _check(rand(gen, 50, 40, dtype=torch.bfloat16), ids, lens, scale=3.0, gen=gen)
    assert not torch.isnan(y).any()


@pytest.mark.parametrize("shape", [(600, 3), (4, 1000), (70, 70), (3000, 1)])
def test_ragged_batches(shape):
    gen = torch.Generator().manual_seed(shape[0])
    lens = torch.randint(0, shape[1] + 1, (shape[0],), generator=gen).cuda()
    _check(rand(gen, 1000, 96), _ids(gen, 1000, *shape, dtype=torch.int32), lens,
           dtype=torch.bfloat16, gen=gen)


def test_padding_that_holds_nan_gives_nothing():
    gen = torch.Generator().manual_seed(4)
    ids, lens = _ids(gen, 50, 4, 9), torch.tensor([3, 0, 9, 1], device="cuda")
    dy = rand(gen, 4, 9, 64)
    bad = dy.clone()
    bad[torch.arange(9, device="cuda") >= lens[:, None]] = float("nan")
    weight = rand(gen, 50, 64)
    assert torch.equal(_check(weight, ids, lens, dy=dy)[1], _grad(weight, ids, lens, bad))


def _grad(weight, ids, lengths=None, dy=None, **kw):
    leaf = weight.detach().requires_grad_(True)
    y = maxsim_amd.embed_tokens(leaf, ids, lengths, **kw)
    return torch.autograd.grad(y, leaf, dy)[0]


def test_ids_outside_the_table():
    gen = torch.Generator().manual_seed(6)
    for dtype, far in ((torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 40)):
        ids = _ids(gen, 300, 40, 20, dtype=dtype)
        ids[0, 0], ids[3, 4], ids[39, 19], ids[7] = 300, -1, far, -far
        if dtype == torch.int64:
            ids[8, 1] = 2 ** 32 + 5  # a row of the table in its low word
        for kind in KINDS:
            _check(rand(gen, 300, 33, dtype=kind[0]), ids, dtype=kind[1], gen=gen)
    nothing = torch.full((5,), 7, device="cuda")
    y, dw = _check(rand(gen, 4, 8), nothing, gen=gen)
    assert torch.isnan(y).all() and not dw.any()
    empty = torch.zeros(0, 8, device="cuda")
    assert torch.isnan(maxsim_amd.embed_tokens(empty, nothing)).all()
    assert _grad(empty, nothing, dy=torch.ones(5, 8, device="cuda")).shape == (0, 8)


def test_padding_idx():
    gen = torch.Generator().manual_seed(7)
    weight, ids = rand(gen, 300, 64), _ids(gen, 300, 800)
    for padding in (0, 5, 299):
        _, dw = _check(weight, ids, padding=padding, gen=gen)
        assert not dw[padding].any()
    dy = rand(gen, 800, 64)
    assert torch.equal(_grad(weight, ids, dy=dy, padding_idx=-1),
                       _grad(weight, ids, dy=dy, padding_idx=299))


@pytest.mark.parametrize("scale", [0.0, -2.5, 27.712812921102035, 1e-30])
@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_scales(kind, scale):
    gen = torch.Generator().manual_seed(8)
    _check(rand(gen, 40, 64, dtype=kind[0]), _ids(gen, 40, 300), scale=scale, dtype=kind[1], gen=gen)


def test_empty_batches():
    weight = torch.ones(5, 8, device="cuda", requires_grad=True)
    for shape in ((0,), (0, 4), (3, 0)):
        ids = torch.zeros(shape, dtype=torch.int64, device="cuda")
        lens = torch.zeros(shape[0], dtype=torch.int64, device="cuda") if len(shape) == 2 else None
        y = maxsim_amd.embed_tokens(weight, ids, lens)
        assert y.shape == (*shape, 8)
        (dw,) = torch.autograd.grad(y.sum(), weight)
        assert dw.shape == weight.shape and not dw.any()


def test_ids_of_any_shape():
    gen = torch.Generator().manual_seed(9)
    weight = rand(gen, 90, 32, dtype=torch.bfloat16)
    for ids in (_ids(gen, 90), _ids(gen, 90, 4, 5, 6), _ids(gen, 90, 30, 40).t(),
                _ids(gen, 90, 12, 20)[::2, 3:9], _ids(gen, 90, 1, 7).expand(5, 7)):
        _check(weight, ids, gen=gen)


def test_layouts_of_the_table():
    gen = torch.Generator().manual_seed(10)
    for dtype in DTYPES:
        wide = rand(gen, 60, 201, dtype=dtype)
        ids = _ids(gen, 60, 500)
        for weight in (wide[:, 1:78], wide[::3, 5:], wide.t(), wide[0].expand(9, 201), wide[:, 200:]):
            want = _check(weight.contiguous(), ids, gen=torch.Generator().manual_seed(1))
            got = _check(weight, ids, gen=torch.Generator().manual_seed(1))
            assert torch.equal(got[0].nan_to_num(), want[0].nan_to_num())
            assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("n", [30, 130])
def test_layouts_of_the_gradient(n):
    gen = torch.Generator().manual_seed(11)
    weight, ids = rand(gen, 160, 77, dtype=torch.float16), _ids(gen, 160, n, 40)
    wide = rand(gen, n, 40, 90, dtype=torch.float16)
    for dy in (wide[..., 3:80], wide[:, :1, :77].expand(n, 40, 77), wide[0, 0, :77].expand(n, 40, 77),
               rand(gen, 77, 40, n, dtype=torch.float16).permute(2, 1, 0),
               rand(gen, 40, n, 77, dtype=torch.float16).transpose(0, 1)):
        got = _check(weight, ids, dy=dy)[1]
        assert torch.equal(got, _grad(weight, ids, dy=dy.contiguous()))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("tokens", [1000, 9000])
def test_what_is_not_finite_stays_in_its_row(tokens, value):
    gen = torch.Generator().manual_seed(tokens)
    weight, ids = rand(gen, 300, 130), _ids(gen, 300, tokens)
    dy = rand(gen, tokens, 130)
    clean = _grad(weight, ids, dy=dy)
    for at in (0, tokens // 2, tokens - 1):
        bad = dy.clone()
        bad[at, 5] = value
        got = _grad(weight, ids, dy=bad)
        row = int(ids[at])
        assert not torch.isfinite(got[row, 5])
        got[row, 5] = clean[row, 5]
        assert torch.equal(got, clean)
    # and what the table holds in the rows that are looked up
    weight[7] = value
    y = maxsim_amd.embed_tokens(weight, ids)
    assert torch.equal(torch.isfinite(y).all(1), ids != 7)


@pytest.mark.parametrize("vocab", [3, 300, 70001])
@pytest.mark.parametrize("tokens", [200, 4000, 9000, 50000])
def test_rows_outside_the_table_in_the_backward(tokens, vocab):
    # through the operator: its rows may hold anything
    from maxsim_amd._ops import ops

    gen = torch.Generator().manual_seed(tokens)
    rows = torch.randint(-3, vocab + 3, (tokens,), generator=gen)
    rows[torch.randint(0, tokens, (9,), generator=gen)] = 2 ** 31 - 1
    rows[torch.randint(0, tokens, (9,), generator=gen)] = -2 ** 31
    dy = rand(gen, tokens, 24)
    got = ops.maxsim_embed_tokens_backward(dy, rows.int().cuda(), vocab, 2.0, torch.float32)
    known = np.where((rows >= 0) & (rows < vocab), rows, -1)
    exact, bound = oracle.embed_backward(f64(dy), known, vocab, 2.0)
    assert_within(got, exact, bound)
    none = ops.maxsim_embed_tokens_backward(dy, torch.full((tokens,), -1, dtype=torch.int32, device="cuda"),
                                            vocab, 2.0, torch.float32)
    assert not none.any()


def test_the_same_bits_every_time():
    gen = torch.Generator().manual_seed(12)
    for tokens in (4000, 50000):
        weight, ids = rand(gen, 5000, 130, dtype=torch.bfloat16), _ids(gen, 5000, tokens)
        dy = rand(gen, tokens, 130, dtype=torch.bfloat16)
        first = _grad(weight, ids, dy=dy)
        for _ in range(4):
            assert torch.equal(_grad(weight, ids, dy=dy), first)
        assert torch.equal(_grad(weight, ids.int(), dy=dy), first)


@pytest.mark.parametrize("others", [0, 3000, 6000])
def test_order_of_a_sum_is_the_tokens(others):
    # 1, 2^25 and -2^25 in the ids' order: (1 + 2^25) - 2^25 is 0 in fp32,
    # 2^25 - 2^25 + 1 is 1
    places = [0, 1 + others // 2, 2 + others]
    ids = torch.arange(others + 3, device="cuda") + 20
    ids[places] = 0
    for order, want in (((1.0, 2.0 ** 25, -2.0 ** 25), 0.0), ((2.0 ** 25, -2.0 ** 25, 1.0), 1.0)):
        dy = torch.zeros(others + 3, 8, device="cuda")
        dy[places] = torch.tensor(order, device="cuda")[:, None]
        dw = _grad(torch.zeros(others + 23, 8, device="cuda"), ids, dy=dy)
        assert dw[0].tolist() == [want] * 8


def test_the_comparison_sees_one_wrong_element():
    gen = torch.Generator().manual_seed(13)
    dy, rows = f64(rand(gen, 500, 16)), _ids(gen, 30, 500).cpu().numpy()
    want, bound = oracle.embed_backward(dy, rows, 30, 2.0)
    wrong = torch.from_numpy(oracle.embed_backward(np.delete(dy, 77, 0), np.delete(rows, 77), 30,
                                                   2.0)[0]).float()
    with pytest.raises(AssertionError):
        assert_within(wrong, want, bound)


def test_against_differences():
    # the result is linear in the table: one difference of any size is exact
    # up to fp32's rounding of the two results
    gen = torch.Generator().manual_seed(14)
    weight, ids, d = rand(gen, 40, 24), _ids(gen, 40, 300), rand(gen, 40, 24)
    dy = rand(gen, 300, 24)
    along = (f64(_grad(weight, ids, dy=dy, scale=1.5)) * f64(d)).sum()
    up = f64(maxsim_amd.embed_tokens(weight + d, ids, scale=1.5))
    down = f64(maxsim_amd.embed_tokens(weight - d, ids, scale=1.5))
    got = ((up - down) * f64(dy)).sum() / 2
    size = (np.abs(up) + np.abs(down)) * np.abs(f64(dy))
    # weight +- d, the products and the sums of at most 300 terms, each a rounding
    assert abs(got - along) <= 2.0 ** -24 * (3 * size.sum() + 310 * size.sum())


def test_saved_ids_may_change():
    gen = torch.Generator().manual_seed(15)
    weight, ids = rand(gen, 40, 24).requires_grad_(True), _ids(gen, 40, 300)
    dy, kept = rand(gen, 300, 24), ids.clone()
    y = maxsim_amd.embed_tokens(weight, ids)
    ids.zero_()
    with torch.no_grad():
        weight.zero_()
    (dw,) = torch.autograd.grad(y, weight, dy)
    assert torch.equal(dw, _grad(weight, kept, dy=dy))


def test_two_lookups_of_one_table():
    gen = torch.Generator().manual_seed(16)
    weight = rand(gen, 40, 24).requires_grad_(True)
    a, b = _ids(gen, 40, 300), _ids(gen, 40, 200)
    da, db = rand(gen, 300, 24), rand(gen, 200, 24)
    out = (maxsim_amd.embed_tokens(weight, a), maxsim_amd.embed_tokens(weight, b, scale=2.0))
    torch.autograd.backward(out, (da, db))
    want = _grad(weight, a, dy=da) + _grad(weight, b, dy=db, scale=2.0)
    torch.testing.assert_close(weight.grad, want, rtol=2.0 ** -23, atol=0)


def test_offsets_past_32_bits():
    # 2^32 elements and more on every side: the last rows are as good as the first
    dim = 4096
    rows = 2 ** 32 // dim + 9
    weight = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    weight[0], weight[-1], weight[-2] = 3, 5, 7
    ids = torch.full((rows,), 1, device="cuda")
    ids[0], ids[1], ids[-1], ids[-2] = rows - 1, 0, 0, rows - 2
    y = maxsim_amd.embed_tokens(weight.requires_grad_(True), ids)
    for at, want in ((0, 5), (1, 3), (-1, 3), (-2, 7), (5, 0)):
        assert bool((y[at] == want).all())
    dy = torch.zeros(1, dim, dtype=torch.bfloat16, device="cuda").expand(rows, dim)
    (dw,) = torch.autograd.grad(y, weight, dy, retain_graph=True)
    assert not dw.any()
    del dw
    dy = torch.zeros_like(y)
    dy[0], dy[1], dy[-1], dy[-2] = 1, 2, 4, 8
    (dw,) = torch.autograd.grad(y, weight, dy)
    assert bool((dw[-1] == 1).all()) and bool((dw[0] == 6).all()) and bool((dw[-2] == 8).all())
    dw[0], dw[-1], dw[-2] = 0, 0, 0
    assert not dw.any()


def test_another_stream():
    gen = torch.Generator().manual_seed(17)
    weight, ids = rand(gen, 3000, 300, dtype=torch.bfloat16), _ids(gen, 3000, 20000)
    dy = rand(gen, 20000, 300, dtype=torch.bfloat16)
    want = _grad(weight, ids, dy=dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [_grad(weight, ids, dy=dy) for _ in range(3)]
    here = _grad(weight, ids, dy=dy)
    side.synchronize()
    assert all(torch.equal(g, want) for g in [*got, here])


def test_captured():
    gen = torch.Generator().manual_seed(18)
    weight = rand(gen, 3000, 300).requires_grad_(True)
    ids, lens = _ids(gen, 3000, 64, 90), torch.randint(0, 91, (64,), generator=gen).cuda()
    dy = rand(gen, 64, 90, 300)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(maxsim_amd.embed_tokens(weight, ids, lens, scale=2.0), weight, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            y = maxsim_amd.embed_tokens(weight, ids, lens, scale=2.0)
            outs.append((y, torch.autograd.grad(y, weight, dy)[0]))
    for turn in range(4):
        ids.copy_(_ids(gen, 3000, 64, 90))
        lens.copy_(torch.randint(0, 91, (64,), generator=gen))
        dy.copy_(rand(gen, 64, 90, 300))
        with torch.no_grad():
            weight.mul_(1.5)
        want = maxsim_amd.embed_tokens(weight.detach(), ids, lens, scale=2.0)
        for graph, (y, dw) in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y.detach(), want)
            assert torch.equal(dw, _grad(weight, ids, lens, dy, scale=2.0)), turn


def test_refusals():
    weight = torch.zeros(5, 8, device="cuda")
    ids = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    lens = torch.zeros(2, dtype=torch.int64, device="cuda")
    f = maxsim_amd.embed_tokens
    for error, match, call in (
            (TypeError, "weight", lambda: f(weight.double(), ids)),
            (TypeError, "ids", lambda: f(weight, ids.float())),
            (TypeError, "ids", lambda: f(weight, ids.to(torch.uint8))),
            (TypeError, "dtype", lambda: f(weight.half(), ids, dtype=torch.float32)),
            (TypeError, "dtype", lambda: f(weight.half(), ids, dtype=torch.bfloat16)),
            (TypeError, "dtype", lambda: f(weight, ids, dtype=torch.float64)),
            (TypeError, "lengths", lambda: f(weight, ids, lens.float())),
            (ValueError, "weight", lambda: f(weight[0], ids)),
            (ValueError, "dim", lambda: f(weight[:, :0], ids)),
            (ValueError, "lengths", lambda: f(weight, ids, lens[:1])),
            (ValueError, "ids must be 2-D", lambda: f(weight, ids[0], lens)),
            (ValueError, "padding_idx", lambda: f(weight, ids, padding_idx=5)),
            (ValueError, "padding_idx", lambda: f(weight, ids, padding_idx=-6)),
            (ValueError, "scale", lambda: f(weight, ids, scale=float("inf"))),
            (ValueError, "scale", lambda: f(weight, ids, scale=float("nan"))),
            (RuntimeError, "device", lambda: f(weight, ids.cpu())),
            (RuntimeError, "device", lambda: f(weight, ids, lens.cpu())),
            (RuntimeError, "HIP", lambda: f(weight.cpu(), ids)),
            (RuntimeError, "dim", lambda: f(torch.zeros(2, 16385, device="cuda"), ids))):
        with pytest.raises(error, match=match):
            call()


def test_transforms():
    gen = torch.Generator().manual_seed(19)
    weight, ids = rand(gen, 30, 16), _ids(gen, 30, 4, 7)
    got = torch.vmap(lambda i: maxsim_amd.embed_tokens(weight, i))(ids)
    assert torch.equal(got, maxsim_amd.embed_tokens(weight, ids))
    leaf = weight.clone().requires_grad_(True)
    y = maxsim_amd.embed_tokens(leaf, ids)
    down = rand(gen, 3, 4, 7, 16)
    got, = torch.autograd.grad(y, leaf, down, is_grads_batched=True, retain_graph=True)
    assert torch.equal(got, torch.stack([torch.autograd.grad(y, leaf, d, retain_graph=True)[0]
                                         for d in down]))
    with pytest.raises(NotImplementedError, match="forward mode"):
        torch.func.jvp(lambda w: maxsim_amd.embed_tokens(w, ids), (weight,), (weight,))
    (dw,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        dw.sum().backward()


def test_compiled():
    gen = torch.Generator().manual_seed(20)
    weight, ids = rand(gen, 30, 16), _ids(gen, 30, 4, 7)
    f = torch.compile(lambda w: maxsim_amd.embed_tokens(w, ids, scale=2.0), backend="aot_eager",
                      fullgraph=True)
    dy = rand(gen, 4, 7, 16)
    leaf = weight.clone().requires_grad_(True)
    y = f(leaf)
    assert torch.equal(y.detach(), maxsim_amd.embed_tokens(weight, ids, scale=2.0))
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], _grad(weight, ids, dy=dy, scale=2.0))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("dim", [7, 64, 768, 2560])
def test_rows_off_every_boundary(dim, kind):
    gen = torch.Generator().manual_seed(21)
    weight, ids = rand(gen, 40, dim, dtype=kind[0]), _ids(gen, 40, 300)
    dy = rand(gen, 300, dim, dtype=kind[1])
    want = _check(weight, ids, dtype=kind[1], dy=dy)
    got = _check(one_element_off(weight), one_element_off(ids), dtype=kind[1], dy=one_element_off(dy))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
