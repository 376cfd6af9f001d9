"""The gradient of up to 2048 tokens, which one launch sorts and adds up in LDS:
buckets filled to the last token, every number of passes, runs cut by the waves'
shares, the order of a sum, graphs and streams; and what that launch does not
take."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._training_helpers import assert_within, f64, rand
from .test_gpu_embed_tokens import KINDS, _check, _grad, _ids

pytestmark = pytest.mark.gpu

BUCKETS = 256  # rows that are alike in their low 8 bits are one workgroup's


@pytest.mark.parametrize("tokens", [1025, 1500, 2047, 2048])
@pytest.mark.parametrize("vocab", [300, 5000, 65536, 65537, 200000, 2 ** 24 + 1])
def test_one_bucket_of_many_rows(vocab, tokens):
    # the list full, in one to three passes by the rows' high bits
    gen = torch.Generator().manual_seed(vocab + tokens)
    ids = torch.randint(0, (vocab - 18) // BUCKETS + 1, (tokens,), generator=gen) * BUCKETS + 17
    ids[-1], ids[0] = 17, (vocab - 18) // BUCKETS * BUCKETS + 17
    _check(rand(gen, vocab, 8 if vocab < 2 ** 24 else 2), ids.cuda(), gen=gen)


@pytest.mark.parametrize("bits", [24, 25, 28, 29])
def test_one_bucket_of_the_largest_tables(bits):
    # two passes, three, and the most bits that an entry has for a row
    gen = torch.Generator().manual_seed(bits)
    vocab, tokens = 2 ** bits, 2048
    weight = torch.zeros(vocab, 1, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    ids = (torch.randint(0, vocab // BUCKETS, (tokens,), generator=gen) * BUCKETS + 255).cuda()
    ids[100:300], ids[300], ids[301] = ids[5], vocab - 1, 255
    _check_large(weight, ids, gen)


@pytest.mark.parametrize("tokens", [300, 2048])
def test_tables_of_too_many_rows_for_it(tokens):
    # 2^30 rows: the path for many tokens, however few there are
    gen = torch.Generator().manual_seed(tokens)
    vocab = 2 ** 30
    weight = torch.zeros(vocab, 1, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    ids = torch.randint(0, vocab, (tokens,), generator=gen).cuda()
    ids[:100], ids[100:200], ids[200] = ids[250], vocab - 1, 0
    _check_large(weight, ids, gen)


def _check_large(weight, ids, gen):
    dy = rand(gen, len(ids), 1, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(maxsim_amd.embed_tokens(weight, ids), weight, dy)
    unique, inverse = torch.unique(ids, return_inverse=True)
    want, bound = oracle.embed_backward(f64(dy), inverse.cpu().numpy(), len(unique), 1.0)
    assert_within(dw[unique], want, bound)
    dw[unique] = 0
    assert int(torch.count_nonzero(dw)) == 0


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("dim", [8, 256, 300, 520, 770, 1024])
@pytest.mark.parametrize("tokens", [900, 2048])
def test_runs_cut_by_the_shares(tokens, dim, kind):
    # one to four waves side by side share the columns, the others the sorted
    # tokens: runs that end at, before and after a share's end, and that are
    # longer than several shares; of 16-bit rows up to twice as wide
    dim = dim if kind[1] == torch.float32 else dim * 2
    rng = np.random.default_rng(tokens + dim)
    runs, left = [], tokens
    while left > 0:
        runs.append(min(left, int(rng.choice([1, 2, 3, 56, 57, 63, 64, 127, 128, 129, 180, 256, 400, 513]))))
        left -= runs[-1]
    rows = rng.permutation(64)[:len(runs)] * BUCKETS + 3
    ids = torch.from_numpy(rng.permutation(np.repeat(rows, runs))).cuda()
    gen = torch.Generator().manual_seed(1)
    _check(rand(gen, 64 * BUCKETS, dim, dtype=kind[0]), ids, dtype=kind[1], gen=gen)


@pytest.mark.parametrize("vocab", [45, 127, 128, 255, 256, 257, 1000, 32000, 131073, 300007])
def test_tables(vocab):
    gen = torch.Generator().manual_seed(vocab)
    weight = rand(gen, vocab, 24, dtype=torch.bfloat16)
    for tokens in (1500, 2047, 2048):
        _check(weight, _ids(gen, vocab, tokens), gen=gen)


@pytest.mark.parametrize("others", [500, 1500, 2045])
@pytest.mark.parametrize("step", [1, BUCKETS])
def test_order_of_a_sum_is_the_tokens(step, others):
    # (1 + 2^25) - 2^25 is 0 in fp32, 2^25 - 2^25 + 1 is 1; among others of the
    # same bucket or of all
    places = [0, 1 + others // 2, 2 + others]
    ids = (torch.arange(others + 3, device="cuda") + 20) * step
    ids[places] = 0
    for order, want in (((1.0, 2.0 ** 25, -2.0 ** 25), 0.0), ((2.0 ** 25, -2.0 ** 25, 1.0), 1.0)):
        dy = torch.zeros(others + 3, 8, device="cuda")
        dy[places] = torch.tensor(order, device="cuda")[:, None]
        dw = _grad(torch.zeros((others + 23) * step, 8, device="cuda"), ids, dy=dy)
        assert dw[0].tolist() == [want] * 8


def test_the_same_bits_every_time():
    gen = torch.Generator().manual_seed(12)
    for tokens in (700, 2000, 2048):
        weight, ids = rand(gen, 5000, 130, dtype=torch.bfloat16), _ids(gen, 5000, tokens)
        dy = rand(gen, tokens, 130, dtype=torch.bfloat16)
        first = _grad(weight, ids, dy=dy)
        for _ in range(4):
            assert torch.equal(_grad(weight, ids, dy=dy), first)
        assert torch.equal(_grad(weight, ids.int(), dy=dy), first)


def test_another_stream():
    gen = torch.Generator().manual_seed(17)
    weight, ids = rand(gen, 30000, 300, dtype=torch.bfloat16), _ids(gen, 30000, 2000)
    dy = rand(gen, 2000, 300, dtype=torch.bfloat16)
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
    ids, lens = _ids(gen, 3000, 31, 60), torch.randint(0, 61, (31,), generator=gen).cuda()
    dy = rand(gen, 31, 60, 300)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(maxsim_amd.embed_tokens(weight, ids, lens, scale=2.0), weight, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = maxsim_amd.embed_tokens(weight, ids, lens, scale=2.0)
        (dw,) = torch.autograd.grad(y, weight, dy)
    for turn in range(4):
        ids.copy_(_ids(gen, 3000, 31, 60))
        lens.copy_(torch.randint(0, 61, (31,), generator=gen))
        dy.copy_(rand(gen, 31, 60, 300))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), maxsim_amd.embed_tokens(weight.detach(), ids, lens, scale=2.0))
        assert torch.equal(dw, _grad(weight, ids, lens, dy, scale=2.0)), turn


def test_one_id_by_itself():
    # ids without axes: a row of the table, and a gradient of one axis
    gen = torch.Generator().manual_seed(20)
    weight = rand(gen, 40, 24, dtype=torch.float16).requires_grad_(True)
    y = maxsim_amd.embed_tokens(weight, torch.tensor(7, device="cuda"), scale=0.5)
    assert y.shape == (24,) and torch.equal(y.detach(), weight.detach()[7] * 0.5)
    for dy in (rand(gen, 24, dtype=torch.float16), rand(gen, 48, dtype=torch.float16)[::2]):
        (dw,) = torch.autograd.grad(y, weight, dy, retain_graph=True)
        assert torch.equal(dw[7], dy * 0.5)
        dw[7] = 0
        assert not dw.any()
