"""maxsim_amd.embed_tokens where a batch has no tokens: a result without rows and
a gradient of zeros, in tables of every width and type."""

from __future__ import annotations

import pytest
import torch

import maxsim_amd
from maxsim_amd._ops import ops

pytestmark = pytest.mark.gpu

KINDS = [(torch.float32, torch.float32), (torch.float16, torch.float16),
         (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16),
         (torch.float32, torch.bfloat16)]  # weight, result
DIMS = [1, 8, 301, 1024, 1025, 2048, 2049, 2560, 4096, 16384]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("dim", DIMS)
def test_empty_batches_of_every_width(dim, kind):
    weight = torch.ones(37, dim, dtype=kind[0], device="cuda", requires_grad=True)
    for shape in ((0,), (0, 4), (3, 0)):
        ids = torch.zeros(shape, dtype=torch.int64, device="cuda")
        lens = torch.zeros(shape[0], dtype=torch.int64, device="cuda") if len(shape) == 2 else None
        y = maxsim_amd.embed_tokens(weight, ids, lens, dtype=kind[1])
        assert y.shape == (*shape, dim) and y.dtype == kind[1]
        torch.full_like(weight.detach(), 7.0)  # what the gradient's memory held before
        (dw,) = torch.autograd.grad(y.sum(), weight)
        assert dw.shape == weight.shape and dw.dtype == kind[0] and not dw.any()


@pytest.mark.parametrize("vocab,dim", [(1, 16384), (5000, 4099), (300007, 1030), (2 ** 29 + 5, 1)])
def test_the_zeros_of_wide_tables(vocab, dim):
    # several rows to a workgroup, rows off every boundary, and more rows than
    # the launch takes tokens of
    rows = torch.empty(0, dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        junk = torch.full((vocab, dim), float("nan"), dtype=dtype, device="cuda")
        del junk
        dy = torch.empty(0, dim, dtype=dtype, device="cuda")
        assert not ops.maxsim_embed_tokens_backward(dy, rows, vocab, 1.0, dtype).any()


def test_a_captured_empty_batch():
    weight = torch.ones(100, 4096, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    ids = torch.zeros(0, 9, dtype=torch.int64, device="cuda")
    run = lambda: torch.autograd.grad(maxsim_amd.embed_tokens(weight, ids).sum(), weight)[0]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = run()
    for _ in range(3):
        dw.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert not dw.any()
