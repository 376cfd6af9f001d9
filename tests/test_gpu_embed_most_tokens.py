"""maxsim_amd.embed_tokens with 2^31 - 1 tokens, the most whose gradient it takes."""

from __future__ import annotations

import pytest
import torch

import maxsim_amd

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


def test_the_gradient_of_the_most_tokens():
    # every row of the table about 2147 times; sums of so many ones are exact.
    # The numbers 0 to 2^31 - 2 in turn modulo the table's rows
    vocab = 1000003
    weight = torch.arange(vocab, device="cuda").remainder_(256).to(torch.bfloat16).view(vocab, 1)
    weight = weight.float().requires_grad_(True)
    ids = torch.arange(MOST, dtype=torch.int32, device="cuda").remainder_(vocab)
    y = maxsim_amd.embed_tokens(weight, ids, dtype=torch.bfloat16)
    for at in (0, 255, vocab + 7, MOST - 1, MOST - 2):
        assert float(y[at].detach()) == at % vocab % 256
    (dw,) = torch.autograd.grad(y, weight, torch.ones(1, 1, dtype=torch.bfloat16, device="cuda").expand(MOST, 1))
    rows = torch.arange(vocab, device="cuda")
    assert torch.equal(dw[:, 0], ((MOST - 1 - rows) // vocab + 1).float())
    # one token more has no gradient that is taken
    with pytest.raises(RuntimeError, match="2\\^31 - 1 tokens"):
        maxsim_amd.embed_tokens(weight, torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(2, 2 ** 30))
