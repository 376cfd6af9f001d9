"""The embedding-head example: layer norm, unit embeddings, packing, the loss
and AdamW together learn, with either kind of state."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "train_embedding_head.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_embedding_head", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.bfloat16, 32),
                                        (torch.float32, 8), (torch.float32, 32)], ids=str)
def test_the_head_learns(example, dtype, bits):
    losses = example.train(steps=60, batch=32, lq=16, ld=60, hidden=256, dim=64, dtype=dtype,
                           state_bits=bits, report=0)
    assert all(math.isfinite(x) for x in losses)
    first, last = sum(losses[:5]) / 5, sum(losses[-5:]) / 5
    assert last < 0.5 * first, (first, last)


def test_states_in_8_bits_follow_those_in_32(example):
    a, b = (example.train(steps=40, batch=32, lq=16, ld=60, hidden=256, dim=64,
                          dtype=torch.float32, state_bits=bits, report=0) for bits in (8, 32))
    assert abs(a[0] - b[0]) < 1e-5  # the first step's loss is before any state
    assert abs(sum(a[-5:]) - sum(b[-5:])) < 0.1 * sum(b[:5])
