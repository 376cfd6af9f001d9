"""Comparison with a bound per element, and shapes, for the tests of the
operators around the scores."""

from __future__ import annotations

import numpy as np
import torch

from oracle.training_oracle import U32

# half a unit in the last place, relative; and half the spacing of the smallest
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().to(torch.float64).cpu().numpy()


def assert_within(actual: torch.Tensor, exact: np.ndarray, bound, what: str = "") -> None:
    """|actual - exact| <= bound (of the fp32 value) + one rounding to
    actual's type, element by element."""
    a = f64(actual)
    assert a.shape == exact.shape, (what, a.shape, exact.shape)
    assert np.isfinite(a).all(), what
    r = ROUND[actual.dtype]
    limit = bound * (1 + 2 * r) + r * np.abs(exact) + TINY[actual.dtype] + U32 * np.abs(exact)
    worst = (np.abs(a - exact) - limit)
    assert (worst <= 0).all(), (what, float(worst.max()), np.unravel_index(worst.argmax(), a.shape))


def rand(gen, *shape, dtype=torch.float32, scale=1.0, device="cuda"):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(device)
