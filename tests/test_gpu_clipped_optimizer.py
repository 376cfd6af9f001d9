"""maxsim_amd.AdamW(max_norm=) in every type and kind of state: each parameter is
stepped on its gradient times the factor of all groups' norm, bit for bit."""

from __future__ import annotations

import pytest
import torch

import maxsim_amd

from ._helpers import DTYPES
from ._training_helpers import rand

pytestmark = pytest.mark.gpu

SHAPES = ((40, 30), (5,), (3000, 4))
OPTIONS = [dict(lr=1e-2, weight_decay=0.05), dict(lr=3e-3, weight_decay=0.0)]  # of the two groups


def _groups(params):
    return [params[:2], params[2:]]


class _Lists:
    """A group's parameters and states for adamw_step."""

    def __init__(self, params, bits, master):
        self.params = [p.detach().clone() for p in params]
        kind = torch.uint8 if bits == 8 else torch.float32
        self.exp_avgs = [torch.zeros(p.shape, dtype=kind, device="cuda") for p in params]
        self.exp_avg_sqs = [torch.zeros(p.shape, dtype=kind, device="cuda") for p in params]
        self.scales = [torch.zeros((p.numel() + 255) // 256, 2, dtype=torch.uint8, device="cuda")
                       for p in params] if bits == 8 else None
        self.masters = [p.detach().float() for p in params] if master else None


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,master", [(t, m) for t in DTYPES for m in (False, True)
                                          if not m or t != torch.float32], ids=str)
def test_every_parameter_is_stepped_on_clipped_gradients(dtype, master, bits):
    gen = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter(rand(gen, *s, dtype=dtype)) for s in SHAPES]
    lists = [_Lists(group, bits, master) for group in _groups(params)]
    unclipped = [_Lists(group, bits, master) for group in _groups(params)]
    opt = maxsim_amd.AdamW([{"params": g, **o} for g, o in zip(_groups(params), OPTIONS)], state_bits=bits,
                           min_8bit_size=1, master_weights=master, max_norm=0.5, seed=7)
    for step in (1, 2, 3):
        for p in params:
            p.grad = rand(gen, *p.shape, dtype=dtype, scale=10.0 ** (step - 2))
        kept = [p.grad.clone() for p in params]
        norm, factor = maxsim_amd.clip_factor(kept, 0.5)
        assert 0 < float(factor) < 0.1
        opt.step()
        assert torch.equal(opt.grad_norm, norm)
        assert all(torch.equal(p.grad, k) for p, k in zip(params, kept))
        for at, (a, b, grads) in enumerate(zip(lists, unclipped, _groups(kept))):
            for t, g in ((a, [x.float() * factor for x in grads]), (b, grads)):
                maxsim_amd.adamw_step(t.params, g, t.exp_avgs, t.exp_avg_sqs, step=step, scales=t.scales,
                                      masters=t.masters, seed=7 + at, **OPTIONS[at])
        for p, q in zip(params, lists[0].params + lists[1].params):
            assert torch.equal(p.detach(), q), step
        for p, q in zip(params, lists[0].exp_avgs + lists[1].exp_avgs):
            assert torch.equal(opt.state[p]["exp_avg"], q), step
        # and that is not the step on the gradients as they are
        assert not all(torch.equal(x, y) for a, b in zip(lists, unclipped)
                       for x, y in zip(a.exp_avg_sqs + (a.scales or []), b.exp_avg_sqs + (b.scales or [])))
