"""State dicts that maxsim_amd.AdamW takes: its own, and what
load hooks make of them (CPU only: nothing steps on a device here)."""

from __future__ import annotations

import copy
import io

import torch

import maxsim_amd


def _params(dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    return [torch.randn(s, generator=gen).to(dtype).requires_grad_(True) for s in ((6, 5), (7,))]


def _own(dtype=torch.float32, **kw):
    params = _params(dtype)
    return params, maxsim_amd.AdamW(params, **kw)


def _own_state(dtype=torch.bfloat16):
    """8-bit states and masters with values that a cast to the parameter's
    dtype would change."""
    params, opt = _own(dtype, state_bits=8, min_8bit_size=20, master_weights=True)
    for p in params:
        opt.state[p].update(opt._new_state(p, opt.param_groups[0]))
        s = opt.state[p]
        s["step"] = 4
        s["master"].add_(2.0 ** -20)
        for name in ("exp_avg", "exp_avg_sq"):
            s[name].copy_(torch.arange(p.numel()).view(p.shape) * (1 if "scales" in s else 0.1))
    return params, opt


def _same(a, b):
    assert a.keys() == b.keys()
    for k, v in a.items():
        if isinstance(v, torch.Tensor):
            assert v.dtype == b[k].dtype and torch.equal(v, b[k]) and v.data_ptr() != b[k].data_ptr()
        else:
            assert v == b[k]


def test_round_trips_keep_every_dtype():
    params, opt = _own_state()
    buffer = io.BytesIO()
    torch.save(opt.state_dict(), buffer)
    buffer.seek(0)
    for saved in (opt.state_dict(), torch.load(buffer, weights_only=True)):
        others, other = _own(torch.bfloat16)
        other.load_state_dict(saved)
        for p, q in zip(params, others):
            _same(opt.state[p], other.state[q])
    twin = copy.deepcopy(opt)
    for p, q in zip(params, twin.param_groups[0]["params"]):
        _same(opt.state[p], twin.state[q])


def test_load_hooks_count():
    # before: what one returns is what is loaded; after: what one leaves stays
    params, opt = _own_state()
    others, other = _own(torch.bfloat16)

    def before(optimizer, state_dict):
        state_dict = copy.deepcopy(state_dict)
        state_dict["state"][0]["master"] += 1.0
        return state_dict

    def after(optimizer):
        s = optimizer.state[others[1]]
        assert s["exp_avg"].dtype == torch.float32  # as it was saved, not as the parameter is
        s["exp_avg"].zero_()

    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(after)
    other.load_state_dict(opt.state_dict())
    assert torch.equal(other.state[others[0]]["master"], opt.state[params[0]]["master"] + 1.0)
    assert (other.state[others[1]]["exp_avg"] == 0).all()
    assert torch.equal(other.state[others[1]]["exp_avg_sq"], opt.state[params[1]]["exp_avg_sq"])


