"""State dicts that maxsim_amd.AdamW takes: its own, torch.optim.AdamW's, and
what load hooks make of them (CPU only: nothing steps on a device here)."""

from __future__ import annotations

import copy
import io

import pytest
import torch

import maxsim_amd


def _params(dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    return [torch.randn(s, generator=gen).to(dtype).requires_grad_(True) for s in ((6, 5), (7,))]


def _torch_state(dtype=torch.float32, steps=3, cls=torch.optim.AdamW, **kw):
    params = _params(dtype)
    opt = cls(params, lr=1e-2, weight_decay=0.05, **kw)
    gen = torch.Generator().manual_seed(1)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen).to(dtype)
        opt.step()
    return opt.state_dict()


def _own(dtype=torch.float32, **kw):
    params = _params(dtype)
    return params, maxsim_amd.AdamW(params, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_takes_torch_adamw(dtype):
    saved = _torch_state(dtype)
    params, opt = _own(dtype, lr=5.0, state_bits=8, master_weights=True, seed=3)
    opt.load_state_dict(saved)
    group = opt.param_groups[0]
    assert group["lr"] == 1e-2 and group["weight_decay"] == 0.05
    # its own options stay as they were
    assert (group["state_bits"], group["min_8bit_size"]) == (8, 4096)
    assert (group["master_weights"], group["seed"]) == (True, 3)
    for i, p in enumerate(params):
        s, want = opt.state[p], saved["state"][i]
        assert s["step"] == 3 and type(s["step"]) is int
        for name in ("exp_avg", "exp_avg_sq"):
            assert s[name].dtype == torch.float32
            assert torch.equal(s[name], want[name].float())
            assert s[name].data_ptr() != want[name].data_ptr()


@pytest.mark.parametrize("saved,text", [
    (lambda: _torch_state(amsgrad=True), "amsgrad"),
    (lambda: _torch_state(maximize=True), "maximize"),
    (lambda: _torch_state(cls=torch.optim.Adam), "decoupled"),
    (lambda: _torch_state(cls=torch.optim.SGD, momentum=0.9), "exp_avg"),
])
def test_refuses_what_it_cannot_step(saved, text):
    params, opt = _own()
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match=text):
        opt.load_state_dict(saved())
    assert opt.state_dict() == before


def test_refuses_codes_without_scales_and_bad_options():
    params, opt = _own()
    saved = _torch_state()
    codes = copy.deepcopy(saved)
    codes["state"][0]["exp_avg"] = torch.zeros(6, 5, dtype=torch.uint8)
    with pytest.raises(ValueError, match="scales"):
        opt.load_state_dict(codes)
    for name, value in (("lr", -1.0), ("betas", (0.9, 1.0)), ("state_bits", 4)):
        bad = copy.deepcopy(saved)
        bad["param_groups"][0][name] = value
        with pytest.raises(ValueError, match=name):
            opt.load_state_dict(bad)


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


def test_states_come_in_their_parameters_order():
    # saved for a contiguous parameter, loaded for a transposed one
    saved = _torch_state()
    first, second = _params()
    first = first.detach().t().contiguous().t().requires_grad_(True)
    opt = maxsim_amd.AdamW([first, second])
    opt.load_state_dict(saved)
    s = opt.state[first]
    assert s["exp_avg"].stride() == first.stride()
    assert torch.equal(s["exp_avg"], saved["state"][0]["exp_avg"])
