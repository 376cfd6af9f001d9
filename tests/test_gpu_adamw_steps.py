"""maxsim_amd.adamw_step over many steps, at the limits of a launch and with
memory that is shared, beside test_gpu_adamw.py's single steps."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._training_helpers import U32, f64
from .test_gpu_adamw import HYPER, _check, _clone, _make, _model, _step, _train

pytestmark = pytest.mark.gpu


# ---- weight decay ------------------------------------------------------------
DECAY_FORMS = {
    "fp32": {},
    "fp32, rate on the device": dict(device_lr=True),
    "fp32, 8-bit states": dict(bits=8),
    "bf16 with masters": dict(dtype=torch.bfloat16, master=True),
}


@pytest.mark.parametrize("lr", [2e-6, 5e-6, 1e-5])
@pytest.mark.parametrize("form", DECAY_FORMS)
def test_small_weight_decay_adds_up(form, lr):
    """lr * weight_decay of 2e-8 to 1e-7, near the spacing of fp32 below 1.  Two
    copies of the parameters get gradients of opposite sign, so that their mean
    moves by the decay alone: p0 (1 - lr decay)^t.  Each step rounds an element
    once, by at most half of 2^-28 (the elements stay below 2^-4), independently
    as long as the gradients are; 65536 pairs and 1000 steps leave a thousandth
    of the decay of that at six sigma, and the decay's own product and sum are
    good to 1e-6."""
    opt = dict(dtype=torch.float32, bits=32, master=False, device_lr=False)
    opt.update(DECAY_FORMS[form])
    n, steps, decay = 65536, 1000, 0.01
    gen = torch.Generator().manual_seed(1)
    start = torch.rand(n, generator=gen) * 0.05 + 0.01
    sides = []
    for _ in range(2):
        t = _make([n], opt["dtype"], opt["dtype"], opt["bits"], opt["master"], seed=2)
        for key in ("exp_avgs", "exp_avg_sqs", "scales"):
            for x in t[key]:
                x.zero_()
        t["params"][0].copy_(start)
        if opt["master"]:
            t["masters"][0].copy_(start)
        sides.append(t)
    rate = torch.full((1,), lr, device="cuda") if opt["device_lr"] else lr
    gen = torch.Generator(device="cuda").manual_seed(1)
    for step in range(steps):
        noise = torch.randn(n, generator=gen, device="cuda").to(opt["dtype"])
        for t, sign in zip(sides, (1, -1)):
            t["grads"][0] = sign * noise
            _step(t, step=step + 1, lr=rate, weight_decay=decay)
    held = "masters" if opt["master"] else "params"
    assert max(float(t[held][0].abs().max()) for t in sides) < 2.0 ** -4
    got = np.mean([f64(t[held][0]).mean() for t in sides]) - f64(start).mean()
    want = f64(start).mean() * ((1 - lr * decay) ** steps - 1)
    sigma = 2.0 ** -28 / np.sqrt(12) * np.sqrt(steps / (2 * n))
    assert abs(got - want) <= 6 * sigma + 1e-3 * abs(want), (got / want, sigma)


@pytest.mark.parametrize("lr,decay", [(2e-6, 0.01), (1e-4, 0.1), (3e-3, 0.1), (0.5, 1.0)])
@pytest.mark.parametrize("master", [False, True])
def test_a_step_rounds_the_parameter_once(master, lr, decay):
    # half a spacing of the result, and the errors of what is subtracted: the
    # update's as in test_gpu_adamw.py and a few roundings of the two parts
    dtype = torch.bfloat16 if master else torch.float32
    t = _make([70001], dtype, dtype, 32, master, seed=4)
    held = "masters" if master else "params"
    p, g, m, v = (f64(t[k][0]) for k in (held, "grads", "exp_avgs", "exp_avg_sqs"))
    b1, b2 = HYPER["betas"]
    want, wm, wv = oracle.adamw(p, g, m, v, 7, lr, b1, b2, HYPER["eps"], decay)
    _step(t, step=7, lr=lr, weight_decay=decay)
    em = 4 * U32 * (b1 * np.abs(m) + (1 - b1) * np.abs(g))
    moved = lr / (1 - b1 ** 7) / (np.sqrt(wv / (1 - b2 ** 7)) + HYPER["eps"])
    bound = (np.spacing((np.abs(want) * (1 + 2.0 ** -22)).astype(np.float32)).astype(float) / 2
             + moved * (em + 32 * U32 * np.abs(wm)) + 4 * U32 * lr * decay * np.abs(p))
    assert (np.abs(f64(t[held][0]) - want) <= bound).all()


@pytest.mark.parametrize("decay", [0.0, 0.1])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_parameters_that_are_not_finite_stay_so(value, decay):
    # p (1 - lr decay) of an infinity is the infinity, and its neighbours do not see it
    for bits in (32, 8):
        t = _make([600], torch.float32, torch.float32, bits, False, seed=3)
        clean = _clone(t)
        _step(clean, weight_decay=decay)
        t["params"][0][300] = value
        _step(t, weight_decay=decay)
        keep = torch.arange(600, device="cuda") != 300
        assert torch.equal(t["params"][0][keep], clean["params"][0][keep])
        got = float(t["params"][0][300])
        assert got == value or (got != got and value != value)


# ---- memory that is shared ---------------------------------------------------
def _shared(bits=32, master=False):
    dtype = torch.bfloat16 if master else torch.float32
    return _make([300, 700, 300], dtype, dtype, bits, master, seed=5)


def _put(key, i, value):
    return lambda t: t[key].__setitem__(i, value(t))


SHARED = [
    ("one state for all", {}, lambda t: t.update(exp_avgs=[t["exp_avgs"][0], t["exp_avgs"][1],
                                                          t["exp_avgs"][0]])),
    ("second moments", {}, _put("exp_avg_sqs", 2, lambda t: t["exp_avg_sqs"][0])),
    ("both moments of a parameter", {}, _put("exp_avg_sqs", 0, lambda t: t["exp_avgs"][0])),
    ("moments of two parameters", {}, _put("exp_avg_sqs", 2, lambda t: t["exp_avgs"][0])),
    ("a moment and a parameter", {}, _put("exp_avgs", 2, lambda t: t["params"][0])),
    ("a moment inside another", {}, _put("exp_avgs", 0, lambda t: t["exp_avgs"][1][200:500])),
    ("8-bit codes", dict(bits=8), _put("exp_avgs", 2, lambda t: t["exp_avgs"][0])),
    ("8-bit codes of both moments", dict(bits=8), _put("exp_avg_sqs", 1, lambda t: t["exp_avgs"][1])),
    ("codes in the gradient", dict(bits=8),
     _put("exp_avgs", 1, lambda t: t["grads"][1].view(torch.uint8)[:700])),
    ("scales", dict(bits=8), _put("scales", 2, lambda t: t["scales"][0])),
    ("scales inside others", dict(bits=8), _put("scales", 0, lambda t: t["scales"][1][1:])),
    ("masters", dict(master=True), _put("masters", 2, lambda t: t["masters"][0])),
    ("a master and a moment", dict(master=True), _put("masters", 2, lambda t: t["exp_avgs"][0])),
    ("a gradient in another's parameter", {}, _put("grads", 2, lambda t: t["params"][0])),
    ("a gradient across its parameter", {},
     lambda t: t.update(params=[t["params"][1][:300]], grads=[t["params"][1][1:301]],
                        exp_avgs=t["exp_avgs"][:1], exp_avg_sqs=t["exp_avg_sqs"][:1])),
]


@pytest.mark.parametrize("case", SHARED, ids=lambda c: c[0])
def test_refuses_what_it_updates_to_share_memory(case):
    # workgroups of one launch would write over each other, or read what
    # another has already moved
    _, make, change = case
    t = _shared(**make)
    change(t)
    before = _clone(t)
    with pytest.raises(ValueError, match="share memory"):
        _step(t)
    assert all(torch.equal(a, b) for k in t for a, b in zip(before[k], t[k]))


def test_takes_gradients_that_share_memory():
    # they are only read; one may also be its own parameter, or its own moment
    t = _shared()
    want = _clone(t)
    want["grads"][2] = want["grads"][0].clone()
    _step(want)
    t["grads"][2] = t["grads"][0]
    _step(t)
    assert all(torch.equal(a, b) for k in ("params", "exp_avgs") for a, b in zip(want[k], t[k]))
    t = _shared()
    want = _clone(t)
    want["grads"] = [want["params"][0].clone(), want["exp_avgs"][1].clone(), want["grads"][2]]
    _step(want)
    t["grads"] = [t["params"][0], t["exp_avgs"][1], t["grads"][2]]
    _step(t)
    assert all(torch.equal(a, b) for k in ("params", "exp_avgs") for a, b in zip(want[k], t[k]))


def test_neighbours_in_one_buffer_do_not_share():
    # everything in one allocation, in any order
    t = _shared()
    want = _clone(t)
    _step(want)
    flat = torch.empty(4 * 1300, device="cuda")
    at = 4 * 1300
    for k in ("exp_avg_sqs", "params", "grads", "exp_avgs"):
        for i in (1, 0, 2):
            at -= t[k][i].numel()
            flat[at:at + t[k][i].numel()] = t[k][i]
            t[k][i] = flat[at:at + t[k][i].numel()]
    _step(t)
    assert all(torch.equal(a, b) for k in want for a, b in zip(want[k], t[k]))


# ---- torch.optim.AdamW's states ----------------------------------------------
def test_goes_on_from_torch_adamw():
    # three steps by torch, then five by either
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)
    a, b = _model(), _model()
    theirs = torch.optim.AdamW(a.parameters(), **kw, foreach=False, fused=False)
    _train(a, theirs, 3)
    b.load_state_dict(a.state_dict())
    opt = maxsim_amd.AdamW(b.parameters())
    opt.load_state_dict(theirs.state_dict())
    _train(a, theirs, 5, seed=2)
    _train(b, opt, 5, seed=2)
    for p, q in zip(a.parameters(), b.parameters()):
        assert opt.state[q]["step"] == 8
        torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-5)


def test_masters_of_states_from_torch():
    # made at the first step that follows, from the parameter as it is then
    params = [torch.randn(40, 30, device="cuda").bfloat16().requires_grad_(True)]
    theirs = torch.optim.AdamW(params, foreach=False, fused=False)
    params[0].grad = torch.randn_like(params[0])
    theirs.step()
    saved = theirs.state_dict()
    opt = maxsim_amd.AdamW(params, master_weights=True)
    opt.load_state_dict(saved)
    with torch.no_grad():
        params[0].mul_(2)
    p, master = params[0].detach().clone(), params[0].detach().float()
    m, v = (saved["state"][0][k].float() for k in ("exp_avg", "exp_avg_sq"))
    maxsim_amd.adamw_step([p], [params[0].grad], [m], [v], step=2, masters=[master])
    opt.step()
    s = opt.state[params[0]]
    assert torch.equal(params[0], p) and torch.equal(s["master"], master)
    assert torch.equal(s["exp_avg"], m) and torch.equal(s["exp_avg_sq"], v) and s["step"] == 2


# ---- the limits of a launch --------------------------------------------------
# tensors that 4 KB of arguments hold: 3968 bytes at 44 each, 12 more with 8-bit
# states and 8 more with masters
LIMITS = {(32, False): 90, (32, True): 76, (8, False): 70, (8, True): 62}


@pytest.mark.parametrize("bits,master", LIMITS)
@pytest.mark.parametrize("times,more", [(1, -1), (1, 0), (1, 1), (2, 0), (2, 1)])
def test_launches_filled_to_the_last_tensor(bits, master, times, more):
    count = times * LIMITS[bits, master] + more
    dtype = torch.bfloat16 if master else torch.float32
    t = _make([(53 * i) % 900 + 1 for i in range(count - 1)] + [5000], dtype, dtype, bits, master,
              seed=count)
    before = _clone(t)
    _step(t)
    _check(before, t)


def test_no_parameters_beside_other_lists():
    x = [torch.zeros(3, device="cuda")]
    maxsim_amd.adamw_step([], [], [], [], step=1, scales=[], masters=())
    for lists in (([], x, [], []), ([], [], x, []), ([], [], [], x)):
        with pytest.raises(ValueError, match="one length"):
            maxsim_amd.adamw_step(*lists, step=1)
    with pytest.raises(ValueError, match="one length"):
        maxsim_amd.adamw_step([], [], [], [], step=1, masters=x)
