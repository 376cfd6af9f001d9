"""maxsim_amd.adamw_step, its 8-bit states and the AdamW optimizer against the
float64 oracle and, bit for bit where the codes need it, numpy's fp32."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._helpers import DTYPES, one_element_off
from ._training_helpers import U32, assert_within, f64, rand

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SIZES = [1, 2, 7, 8, 9, 255, 256, 257, 2047, 2048, 4095, 4096, 4097, 10000, 70001]


def _make(sizes, dtype, gdtype, bits, master, seed):
    """Lists of tensors in the middle of training, gradients of many sizes."""
    gen = torch.Generator().manual_seed(seed)
    out = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], scales=[], masters=[])
    for i, n in enumerate(sizes):
        size = torch.exp(2 * torch.randn(n, generator=gen)) * 1e-3
        p = torch.randn(n, generator=gen) * 0.1
        g = torch.randn(n, generator=gen) * size
        g[torch.randint(0, n, (n // 8,), generator=gen)] = 0
        m, v = torch.randn(n, generator=gen) * size * 0.3, torch.rand(n, generator=gen) * size ** 2
        v[torch.randint(0, n, (n // 9,), generator=gen)] = 0
        if bits == 8:
            zero = np.full(n, 2 ** 19)
            mc, me = oracle.encode(m.numpy(), True, zero)
            vc, ve = oracle.encode(v.numpy(), False, zero)
            m, v = torch.from_numpy(mc), torch.from_numpy(vc)
            out["scales"].append(torch.from_numpy(np.stack([me, ve], 1)).cuda())
        out["params"].append(p.to(dtype).cuda())
        out["grads"].append(g.to(gdtype).cuda())
        out["exp_avgs"].append(m.cuda())
        out["exp_avg_sqs"].append(v.cuda())
        if master:
            out["masters"].append(p.cuda())
    return out


def _step(t, step=7, seed=3, **hyper):
    maxsim_amd.adamw_step(t["params"], t["grads"], t["exp_avgs"], t["exp_avg_sqs"], step=step,
                          scales=t["scales"] or None, masters=t["masters"] or None, seed=seed,
                          **{**HYPER, **hyper})


def _clone(t):
    return {k: [x.clone() for x in v] for k, v in t.items()}


def _check(before, after, step=7, seed=3, **hyper):
    h = {**HYPER, **hyper}
    b1, b2 = h["betas"]
    position = 0
    for i, p0 in enumerate(before["params"]):
        eight = bool(before["scales"])
        start = before["masters"][i] if before["masters"] else p0
        p, g = f64(start), f64(before["grads"][i])
        if eight:
            sc = before["scales"][i].cpu().numpy()
            m = oracle.decode(before["exp_avgs"][i].cpu().numpy(), sc[:, 0], True)
            v = oracle.decode(before["exp_avg_sqs"][i].cpu().numpy(), sc[:, 1], False)
        else:
            m, v = f64(before["exp_avgs"][i]), f64(before["exp_avg_sqs"][i])
        want, wm, wv = oracle.adamw(p, g, m, v, step, h["lr"], b1, b2, h["eps"],
                                    h["weight_decay"])
        # the update's quotient is off by as many roundings as it has steps and
        # by m's own error, which cancellation may leave large beside m
        em = 4 * U32 * (b1 * np.abs(m) + (1 - b1) * np.abs(g))
        vh = np.sqrt(wv / (1 - b2 ** step)) + h["eps"]
        moved = h["lr"] / (1 - b1 ** step) / vh
        ep = 4 * U32 * np.abs(p) + moved * (em + 30 * U32 * np.abs(wm))
        assert_within(after["params"][i], want, ep, f"param {i}")
        if before["masters"]:
            assert_within(after["masters"][i], want, ep, f"master {i}")
            assert torch.equal(after["params"][i], after["masters"][i].to(p0.dtype))
        if not eight:
            assert_within(after["exp_avgs"][i], wm, em, f"exp_avg {i}")
            assert_within(after["exp_avg_sqs"][i], wv, 6 * U32 * wv, f"exp_avg_sq {i}")
        else:
            # the codes exactly: fp32 products and sums, each rounded, as numpy's
            f = np.float32
            g32, m32, v32 = g.astype(f), m.astype(f), v.astype(f)
            nm = m32 * f(b1) + g32 * f(1 - b1)
            nv = v32 * f(b2) + (g32 * g32) * f(1 - b2)
            at = np.arange(len(p), dtype=np.uint64) + np.uint64(position)
            dm, dv = oracle.dither(at, step, seed)
            cm, em8 = oracle.encode(nm, True, dm)
            cv, ev8 = oracle.encode(nv, False, dv)
            sc = after["scales"][i].cpu().numpy()
            assert (sc[:, 0] == em8).all() and (sc[:, 1] == ev8).all()
            assert (after["exp_avgs"][i].cpu().numpy() == cm).all(), f"exp_avg {i}"
            assert (after["exp_avg_sqs"][i].cpu().numpy() == cv).all(), f"exp_avg_sq {i}"
            values = maxsim_amd.adamw_state_values(after["exp_avgs"][i], after["exp_avg_sqs"][i],
                                                   after["scales"][i])
            assert (f64(values[0]) == oracle.decode(cm, em8, True)).all()
            assert (f64(values[1]) == oracle.decode(cv, ev8, False)).all()
        position += -(-len(p) // 256) * 256


COMBOS = [(d, g, b, m) for d in DTYPES for g in {d, torch.float32} for b in (32, 8)
          for m in ((False,) if d == torch.float32 else (False, True))]


@pytest.mark.parametrize("dtype,gdtype,bits,master", COMBOS,
                         ids=lambda v: str(v).replace("torch.", ""))
def test_types_and_sizes(dtype, gdtype, bits, master):
    t = _make(SIZES, dtype, gdtype, bits, master, seed=1)
    before = _clone(t)
    _step(t)
    _check(before, t)
    assert all(torch.equal(a, b) for a, b in zip(before["grads"], t["grads"]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 47, 48, 49, 200])
def test_more_tensors_than_a_launch_takes(count, bits):
    sizes = [(37 * i) % 700 + 1 for i in range(count)]
    sizes[count // 2] = 30000
    t = _make(sizes, torch.bfloat16, torch.bfloat16, bits, True, seed=count)
    before = _clone(t)
    _step(t)
    _check(before, t)


def test_mixed_types_in_one_call():
    a = _make([300, 5000], torch.float32, torch.float32, 8, False, seed=2)
    b = _make([77, 4097], torch.bfloat16, torch.float32, 8, False, seed=3)
    t = {k: [x for pair in zip(a[k], b[k]) for x in pair] for k in a}
    before = _clone(t)
    _step(t)
    _check(before, t)


@pytest.mark.parametrize("hyper", [dict(weight_decay=0.0), dict(lr=0.0), dict(betas=(0.0, 0.0)),
                                   dict(eps=1e-3), dict(betas=(0.95, 0.9))], ids=str)
@pytest.mark.parametrize("step", [1, 2, 100000])
def test_settings(step, hyper):
    for bits in (32, 8):
        t = _make([1000, 256], torch.float32, torch.float32, bits, False, seed=4)
        before = _clone(t)
        _step(t, step=step, seed=-5 if step == 1 else 2 ** 40 + 1, **hyper)
        _check(before, t, step=step, seed=(-5 if step == 1 else 2 ** 40 + 1) & 0xFFFFFFFF, **hyper)


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    t = _make([60 * 70, 4096, 300], torch.bfloat16, torch.float32, bits, True, seed=5)
    want = _clone(t)
    _step(want)
    # memory order counts: a transposed parameter with its states likewise
    for k in ("params", "exp_avgs", "exp_avg_sqs", "masters"):
        t[k][0] = t[k][0].view(70, 60).t()
        t[k][1] = one_element_off(t[k][1])
    t["grads"][0] = t["grads"][0].view(70, 60).t().contiguous()  # another order than its parameter
    t["grads"][1] = one_element_off(t["grads"][1])
    t["grads"][2] = t["grads"][2].repeat_interleave(2)[::2]
    _step(t)
    for k in ("params", "exp_avgs", "exp_avg_sqs", "masters"):
        assert torch.equal(t[k][0].t().reshape(-1), want[k][0])
        assert torch.equal(t[k][1], want[k][1]) and torch.equal(t[k][2], want[k][2])


def test_no_elements_and_no_tensors():
    maxsim_amd.adamw_step([], [], [], [], step=1)
    t = _make([300, 300], torch.float32, torch.float32, 32, False, seed=6)
    t = {k: ([v[0], v[0][:0], v[1]] if v else v) for k, v in t.items()}
    before = _clone(t)
    _step(t)
    _check({k: [v[0], v[2]] if v else v for k, v in before.items()},
           {k: [v[0], v[2]] if v else v for k, v in t.items()})


def test_states_from_zero():
    for bits in (32, 8):
        t = _make([5000], torch.float32, torch.float32, bits, False, seed=7)
        for k in ("exp_avgs", "exp_avg_sqs", "scales"):
            for x in t[k]:
                x.zero_()
        before = _clone(t)
        _step(t, step=1)
        _check(before, t, step=1)


def test_extreme_gradients_in_8_bits():
    # from fp32's smallest to squares near its largest, and zeros, per block
    gen = torch.Generator().manual_seed(8)
    n = 256 * 12
    scale = torch.logspace(-44, 18, 12).repeat_interleave(256)
    t = _make([n], torch.float32, torch.float32, 8, False, seed=8)
    t["grads"][0] = (torch.randn(n, generator=gen) * scale).cuda()
    t["grads"][0][:256] = 0
    before = _clone(t)
    _step(t, eps=1e-3)
    _check(before, t, eps=1e-3)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite(bad):
    t = _make([1000], torch.float32, torch.float32, 32, False, seed=9)
    u = _make([1000], torch.float32, torch.float32, 8, False, seed=9)
    for s in (t, u):
        clean = _clone(s)
        _step(clean)
        s["grads"][0][300] = bad
        _step(s)
        keep = torch.arange(1000, device="cuda") != 300
        assert s["params"][0][300].isnan()
        assert torch.equal(s["params"][0][keep], clean["params"][0][keep])
    m, v = maxsim_amd.adamw_state_values(u["exp_avgs"][0], u["exp_avg_sqs"][0], u["scales"][0])
    assert m[256:512].isnan().all() and v[256:512].isnan().all()
    assert m[:256].isfinite().all() and m[512:].isfinite().all()


def test_moments_move_by_less_than_a_code_step():
    """With b2 = 0.999 each step moves v by a thousandth and a code step is an
    eighth: after 700 steps without a gradient half of it is left, on average
    (0.999^700 = 0.4964; an element's noise is about 0.2, 4096 of them 0.003)."""
    n = 4096
    t = _make([n], torch.float32, torch.float32, 8, False, seed=10)
    t["grads"][0].zero_()
    code, e = oracle.encode(np.ones(n, np.float32), False, np.zeros(n, np.int64))
    t["exp_avg_sqs"][0].copy_(torch.from_numpy(code))
    t["scales"][0][:, 1] = torch.from_numpy(e).cuda()
    for step in range(700):
        _step(t, step=step + 1)
    _, v = maxsim_amd.adamw_state_values(t["exp_avgs"][0], t["exp_avg_sqs"][0], t["scales"][0])
    assert abs(float(v.double().mean()) - 0.999 ** 700) < 0.03


def test_past_two_to_the_31_elements():
    n = 2 ** 31 + 5000
    t = {"params": [torch.zeros(n, dtype=torch.bfloat16, device="cuda")],
         "grads": [torch.zeros(n, dtype=torch.bfloat16, device="cuda")],
         "exp_avgs": [torch.zeros(n, dtype=torch.uint8, device="cuda")],
         "exp_avg_sqs": [torch.zeros(n, dtype=torch.uint8, device="cuda")],
         "scales": [torch.zeros((n + 255) // 256, 2, dtype=torch.uint8, device="cuda")],
         "masters": []}
    gen = torch.Generator().manual_seed(11)
    t["params"][0][-3000:] = rand(gen, 3000, dtype=torch.bfloat16)
    t["grads"][0][-3000:] = rand(gen, 3000, dtype=torch.bfloat16)
    start = t["params"][0][-3000:].clone()
    _step(t, step=1)
    at = n - 3000 - (n - 3000) % 256
    want = oracle.adamw(f64(start), f64(t["grads"][0][-3000:]), 0.0, 0.0, 1, HYPER["lr"], 0.9, 0.999,
                        1e-8, 0.1)
    assert_within(t["params"][0][-3000:], want[0], 40 * U32 * (np.abs(want[0]) + HYPER["lr"]))
    m, _ = maxsim_amd.adamw_state_values(t["exp_avgs"][0][at:], t["exp_avg_sqs"][0][at:],
                                         t["scales"][0][at // 256:])
    got = f64(m)[n - 3000 - at:]
    largest = np.repeat(np.abs(f64(m).reshape(-1))[: len(m) // 256 * 256].reshape(-1, 256).max(1), 256)
    assert (np.abs(got[:2048] - want[1][:2048]) <=
            np.abs(want[1][:2048]) / 8 + largest[n - 3000 - at:][:2048] * 2.0 ** -15).all()
    assert (t["params"][0][:-3000] == 0).all() and (t["exp_avg_sqs"][0][:-3000] == 0).all()


def test_same_bits_every_time_and_other_streams():
    t = _make([5000, 70000], torch.bfloat16, torch.bfloat16, 8, True, seed=12)
    a, b = _clone(t), _clone(t)
    _step(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for k in a for x, y in zip(a[k], b[k]))
    c = _clone(t)
    _step(c, seed=4)  # other random bits: other codes, the same parameters
    assert torch.equal(a["masters"][1], c["masters"][1])
    assert not torch.equal(a["exp_avg_sqs"][1], c["exp_avg_sqs"][1])


def test_step_and_rate_on_the_device_in_a_graph():
    t = _make([3000, 300], torch.bfloat16, torch.bfloat16, 8, True, seed=13)
    ref = _clone(t)
    step = torch.ones(1, dtype=torch.int64, device="cuda")
    lr = torch.full((1,), 1e-3, device="cuda")
    warm = _clone(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(warm, step=step, lr=lr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(t, step=step, lr=lr)
    for k in range(4):
        step.fill_(k + 1)
        lr.fill_(1e-3 / (k + 1))
        graph.replay()
        before = _clone(ref)
        _step(ref, step=k + 1, lr=1e-3 / (k + 1))
        torch.cuda.synchronize()
        _check(before, ref, step=k + 1, lr=1e-3 / (k + 1))
        for key in ("exp_avgs", "exp_avg_sqs", "scales"):
            assert all(torch.equal(x, y) for x, y in zip(t[key], ref[key])), (k, key)
        for x, y in zip(t["masters"], ref["masters"]):
            torch.testing.assert_close(x, y, rtol=1e-6, atol=1e-8)
            y.copy_(x)
        for x, y in zip(t["params"], ref["params"]):
            y.copy_(x)


def test_saved_tensors_notice_the_step():
    w = torch.randn(64, device="cuda", requires_grad=True)
    y = maxsim_amd.layer_norm(torch.randn(4, 64, device="cuda", requires_grad=True), w)
    maxsim_amd.adamw_step([w], [torch.ones_like(w)], [torch.zeros_like(w)],
                          [torch.zeros_like(w)], step=1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


# ---- the optimizer -----------------------------------------------------------
def _model(dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    m = torch.nn.Sequential(torch.nn.Linear(96, 64), torch.nn.LayerNorm(64),
                            torch.nn.Linear(64, 33))
    return m.to(dtype).cuda()


def _train(model, opt, steps, seed=1):
    gen = torch.Generator().manual_seed(seed)
    dtype = next(model.parameters()).dtype
    for _ in range(steps):
        x, y = rand(gen, 50, 96, dtype=dtype), rand(gen, 50, 33, dtype=dtype)
        opt.zero_grad()
        (model(x) - y).float().square().mean().backward()
        opt.step()


def test_optimizer_is_adamw():
    a, b = _model(), _model()
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)
    _train(a, maxsim_amd.AdamW(a.parameters(), **kw), 10)
    _train(b, torch.optim.AdamW(b.parameters(), **kw, foreach=False, fused=False), 10)
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-5)


def test_optimizer_state_and_its_round_trip():
    for dtype, kw in ((torch.bfloat16, dict(state_bits=8, min_8bit_size=500, master_weights=True)),
                      (torch.float32, dict(state_bits=8, min_8bit_size=500)), (torch.float16, {})):
        a = _model(dtype)
        opt = maxsim_amd.AdamW(a.parameters(), lr=1e-3, **kw)
        _train(a, opt, 3)
        for p in a.parameters():
            s = opt.state[p]
            eight = "state_bits" in kw and p.numel() >= 500
            assert s["step"] == 3 and ("scales" in s) == eight
            assert s["exp_avg"].dtype == (torch.uint8 if eight else torch.float32)
            assert ("master" in s) == (dtype == torch.bfloat16)
        b = _model(dtype, seed=5)
        b.load_state_dict(a.state_dict())
        other = maxsim_amd.AdamW(b.parameters(), lr=5.0, **kw)
        other.load_state_dict(opt.state_dict())
        for p, q in zip(a.parameters(), b.parameters()):
            for k, v in opt.state[p].items():
                w = other.state[q][k]
                if isinstance(v, torch.Tensor):
                    assert v.dtype == w.dtype and torch.equal(v, w) and v.data_ptr() != w.data_ptr()
                else:
                    assert v == w
        _train(a, opt, 2, seed=9)
        _train(b, other, 2, seed=9)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def test_optimizer_groups_and_missing_gradients():
    gen = torch.Generator().manual_seed(14)
    p = [rand(gen, 40, 50).requires_grad_(True), rand(gen, 5000).requires_grad_(True),
         rand(gen, 30).requires_grad_(True)]
    start = [x.detach().clone() for x in p]
    opt = maxsim_amd.AdamW([dict(params=p[:2], weight_decay=0.2, state_bits=8),
                            dict(params=p[2:], lr=torch.tensor([0.5], device="cuda"))], lr=0.1)
    p[0].grad, p[2].grad = torch.ones_like(p[0]), torch.ones_like(p[2])
    opt.step()
    assert torch.equal(p[1], start[1]) and not opt.state[p[1]]
    torch.testing.assert_close(p[0], start[0] * (1 - 0.1 * 0.2) - 0.1, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(p[2], start[2] * (1 - 0.5 * 0.01) - 0.5, rtol=1e-5, atol=1e-5)
    p[1].grad = -torch.ones_like(p[1])
    opt.step()
    assert opt.state[p[1]]["step"] == 1 and opt.state[p[0]]["step"] == 2
    assert "scales" in opt.state[p[1]] and "scales" not in opt.state[p[0]]
    torch.testing.assert_close(p[1], start[1] * (1 - 0.1 * 0.2) + 0.1, rtol=1e-5, atol=1e-5)
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0


def test_optimizer_learns_with_8_bit_states():
    """A regression that fp32 states solve: 8-bit states end as near."""
    losses = []
    for kw in ({}, dict(state_bits=8, min_8bit_size=1)):
        torch.manual_seed(0)
        x = torch.randn(512, 96, device="cuda")
        y = torch.tanh(x @ torch.randn(96, 33, device="cuda") * 0.2)
        m = _model()
        opt = maxsim_amd.AdamW(m.parameters(), lr=3e-3, **kw)
        for _ in range(300):
            opt.zero_grad()
            loss = (m(x) - y).square().mean()
            loss.backward()
            opt.step()
        losses.append(float(loss.detach()))
    assert losses[1] < 1.25 * losses[0] + 1e-4, losses


# ---- refusals ----------------------------------------------------------------
def test_refusals():
    def call(change=None, bits=32, dtype=torch.float32, master=False, **kw):
        t = _make([600, 300], dtype, dtype, bits, master, seed=15)
        if change:
            change(t)
        _step(t, **kw)

    def put(key, f, i=1):
        return lambda t: t[key].__setitem__(i, f(t[key][i]))

    half = dict(dtype=torch.bfloat16)
    cases = [
        (RuntimeError, "HIP", dict(change=put("params", lambda x: x.cpu(), 0))),
        (RuntimeError, "same device", dict(change=put("params", lambda x: x.cpu()))),
        (RuntimeError, "same device", dict(change=put("grads", lambda x: x.cpu()))),
        (RuntimeError, "same device", dict(change=put("exp_avgs", lambda x: x.cpu()))),
        (TypeError, "params must be", dict(change=put("params", lambda x: x.double()))),
        (TypeError, "grads.1. must be", dict(change=put("grads", lambda x: x.half()))),
        (TypeError, "grads.1. must be dense", dict(change=put("grads", lambda x: x.to_sparse()))),
        (TypeError, "exp_avgs.1. must be", dict(change=put("exp_avgs", lambda x: x.half()))),
        (TypeError, "exp_avg_sqs.1. must be", dict(bits=8, change=put("exp_avg_sqs", lambda x: x.float()))),
        (TypeError, "scales.1. must be", dict(bits=8, change=put("scales", lambda x: x.int()))),
        (ValueError, "scales.1. must be", dict(bits=8, change=put("scales", lambda x: x[:1]))),
        (TypeError, "takes no master", dict(change=lambda t: t.update(masters=t["exp_avgs"]))),
        (TypeError, "masters.0. must be", dict(**half, master=True, change=put("masters", lambda x: x.half(), 0))),
        (ValueError, "shape", dict(change=put("grads", lambda x: x[:5]))),
        (ValueError, "shape and strides", dict(change=put("exp_avgs", lambda x: x[:5]))),
        (ValueError, "gaps", dict(change=put("params", lambda x: x.repeat(2)[::2]))),
        (ValueError, "gaps", dict(change=put("params", lambda x: x[:1].expand(300)))),
        (ValueError, "one length", dict(change=lambda t: t["grads"].pop())),
        (ValueError, "one length", dict(bits=8, change=lambda t: t["scales"].pop())),
        (ValueError, "step", dict(step=0)),
        (ValueError, "lr", dict(lr=-1.0)),
        (ValueError, "lr", dict(lr=float("nan"))),
        (ValueError, "betas", dict(betas=(1.0, 0.9))),
        (ValueError, "eps", dict(eps=-1.0)),
        (ValueError, "weight_decay", dict(weight_decay=-0.1)),
        (TypeError, "step must be", dict(step=torch.ones(1, device="cuda"))),
        (ValueError, "one value", dict(step=torch.ones(2, dtype=torch.int64, device="cuda"))),
        (TypeError, "lr must be", dict(lr=torch.ones(1, dtype=torch.float64, device="cuda"))),
        (RuntimeError, "same device", dict(lr=torch.ones(1))),
    ]
    for error, text, kw in cases:
        with pytest.raises(error, match=text):
            call(**kw)
    x = torch.zeros(600, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="scales must be"):
        maxsim_amd.adamw_state_values(x, x, torch.zeros(2, 2, dtype=torch.uint8, device="cuda"))
    with pytest.raises(TypeError, match="uint8"):
        maxsim_amd.adamw_state_values(x.float(), x, x)
    for kw, text in ((dict(lr=-1), "lr"), (dict(state_bits=4), "state_bits"),
                     (dict(betas=(0.9, 1.0)), "betas"), (dict(eps=float("nan")), "eps"),
                     (dict(weight_decay=-1), "weight_decay")):
        with pytest.raises(ValueError, match=text):
            maxsim_amd.AdamW([x.float().requires_grad_(True)], **kw)
        with pytest.raises(ValueError, match=text):  # a group's own options too
            maxsim_amd.AdamW([dict(params=[x.float().requires_grad_(True)], **kw)])
    p = torch.zeros(4, 8, device="cuda", requires_grad=True)
    p.grad = torch.ones(4, 8, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        maxsim_amd.AdamW([p]).step()


def test_refuses_parameters_that_share_memory():
    # in one launch their blocks would run over each other
    flat = torch.zeros(700, device="cuda")
    for a, b in ((slice(0, 300), slice(0, 300)), (slice(0, 300), slice(299, 700))):
        t = _make([300, b.stop - b.start], torch.float32, torch.float32, 32, False, seed=4)
        t["params"] = [flat[b], flat[a]] if a != b else [flat[a], flat[a]]
        if a != b:
            for key in ("grads", "exp_avgs", "exp_avg_sqs"):
                t[key] = t[key][::-1]
        with pytest.raises(ValueError, match="share memory"):
            _step(t)
    # neighbours in one buffer and empty parameters do not
    t = _make([300, 400], torch.float32, torch.float32, 32, False, seed=4)
    t["params"] = [flat[:300], flat[300:]]
    for key in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
        t[key] += [torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda")]
    _step(t)
    assert flat.isfinite().all() and flat.count_nonzero() > 650
