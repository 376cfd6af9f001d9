"""The norm of all gradients, clipping in place and the AdamW step on clipped
gradients, against the float64 oracle."""

from __future__ import annotations

import copy
import math

import numpy as np
import pytest
import torch

import maxsim_amd
from oracle import training_oracle as oracle

from ._helpers import DTYPES, one_element_off
from ._training_helpers import ROUND, TINY, U32, assert_within, f64, rand

pytestmark = pytest.mark.gpu

SIZES = [1, 2, 3, 7, 8, 9, 255, 257, 4096, 16384, 16385, 32768, 32769, 65537, 70001]


def _list(sizes, dtypes, seed=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    return [rand(gen, n, dtype=dtypes[i % len(dtypes)], scale=scale) for i, n in enumerate(sizes)]


def _check_norm(norm, grads):
    # 64-bit sums, one rounding to fp32: their own error is far below it
    want = oracle.grad_norm([f64(g) for g in grads])
    assert norm.dtype == torch.float32 and norm.shape == () and norm.is_cuda
    assert abs(float(norm) - want) <= want * U32 * (1 + 2.0 ** -20) + 2.0 ** -150
    return want


@pytest.mark.parametrize("dtypes", [[t] for t in DTYPES] + [DTYPES], ids=str)
@pytest.mark.parametrize("sizes", [[1], [3], SIZES, SIZES[::-1], [0, 5, 0, 0, 9, 0], [200003],
                                   [11] * 197, [11] * 198, [11] * 199, [7] * 596 + [40000]],
                         ids=lambda s: f"{len(s)}x{s[0]}")
def test_norms(sizes, dtypes):
    grads = _list(sizes, dtypes)
    norm = maxsim_amd.grad_norm(grads)
    want = _check_norm(norm, grads)
    again, factor = maxsim_amd.clip_factor(grads, 0.01, eps=1e-3)
    assert torch.equal(norm, again)
    f = oracle.clip_factor(want, 0.01, 1e-3)
    assert abs(float(factor) - f) <= f * U32 * (1 + 2.0 ** -20)


@pytest.mark.parametrize("value", [1e-45, 1e-30, 1e-20, 1.0, 1e19, 3e38])
def test_gradients_of_any_size(value):
    for n in (1, 100, 40001):
        g = torch.full((n,), value, device="cuda")
        exact = float(g[0]) * math.sqrt(n)
        norm, factor = maxsim_amd.clip_factor([g], 1.0, eps=0.0)
        want = np.float32(exact) if exact < 3.4e38 else np.inf
        assert float(norm) == pytest.approx(float(want), rel=2 * U32, abs=2.0 ** -149)
        # the factor knows the norm that fp32 does not
        assert float(factor) == pytest.approx(min(1.0, 1.0 / exact), rel=2 * U32, abs=2.0 ** -149)


def test_one_of_many_counts():
    # a single element among 70 million: no sum in 32 bits would see it
    g = torch.full((70_000_001,), 1.0, dtype=torch.bfloat16, device="cuda")
    g[12345678] = 200.0
    want = math.sqrt(70_000_000 + 40_000)
    assert float(maxsim_amd.grad_norm([g])) == pytest.approx(want, rel=2 * U32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gradients_that_are_not_finite(dtype):
    for value, factor in ((math.inf, 0.0), (-math.inf, 0.0), (math.nan, math.nan)):
        for at in (0, 39999, 40000):
            grads = _list([40001, 5], [dtype])
            grads[0][at] = value
            norm, f = maxsim_amd.clip_factor(grads, 1.0)
            assert math.isnan(norm) if math.isnan(value) else float(norm) == math.inf
            assert math.isnan(f) if math.isnan(factor) else float(f) == factor


def test_the_limit():
    g = torch.tensor([3.0, 4.0], device="cuda")
    for max_norm, eps, want in ((5.0, 0.0, 1.0), (10.0, 0.0, 1.0), (2.5, 0.0, 0.5), (0.0, 1e-6, 0.0),
                                (math.inf, 0.0, 1.0), (5.0, 5.0, 0.5)):
        assert float(maxsim_amd.clip_factor([g], max_norm, eps=eps)[1]) == want
    zero = torch.zeros(3, device="cuda")
    assert float(maxsim_amd.clip_factor([zero], 1.0)[1]) == 1.0
    assert float(maxsim_amd.grad_norm([zero])) == 0.0


@pytest.mark.parametrize("dtypes", [[t] for t in DTYPES] + [DTYPES], ids=str)
@pytest.mark.parametrize("sizes", [[1], SIZES, [0, 5, 0], [11] * 399 + [70001], [3000] * 198,
                                   [3000] * 199, [256 * 2048], [256 * 2048 + 1], [0] * 200 + [7],
                                   [2100000], [4300000]],
                         ids=lambda s: f"{len(s)}x{s[0]}")
def test_clipping(sizes, dtypes):
    grads = _list(sizes, dtypes, seed=1)
    before = [g.clone() for g in grads]
    versions = [g._version for g in grads]
    norm = maxsim_amd.clip_grad_norm(grads, 1e-3, eps=1e-9)
    want = _check_norm(norm, before)
    factor = oracle.clip_factor(want, 1e-3, 1e-9)
    for g, b in zip(grads, before):
        # the factor's rounding, the product's in fp32, the result's
        assert_within(g, f64(b) * factor, 2 * U32 * np.abs(f64(b) * factor) + TINY[torch.float32])
    assert all(g._version > v for g, v in zip(grads, versions))
    # one factor for all
    _, f = maxsim_amd.clip_factor(before, 1e-3, eps=1e-9)
    for g, b in zip(grads, before):
        assert torch.equal(g, (b.float() * f).to(b.dtype))


def test_within_the_limit_nothing_moves():
    grads = _list(SIZES, DTYPES, seed=2)
    before = [g.clone() for g in grads]
    maxsim_amd.clip_grad_norm(grads, 1e6)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))


def test_neighbours_in_memory_stay():
    flat = torch.ones(100001, dtype=torch.bfloat16, device="cuda")
    parts = [flat[3:40004], flat[40005:40006], flat[40007:100000]]
    maxsim_amd.clip_grad_norm(parts, 1.0)
    outside = torch.ones_like(flat, dtype=torch.bool)
    for lo, hi in ((3, 40004), (40005, 40006), (40007, 100000)):
        outside[lo:hi] = False
    assert bool((flat[outside] == 1).all()) and bool((flat[~outside] < 0.01).all())


def test_layouts():
    gen = torch.Generator().manual_seed(3)
    wide = rand(gen, 40, 60)
    for g in (wide[:, 3:50], wide.t(), wide[::2], wide[0].expand(7, 60), one_element_off(wide),
              rand(gen, 3, 4, 5).permute(2, 0, 1), torch.tensor(2.0, device="cuda")):
        _check_norm(maxsim_amd.grad_norm([g]), [g])
        _check_norm(maxsim_amd.grad_norm(g), [g])
        _check_norm(maxsim_amd.grad_norm(x for x in (g, g)), [g, g])
    turned = wide.clone().t()
    want = turned.clone()
    f = maxsim_amd.clip_factor([turned], 1.0)[1]
    maxsim_amd.clip_grad_norm(turned, 1.0)
    assert torch.equal(turned, want * f)


def test_the_same_bits_every_time():
    grads = _list([300007, 11, 70001], DTYPES, seed=4)
    first = maxsim_amd.clip_factor(grads, 1.0)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(maxsim_amd.clip_factor(grads, 1.0), first))


def test_captured():
    grads = _list([70001, 33, 4096], DTYPES, seed=5)
    fresh = [_list([70001, 33, 4096], DTYPES, seed=s, scale=10.0 ** -s) for s in (1, 2, 3, 4)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        maxsim_amd.clip_grad_norm([g.clone() for g in grads], 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = maxsim_amd.clip_grad_norm(grads, 1.0)
    for new in fresh:
        for g, n in zip(grads, new):
            g.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = maxsim_amd.clip_grad_norm(new, 1.0)
        assert torch.equal(norm, want)
        assert all(torch.equal(g, n) for g, n in zip(grads, new))


def test_another_stream():
    grads = _list([300007, 11], DTYPES, seed=6)
    want = maxsim_amd.clip_factor(grads, 1.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = maxsim_amd.clip_factor(grads, 1.0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_gradients():
    assert float(maxsim_amd.grad_norm([])) == 0.0
    assert float(maxsim_amd.clip_grad_norm([], 1.0)) == 0.0
    assert [float(x) for x in maxsim_amd.clip_factor((), 1.0)] == [0.0, 1.0]
    nothing = [torch.zeros(0, device="cuda"), torch.zeros(3, 0, device="cuda")]
    assert float(maxsim_amd.clip_grad_norm(nothing, 1.0)) == 0.0


def test_refusals():
    g = torch.ones(8, device="cuda")
    sparse = torch.eye(3, device="cuda").to_sparse()
    for error, match, call in (
            (TypeError, "grads", lambda: maxsim_amd.grad_norm([g.double()])),
            (TypeError, "dense", lambda: maxsim_amd.grad_norm([g, sparse])),
            (TypeError, "dense", lambda: maxsim_amd.clip_grad_norm([sparse], 1.0)),
            (ValueError, "max_norm", lambda: maxsim_amd.clip_factor([g], -1.0)),
            (ValueError, "max_norm", lambda: maxsim_amd.clip_grad_norm([g], math.nan)),
            (ValueError, "eps", lambda: maxsim_amd.clip_factor([g], 1.0, eps=-1.0)),
            (ValueError, "eps", lambda: maxsim_amd.clip_grad_norm([g], 1.0, eps=math.nan)),
            (RuntimeError, "device", lambda: maxsim_amd.grad_norm([g, g.cpu()])),
            (RuntimeError, "HIP", lambda: maxsim_amd.grad_norm([g.cpu()])),
            (ValueError, "gaps", lambda: maxsim_amd.clip_grad_norm([g[::2]], 1.0)),
            (ValueError, "gaps", lambda: maxsim_amd.clip_grad_norm([g[:1].expand(4)], 1.0)),
            (ValueError, "share memory", lambda: maxsim_amd.clip_grad_norm([g, g], 1.0)),
            (ValueError, "share memory", lambda: maxsim_amd.clip_grad_norm([g[:5], g[4:]], 1.0))):
        with pytest.raises(error, match=match):
            call()
    assert bool((g == 1).all())


# ---------------------------------------------------------------------------
# The step on clipped gradients
# ---------------------------------------------------------------------------
def _state(dtype, gdtype, bits, master, seed=0, sizes=(300, 4097, 70001)):
    gen = torch.Generator().manual_seed(seed)
    out = {k: [] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "scales", "masters")}
    for n in sizes:
        p = rand(gen, n)
        out["params"].append(p.to(dtype))
        out["grads"].append(rand(gen, n, dtype=gdtype))
        kind = torch.uint8 if bits == 8 else torch.float32
        out["exp_avgs"].append(torch.zeros(n, dtype=kind, device="cuda"))
        out["exp_avg_sqs"].append(torch.zeros(n, dtype=kind, device="cuda"))
        if bits == 8:
            out["scales"].append(torch.zeros((n + 255) // 256, 2, dtype=torch.uint8, device="cuda"))
        if master:
            out["masters"].append(p)
    return out


def _step(t, step, grads=None, **kw):
    maxsim_amd.adamw_step(t["params"], grads or t["grads"], t["exp_avgs"], t["exp_avg_sqs"], step=step,
                          lr=1e-2, scales=t["scales"] or None, masters=t["masters"] or None, seed=9,
                          **kw)


def _equal(a, b):
    return all(torch.equal(x, y) for k in a if k != "grads" for x, y in zip(a[k], b[k]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gdtype,master", [(torch.float32, torch.float32, False),
                                                 (torch.bfloat16, torch.float32, False),
                                                 (torch.bfloat16, torch.bfloat16, True),
                                                 (torch.float16, torch.float16, False),
                                                 (torch.float16, torch.float32, True)], ids=str)
def test_a_scaled_step_is_the_step_on_scaled_gradients(dtype, gdtype, master, bits):
    # the product in fp32, unrounded to the gradients' type: the step on fp32
    # gradients that are the products has the same bits
    a, b, c = (_state(dtype, gdtype, bits, master) for _ in range(3))
    kept = [g.clone() for g in a["grads"]]
    for step in (1, 2, 3):
        norm, factor = maxsim_amd.clip_factor(a["grads"], 1.0 / step)
        assert 0 < float(factor) < 1e-2
        _step(a, step, grad_scale=factor)
        _step(b, step, [g.float() * factor for g in b["grads"]])
        _step(c, step)
    assert _equal(a, b) and not _equal(a, c)
    assert all(torch.equal(g, k) for g, k in zip(a["grads"], kept))
    one = torch.ones(1, device="cuda")
    a, b = (_state(dtype, gdtype, bits, master) for _ in range(2))
    _step(a, 1, grad_scale=one)
    _step(b, 1)
    assert _equal(a, b)


def test_scale_refusals():
    t = _state(torch.float32, torch.float32, 32, False, sizes=(8,))
    for error, value in ((TypeError, torch.ones((), dtype=torch.float64, device="cuda")),
                         (ValueError, torch.ones(2, device="cuda")),
                         (RuntimeError, torch.ones(()))):
        with pytest.raises(error, match="grad_scale"):
            _step(t, 1, grad_scale=value)


def test_a_captured_clipped_step():
    a, b = (_state(torch.bfloat16, torch.bfloat16, 8, True) for _ in range(2))
    counts = torch.zeros(1, dtype=torch.int64, device="cuda")

    def run(t, step, norm_of):
        norm, factor = maxsim_amd.clip_factor(t["grads"], norm_of)
        _step(t, step, grad_scale=factor)
        return norm

    run(_state(torch.bfloat16, torch.bfloat16, 8, True), 1, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run(a, counts, 1.0)
    gen = torch.Generator().manual_seed(1)
    for step in (1, 2, 3, 4):
        counts.fill_(step)
        for x, y in zip(a["grads"], b["grads"]):
            x.copy_(rand(gen, *x.shape))
            y.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, run(b, step, 1.0))
        assert _equal(a, b), step


# ---------------------------------------------------------------------------
# The optimizer
# ---------------------------------------------------------------------------
def _params(dtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(rand(gen, *s, dtype=dtype)) for s in ((40, 30), (5,), (3000, 4))]


def _set_grads(params, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = rand(gen, *p.shape, dtype=p.dtype, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_the_optimizer_clips(dtype):
    a, b = _params(dtype), _params(dtype)
    groups = lambda p: [{"params": p[:2], "lr": 1e-2}, {"params": p[2:], "weight_decay": 0.0}]
    opt = maxsim_amd.AdamW(groups(a), state_bits=8, max_norm=0.5)
    plain = maxsim_amd.AdamW(groups(b), state_bits=8)
    for step in range(3):
        for p in (a, b):
            _set_grads(p, step, scale=10.0 ** (step - 2))
        kept = [p.grad.clone() for p in a]
        opt.step()
        # the norm is over all groups, and the gradients stay
        _check_norm(opt.grad_norm, kept)
        assert all(torch.equal(p.grad, k) for p, k in zip(a, kept))
        _, factor = maxsim_amd.clip_factor(kept, 0.5)
        for p in b:
            p.grad = p.grad.float() * factor if p.dtype == torch.float32 else p.grad
        if dtype == torch.float32:
            plain.step()
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_against_torch():
    # gradients clipped by torch, stepped by torch: the same numbers but for
    # fp32 roundings, a few 1e-7 of a step each
    a, b = _params(), _params()
    opt = maxsim_amd.AdamW(a, lr=1e-2, max_norm=1.0)
    theirs = torch.optim.AdamW(b, lr=1e-2)
    for step in range(5):
        for p in (a, b):
            _set_grads(p, step)
        opt.step()
        norm = torch.nn.utils.clip_grad_norm_(b, 1.0)
        theirs.step()
        assert float(opt.grad_norm) == pytest.approx(float(norm), rel=1e-5)
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y, rtol=0, atol=5 * 1e-2 * 1e-4)


def test_the_optimizer_without_gradients():
    params = _params()
    opt = maxsim_amd.AdamW(params, max_norm=1.0)
    opt.step()
    assert float(opt.grad_norm) == 0.0
    params[1].grad = torch.full_like(params[1], 2.0)
    opt.step()
    assert float(opt.grad_norm) == pytest.approx(2.0 * math.sqrt(5), rel=1e-6)
    assert opt.state[params[0]] == {}
    params[0].grad = torch.eye(40, 30, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()


def test_the_limit_survives_copies_and_stays_out_of_the_state_dict():
    params = _params()
    opt = maxsim_amd.AdamW(params, max_norm=0.25)
    other = copy.deepcopy(opt)
    assert other.max_norm == 0.25
    assert "max_norm" not in opt.state_dict()["param_groups"][0]
    fresh = maxsim_amd.AdamW(params, max_norm=0.5)
    fresh.load_state_dict(opt.state_dict())
    assert fresh.max_norm == 0.5
    for value in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            maxsim_amd.AdamW(params, max_norm=value)
