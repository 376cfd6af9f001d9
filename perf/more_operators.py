"""The measured cases of the operators at the two ends of a training step: the
ones that make an encoder's first hidden states from token ids, and that keep
the gradients' length within bounds before the parameters move.

* token ids looked up in an embedding table, with a scale, and the table's
  gradient;
* the norm of all gradients together;
* gradients clipped to a norm in place;
* the AdamW step on gradients clipped on the way, which leaves them as they are.

``listed`` names the cases, ``draw`` gives others of the same ranges,
``prepare`` makes a case's inputs on the GPU from a seed, ``run`` is one pass
(the package's functions where ``own`` is true, the same formulas in
elementary torch operations where it is not), ``work`` its unavoidable bytes
and operations and ``exact`` its results in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}

STEP, LR, BETA1, BETA2, EPS, DECAY = 1000, 1e-4, 0.9, 0.999, 1e-8, 0.01
CLIP_EPS = 1e-6    # the usual one beside the norm in a clipping factor
ALIGN = 256        # elements from one tensor's start to the next one's, a multiple


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _embed(name, mode, dtype, vocab, n, length, dim, lo=0, wdtype=None, scaled=False, ids="text"):
    """``n`` sequences padded to ``length`` tokens, real lengths from ``lo`` up
    (0: no lengths, every token is real), looked up in ``vocab`` rows of
    ``dim``; the table in ``wdtype`` (the result's own type if not given),
    ``scaled`` by the root of ``dim``.  ids: "text" (few of them often) or
    "positions" (each token's place in its sequence)."""
    return dict(name=name, kind="embed", mode=mode, dtype=dtype, vocab=vocab, n=n, length=length,
                dim=dim, lo=lo, wdtype=wdtype or dtype, scaled=scaled, ids=ids)


def _grads(name, mode, dtype, gdtype, vocab, layers, hidden, inner, over=True, master=False):
    """An encoder of ``layers`` layers of ``hidden`` (0: the embedding head
    alone) with a feed-forward part of ``inner`` and ``vocab`` token
    embeddings; parameters in ``dtype``, gradients in ``gdtype``, whose norm is
    ``over`` the limit or under it; 32-bit masters of 16-bit parameters."""
    return dict(name=name, kind="grads", mode=mode, dtype=dtype, gdtype=gdtype, vocab=vocab,
                layers=layers, hidden=hidden, inner=inner, over=over, master=master)


def listed():
    return [
        # -- token embeddings
        # the smallest call: one server batch of 8 queries of 32 tokens
        _embed("embed_query_bf16", "infer", "bf16", 32000, 8, 32, 768),
        # an evaluation set's documents, token by token, into a narrow encoder
        _embed("embed_documents_f16", "infer", "f16", 50021, 501, 276, 384),
        # a training batch's queries: almost all of the gradient is zeros
        _embed("embed_train_queries_bf16", "train", "bf16", 32000, 64, 32, 768),
        # the largest contrastive batch's padded documents, the table kept in 32 bits
        _embed("embed_train_large_bf16", "train", "bf16", 32000, 512, 1024, 768, lo=128,
               wdtype="f32", scaled=True),
        # full precision, rows off any 16-byte boundary's multiple
        _embed("embed_train_f32_odd", "train", "f32", 50021, 389, 47, 301, lo=1),
        # a table of positions: every row is used by every sequence that is long enough
        _embed("embed_train_positions_f16", "train", "f16", 512, 64, 180, 768, lo=45,
               ids="positions"),
        # -- the norm of all gradients
        # the smallest call: a frozen encoder's embedding head
        _grads("norm_head_f32", "norm", "f32", "f32", 0, 0, 768, 0),
        # a whole encoder's, the token embeddings' among them
        _grads("norm_encoder_bf16", "norm", "bf16", "bf16", 32000, 12, 768, 2048),
        # -- clipping in place.  A clipped set is at the limit: the next pass
        # over the same one finds next to nothing to clip, so that the set
        # whose time goes to memory is one that is under it, as most steps' are
        _grads("clip_head_bf16", "clip", "bf16", "bf16", 0, 0, 768, 0),
        _grads("clip_encoder_f32", "clip", "f32", "f32", 32000, 12, 768, 2048, over=False),
        # -- the AdamW step on clipped gradients
        _grads("step_head_f32", "step", "f32", "f32", 0, 0, 768, 0),
        _grads("step_encoder_bf16", "step", "bf16", "bf16", 32000, 12, 768, 2048, master=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case.  Sizes are spread over their logarithm, odd ones among
    them; one that costs more than the largest listed is drawn again."""
    while True:
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if rng.random() < 0.6:
            length = _log_int(rng, 1, 1024)
            vocab, ids = _log_int(rng, 2, 131072), "text"
            if rng.random() < 0.2:
                ids, vocab = "positions", rng.randint(length, 2 * length)
            dim = rng.choice([64, 96, 128, 300, 301, 384, 768, 768, 2560, _log_int(rng, 64, 2560)])
            case = _embed("", rng.choice(["infer", "train", "train"]), dtype, vocab,
                          _log_int(rng, 1, 16384), length, dim,
                          lo=rng.choice([0, rng.randint(1, length)]),
                          wdtype=rng.choice([dtype, "f32"]), scaled=rng.choice([True, False]),
                          ids=ids)
            if case["n"] * length > 524288:
                continue
        else:
            hidden = rng.choice([96, 128, 300, 384, 389, 768])
            case = _grads("", rng.choice(["norm", "clip", "step"]), dtype,
                          rng.choice([dtype, dtype, "f32"]), rng.choice([0, _log_int(rng, 100, 32000)]),
                          rng.randint(0, 12), hidden, rng.randint(hidden, 3 * hidden),
                          over=rng.choice([True, False]),
                          master=dtype != "f32" and rng.choice([True, False]))
        del case["name"]
        if work(case)["bytes"] <= 1.7e9:
            return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _frequencies(vocab):
    """How often each token comes up: the r-th most frequent as 1 / (r + 2.7)."""
    p = 1 / (torch.arange(vocab, dtype=torch.float64) + 3.7)
    return p / p.sum()


def _lengths(n, lo, hi, gen):
    """Uniform lengths: the distribution's own quantiles in an order of the
    seed's, so that every seed has the same rows in all."""
    at = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    x = torch.floor(lo + at * (hi + 1 - lo)).to(torch.int64)
    return x[torch.randperm(n, generator=gen)]


def _prepare_embed(case, gen, host):
    n, length, vocab, dim = case["n"], case["length"], case["vocab"], case["dim"]
    train = case["mode"] == "train"
    weight = torch.randn(vocab, dim, generator=gen, device="cuda").mul_(0.02)
    if case["ids"] == "positions":
        ids = torch.arange(length, device="cuda").expand(n, length).contiguous()
    else:
        edges = _frequencies(vocab).cumsum(0).cuda()
        u = torch.rand(n, length, generator=gen, device="cuda", dtype=torch.float64)
        ids = torch.searchsorted(edges, u, right=True).clamp_(max=vocab - 1)
        ids[:, 0] = 1  # the token that every sequence starts with
    state = dict(weight=weight.to(DTYPES[case["wdtype"]]).requires_grad_(train), ids=ids,
                 lengths=None, scale=math.sqrt(dim) if case["scaled"] else 1.0)
    if case["lo"]:
        state["lengths"] = _lengths(n, case["lo"], length, host).cuda()
    if train:
        dy = torch.empty(n, length, dim, dtype=DTYPES[case["dtype"]], device="cuda")
        some = max(1, (1 << 26) // (length * dim))
        for i in range(0, n, some):  # part by part: the largest is large in 32 bits
            part = dy[i:i + some]
            part.copy_(torch.randn(*part.shape, generator=gen, device="cuda").mul_(1e-2))
        state["dy"] = dy
    return state


def _shapes(case):
    h, inner, vocab = case["hidden"], case["inner"], case["vocab"]
    layer = [(h, h), (h,)] * 4 + [(inner, h), (inner,), (h, inner), (h,)] + [(h,)] * 4
    table = [(vocab, h)] if vocab else []
    return table + layer * case["layers"] + [(h,), (h,), (128, h), (128,)]


def _limit(case):
    # 16-bit floats' gradients come with a loss scale: their smallest numbers are large
    return 1024.0 if case["gdtype"] == "f16" else 1.0


def _prepare_grads(case, gen):
    """The tensors are views of one buffer of each kind, each from a multiple
    of ALIGN elements; between them the buffers hold zeros."""
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // ALIGN) * ALIGN
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for at, n in zip(starts, sizes):
        used[at:at + n] = True

    def normal(scale):
        return torch.randn(total, generator=gen, device="cuda").mul_(scale).mul_(used)

    def views(flat):
        return [flat[at:at + n].view(s) for at, n, s in zip(starts, sizes, shapes)]

    # in the middle of training: gradients of many magnitudes, about twice as
    # long as the limit or half of it
    size = torch.exp(torch.randn(total, generator=gen, device="cuda"))
    grad = normal(1) * size
    far = _limit(case) * (2.0 if case["over"] else 0.5) / grad.double().norm()
    far = far * (0.8 + 0.4 * torch.rand((), generator=gen, device="cuda"))
    flat = {"grad": (grad * far).to(DTYPES[case["gdtype"]])}
    if case["mode"] == "step":
        size *= far
        flat["master"] = normal(0.03)
        flat["param"] = flat["master"].to(DTYPES[case["dtype"]])
        if not case["master"]:
            del flat["master"]
        flat["exp_avg"] = normal(0.12) * size
        flat["exp_avg_sq"] = (1 + 0.2 * normal(1)).abs() * (0.5 * size) ** 2 * used
    state = {"flat": flat, "max_norm": _limit(case)}
    for name in ("param", "grad", "exp_avg", "exp_avg_sq", "master"):
        state[name] = views(flat[name]) if name in flat else None
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "embed":
        state = _prepare_embed(case, gen, torch.Generator().manual_seed(seed))
    else:
        state = _prepare_grads(case, gen)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------
# One pass, plain
# ---------------------------------------------------------------------------
def _plain_embed(st):
    w, ids, lens = st["weight"].detach(), st["ids"], st["lengths"]
    dt = DTYPES[st["case"]["dtype"]]
    y = (w[ids].float() * st["scale"]).to(dt)
    real = None
    if lens is not None:
        real = torch.arange(ids.shape[1], device=ids.device) < lens[:, None]
        y = torch.where(real[..., None], y, 0)
    if "dy" not in st:
        return {"y": y}
    dy = st["dy"].float()
    if real is not None:
        dy, ids = dy[real], ids[real]
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, ids.reshape(-1), dy.reshape(-1, w.shape[1]))
    return {"y": y, "dweight": (dw * st["scale"]).to(w.dtype)}


def _plain_norm(flat):
    x = flat["grad"].float()
    return torch.sqrt((x * x).sum(dtype=torch.float64)).float()


def _plain_grads(st):
    f, mode = st["flat"], st["case"]["mode"]
    norm = _plain_norm(f)
    if mode == "norm":
        return {"norm": norm}
    factor = (st["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)
    g = f["grad"].float() * factor
    if mode == "clip":
        f["grad"].copy_(g)
        return {"norm": norm, "grad": f["grad"]}
    p = f["master"] if st["case"]["master"] else f["param"].float()
    m = f["exp_avg"] * BETA1 + g * (1 - BETA1)
    v = f["exp_avg_sq"] * BETA2 + (g * g) * (1 - BETA2)
    c1, c2 = 1 - BETA1 ** STEP, 1 - BETA2 ** STEP
    p = p * (1 - LR * DECAY) - (LR / c1) * (m / (torch.sqrt(v) / math.sqrt(c2) + EPS))
    f["param"].copy_(p)
    if st["case"]["master"]:
        f["master"].copy_(p)
    f["exp_avg"].copy_(m)
    f["exp_avg_sq"].copy_(v)
    return _step_outputs(st, norm)


def _step_outputs(st, norm):
    return {"norm": norm, **{k: v for k, v in st["flat"].items() if k != "grad"}}


# ---------------------------------------------------------------------------
# One pass, by the package
# ---------------------------------------------------------------------------
def _own_embed(st):
    import maxsim_amd

    y = maxsim_amd.embed_tokens(st["weight"], st["ids"], st["lengths"], scale=st["scale"],
                                dtype=DTYPES[st["case"]["dtype"]])
    if "dy" not in st:
        return {"y": y}
    (dw,) = torch.autograd.grad(y, st["weight"], st["dy"])
    return {"y": y.detach(), "dweight": dw}


def _own_grads(st):
    import maxsim_amd

    mode = st["case"]["mode"]
    if mode == "norm":
        return {"norm": maxsim_amd.grad_norm(st["grad"])}
    if mode == "clip":
        norm = maxsim_amd.clip_grad_norm(st["grad"], st["max_norm"], eps=CLIP_EPS)
        return {"norm": norm, "grad": st["flat"]["grad"]}
    norm, factor = maxsim_amd.clip_factor(st["grad"], st["max_norm"], eps=CLIP_EPS)
    maxsim_amd.adamw_step(st["param"], st["grad"], st["exp_avg"], st["exp_avg_sq"], step=STEP,
                          lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                          masters=st["master"], grad_scale=factor)
    return _step_outputs(st, norm)


def run(state):
    if state["case"]["kind"] == "embed":
        return _own_embed(state) if own else _plain_embed(state)
    return _own_grads(state) if own else _plain_grads(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs written once.  Of a table, the rows that some
    token is; of padding, the zeros that are written."""
    if case["kind"] == "embed":
        s, ws, dim = BYTES[case["dtype"]], BYTES[case["wdtype"]], case["dim"]
        padded = case["n"] * case["length"]
        real = padded * (case["lo"] + case["length"]) / (2 * case["length"]) if case["lo"] else padded
        if case["ids"] == "positions":
            rows = case["length"]
        else:
            p = _frequencies(case["vocab"])
            rows = float((1 - torch.exp(real * torch.log1p(-p))).sum())
        moved = 8 * real + rows * dim * ws + padded * dim * s
        if case["mode"] == "infer":
            return {"bytes": moved, "flops": real * dim}
        return {"bytes": moved + real * dim * s + case["vocab"] * dim * ws, "flops": 2 * real * dim}
    n = sum(math.prod(x) for x in _shapes(case))
    s, gs, mode = BYTES[case["dtype"]], BYTES[case["gdtype"]], case["mode"]
    if mode == "norm":
        return {"bytes": n * gs, "flops": 2 * n}
    if mode == "clip":
        return {"bytes": n * gs * (2 if case["over"] else 1), "flops": 3 * n}
    # the gradient in; the parameter and its states in and out; beside a master
    # the parameter itself is written only
    return {"bytes": n * (gs + 2 * s + 4 * 4 + (4 * 2 - s if case["master"] else 0)),
            "flops": 18 * n}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_embed(st):
    w, scale = st["weight"].detach().double(), st["scale"]
    n, length = st["ids"].shape
    lens = [length] * n if st["lengths"] is None else st["lengths"].tolist()
    y = torch.zeros(n, length, w.shape[1], dtype=torch.float64, device=w.device)
    for i, k in enumerate(lens):
        torch.index_select(w, 0, st["ids"][i, :k], out=y[i, :k])
    out = {"y": y.mul_(scale)}
    if "dy" in st:
        dw = torch.zeros_like(w)
        at = torch.cat([st["ids"][i, :k] for i, k in enumerate(lens)])
        rows = torch.cat([st["dy"][i, :k] for i, k in enumerate(lens)])
        for lo in range(0, w.shape[1], 256):  # some columns at a time
            dw[:, lo:lo + 256] = torch.zeros_like(dw[:, lo:lo + 256]).index_put_(
                (at,), rows[:, lo:lo + 256].double(), accumulate=True)
        out["dweight"] = dw.mul_(scale)
    return out


def _exact_grads(st):
    f, case = st["flat"], st["case"]
    norm = torch.stack([torch.linalg.vector_norm(t.double()) for t in st["grad"]]).square().sum().sqrt()
    if case["mode"] == "norm":
        return {"norm": norm}
    factor = min(1.0, st["max_norm"] / (float(norm) + CLIP_EPS))
    g = f["grad"].double() * factor
    if case["mode"] == "clip":
        return {"norm": norm, "grad": g}
    p = (f["master"] if case["master"] else f["param"]).double()
    m = torch.lerp(g, f["exp_avg"].double(), BETA1)
    v = torch.lerp(g.square(), f["exp_avg_sq"].double(), BETA2)
    mhat, vhat = m / (1 - BETA1 ** STEP), v / (1 - BETA2 ** STEP)
    p = p - LR * (mhat / (vhat.sqrt() + EPS) + DECAY * p)
    out = {"exp_avg": m, "exp_avg_sq": v, "param": p}
    if case["master"]:
        out["master"] = p
    return _step_outputs({"flat": {k: out[k] for k in f if k != "grad"}}, norm)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_embed(st) if case["kind"] == "embed" else _exact_grads(st)
