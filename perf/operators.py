"""The measured cases of the operators around the scoring kernels: the ones that
turn an encoder's hidden states into scored token embeddings, and that train
what made them.

* layer norm over the hidden states, forward and backward;
* token embeddings normalised to unit length, padded or packed on the way,
  forward and backward;
* the AdamW step over all of a model's tensors, with 32-bit and 8-bit states.

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

LN_EPS = 1e-5      # the usual one of encoders
NORM_EPS = 1e-12   # the usual one of unit embeddings
STEP, LR, BETA1, BETA2, EPS, DECAY = 1000, 1e-4, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256        # elements that share the scales of their 8-bit states


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _layer_norm(name, mode, dtype, rows, dim, wdtype=None):
    """``rows`` tokens of ``dim``; the weights in ``wdtype`` (the rows' own
    type if not given)."""
    return dict(name=name, kind="layer_norm", mode=mode, dtype=dtype, rows=rows, dim=dim,
                wdtype=wdtype or dtype)


def _normalize(name, mode, dtype, n, length, dim, lo=0):
    """``n`` sequences padded to ``length`` tokens of ``dim``, real lengths
    from ``lo`` up (0: no lengths, every token is real)."""
    return dict(name=name, kind="normalize", mode=mode, dtype=dtype, n=n, length=length, dim=dim,
                lo=lo)


def _adamw(name, dtype, gdtype, bits, layers, hidden, inner, master=False):
    """An encoder of ``layers`` layers (0: the embedding head alone) of
    ``hidden`` with a feed-forward part of ``inner``; parameters in
    ``dtype``, gradients in ``gdtype``, 32-bit masters of 16-bit parameters."""
    return dict(name=name, kind="adamw", dtype=dtype, gdtype=gdtype, bits=bits, layers=layers,
                hidden=hidden, inner=inner, master=master)


def listed():
    return [
        # -- layer norm of hidden states
        # the smallest call: one server batch of 8 queries of 32 tokens
        _layer_norm("ln_query_bf16", "infer", "bf16", 256, 768),
        # an evaluation set's documents through a narrow encoder's last norm
        _layer_norm("ln_documents_f16", "infer", "f16", 138276, 384),
        # the largest contrastive batch's document tokens, with the norm's
        # weights kept in 32 bits as mixed-precision training does
        _layer_norm("ln_train_large_bf16", "train", "bf16", 294912, 768, "f32"),
        # full-precision training, rows off any 16-byte boundary's multiple
        _layer_norm("ln_train_f32_odd", "train", "f32", 18433, 301),
        # a small batch of a wide model
        _layer_norm("ln_train_wide_bf16", "train", "bf16", 2049, 2560),
        # -- unit token embeddings
        # a training batch's queries, every token real
        _normalize("unit_queries_train_bf16", "train", "bf16", 64, 32, 128),
        # a reranker's 32,000 padded candidates
        _normalize("unit_candidates_f16", "infer", "f16", 32000, 300, 128, lo=32),
        # the largest contrastive batch's documents, normalised and packed
        _normalize("unit_pack_train_bf16", "pack", "bf16", 512, 1024, 128, lo=128),
        # an odd, ragged batch in full precision
        _normalize("unit_train_f32_odd", "train", "f32", 389, 413, 77, lo=1),
        # -- the AdamW step
        # the smallest call: a frozen encoder's embedding head
        _adamw("adamw_head_f32", "f32", "f32", 32, 0, 768, 0),
        # a whole encoder in full precision
        _adamw("adamw_encoder_f32", "f32", "f32", 32, 12, 768, 2048),
        # the same in bf16 with 32-bit masters and 8-bit states
        _adamw("adamw_encoder_bf16_8bit", "bf16", "bf16", 8, 12, 768, 2048, master=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case.  Sizes are spread over their logarithm, odd ones among
    them; one that costs more than the largest listed is drawn again."""
    while True:
        kind = rng.choice(["layer_norm", "normalize", "adamw"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if kind == "layer_norm":
            dim = rng.choice([64, 96, 128, 256, 300, 301, 384, 768, 768, 2560, _log_int(rng, 64, 2560)])
            case = _layer_norm("", rng.choice(["infer", "train", "train"]), dtype,
                               _log_int(rng, 1, 294912), dim, rng.choice([dtype, "f32"]))
        elif kind == "normalize":
            mode = rng.choice(["infer", "train", "pack"])
            length = _log_int(rng, 8, 1024)
            lo = rng.randint(1, length)
            case = _normalize("", mode, dtype, _log_int(rng, 1, 32000), length,
                              rng.choice([64, 77, 96, 128, 128, 128, 256, 300, 768]),
                              lo=lo if mode == "pack" else rng.choice([0, lo]))
        else:
            hidden = rng.choice([96, 128, 300, 384, 389, 768])
            bits = rng.choice([8, 32])
            case = _adamw("", dtype, rng.choice([dtype, "f32"]), bits, rng.randint(0, 12), hidden,
                          rng.randint(hidden, 3 * hidden),
                          master=dtype != "f32" and rng.choice([True, False]))
        del case["name"]
        if work(case)["bytes"] <= 1.9e9:
            return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _lengths(n, lo, hi, gen):
    """Uniform lengths: the distribution's own quantiles in an order of the
    seed's, so that every seed has the same rows in all."""
    at = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    x = torch.floor(lo + at * (hi + 1 - lo)).to(torch.int64)
    return x[torch.randperm(n, generator=gen)]


def _prepare_layer_norm(case, gen):
    rows, dim = case["rows"], case["dim"]
    # hidden states: a spread of its own for each column, a few of them large
    spread = torch.exp(0.5 * torch.randn(dim, generator=gen, device="cuda"))
    spread[torch.randint(0, dim, (3,), generator=gen, device="cuda")] *= 8
    x = torch.randn(rows, dim, generator=gen, device="cuda").mul_(spread).add_(0.1 * spread)
    w = 1 + 0.1 * torch.randn(dim, generator=gen, device="cuda")
    b = 0.1 * torch.randn(dim, generator=gen, device="cuda")
    wd, train = DTYPES[case["wdtype"]], case["mode"] == "train"
    state = dict(x=x.to(DTYPES[case["dtype"]]).requires_grad_(train),
                 weight=w.to(wd).requires_grad_(train), bias=b.to(wd).requires_grad_(train))
    if train:
        dy = torch.randn(rows, dim, generator=gen, device="cuda").mul_(1e-2)
        state["dy"] = dy.to(DTYPES[case["dtype"]])
    return state


def _prepare_normalize(case, gen, host):
    n, length, dim, dt = case["n"], case["length"], case["dim"], DTYPES[case["dtype"]]
    # a projection's outputs: the rows' norms differ
    x = torch.empty(n, length, dim, dtype=dt, device="cuda")
    some = max(1, (1 << 26) // (length * dim))
    for i in range(0, n, some):  # part by part: the largest set is large in 32 bits
        part = torch.randn(min(some, n - i), length, dim, generator=gen, device="cuda")
        part *= torch.exp(0.3 * torch.randn(*part.shape[:2], 1, generator=gen, device="cuda"))
        x[i:i + some] = part
    state = dict(x=x.requires_grad_(case["mode"] != "infer"), lengths=None)
    rows = n * length
    if case["lo"]:
        lens = _lengths(n, case["lo"], length, host)
        state["lengths"] = lens.to(torch.int32).cuda()
        rows = int(lens.sum())
    if case["mode"] != "infer":
        shape = (rows, dim) if case["mode"] == "pack" else (n, length, dim)
        dy = torch.randn(*shape, generator=gen, device="cuda").mul_(1e-2)
        state["dy"] = dy.to(dt)
    return state


def _shapes(case):
    h, inner = case["hidden"], case["inner"]
    layer = [(h, h), (h,)] * 4 + [(inner, h), (inner,), (h, inner), (h,)] + [(h,)] * 4
    return layer * case["layers"] + [(h,), (h,), (128, h), (128,)]


def _prepare_adamw(case, gen, seed):
    """The tensors are views of one buffer of each kind, each from a whole
    block of BLOCK elements; between them the buffers hold zeros."""
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for at, n in zip(starts, sizes):
        used[at:at + n] = True

    def normal(scale):
        return torch.randn(total, generator=gen, device="cuda").mul_(scale).mul_(used)

    def views(flat):
        return [flat[at:at + n].view(s) for at, n, s in zip(starts, sizes, shapes)]

    # in the middle of training: gradients of many magnitudes
    size = torch.exp(torch.randn(total, generator=gen, device="cuda")) * 1e-4
    flat = {"master": normal(0.03)}
    flat["param"] = flat["master"].to(DTYPES[case["dtype"]])
    if not case["master"]:
        del flat["master"]
    flat["grad"] = (normal(1) * size).to(DTYPES[case["gdtype"]])
    flat["exp_avg"] = normal(0.25) * size
    flat["exp_avg_sq"] = (1 + 0.2 * normal(1)).abs() * size * size * used
    if case["bits"] == 8:
        m8, em = _encode(flat["exp_avg"], True, _dither(total, 0, 0, "cuda")[0])
        v8, ev = _encode(flat["exp_avg_sq"], False, _dither(total, 0, 0, "cuda")[1])
        flat.update(exp_avg=m8, exp_avg_sq=v8, scales=torch.stack([em, ev], 1).contiguous())
    state = {"flat": flat, "seed": seed & 0xffff}
    for name in ("param", "grad", "exp_avg", "exp_avg_sq", "master"):
        state[name] = views(flat[name]) if name in flat else None
    state["scales"] = None
    if case["bits"] == 8:
        state["scales"] = [flat["scales"][at // BLOCK:(at + n + BLOCK - 1) // BLOCK]
                           for at, n in zip(starts, sizes)]
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "layer_norm":
        state = _prepare_layer_norm(case, gen)
    elif case["kind"] == "normalize":
        state = _prepare_normalize(case, gen, torch.Generator().manual_seed(seed))
    else:
        state = _prepare_adamw(case, gen, seed)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------
# The 8-bit states
# ---------------------------------------------------------------------------
# A block of BLOCK elements shares, for each of its two states, the exponent
# field E of its largest magnitude.  A first moment is a sign and a magnitude
# of 4 exponent and 3 mantissa bits with the largest at exponent field 14; a
# second moment has no sign and 5 exponent bits, the largest at 30.  The codes
# are the top bits of the 32-bit pattern of the value moved to that exponent,
# rounded up or down at random in proportion (20 bits of a hash of the
# element's position, the step and the seed are added below the cut).  A second
# moment that is not 0 never becomes 0.  E = 255: the block held a value that
# is not finite, and stands for NaN.
TOP = {True: 14, False: 30}
LOWEST = {True: 32, False: 48}


def _pow2(k):
    return ((k + 127) << 23).view(torch.float32)


def _dither(n, step, seed, device):
    """20 bits for each of the two states of ``n`` elements."""
    low = 0xffffffff
    key = (seed * 0x9e3779b1 + step * 0x3c6ef373) & low
    i = torch.arange(n, dtype=torch.int64, device=device)
    x = ((i & low) * 0x9e3779b1 + (i >> 32) * 0xa54ff53b + key) & low
    x = x ^ (x >> 16)
    x = (x * 0x6a09e667) & low
    x = x ^ (x >> 15)
    x = (x * 0xbb67ae85) & low
    x = x ^ (x >> 16)
    return ((x & 0xffff) * 16 + 8).to(torch.int32), ((x >> 16) * 16 + 8).to(torch.int32)


def _encode(x, signed, dither):
    """fp32 [n] (n a multiple of BLOCK) -> codes uint8 [n], exponents uint8 [n / BLOCK]."""
    a = x.abs()
    e = (a.view(torch.int32).view(-1, BLOCK).amax(1) >> 23).clamp(min=LOWEST[signed])
    fine = (e < 255)[:, None]
    scale = _pow2(TOP[signed] + 126 - e.clamp(max=254))[:, None]
    u = (a.view(-1, BLOCK) * scale * 2.0 ** -126).view(torch.int32)
    q = (u + dither.view(-1, BLOCK)) >> 20
    if signed:
        q = q | (torch.signbit(x).to(torch.int32) << 7).view(-1, BLOCK)
    else:
        q = torch.where((a.view(-1, BLOCK) > 0) & (q == 0), 1, q)
    q = torch.where(fine, q, 0)
    return q.to(torch.uint8).view(-1), e.to(torch.uint8)


def _decode(codes, e, signed):
    q, e = codes.to(torch.int32).view(-1, BLOCK), e.to(torch.int32)[:, None]
    # E of a state that was never written is 0, and so are its codes
    scale = _pow2(e.clamp(LOWEST[signed], 254) - TOP[signed] - 126)
    x = ((q & 127 if signed else q) << 20).view(torch.float32) * 2.0 ** 126 * scale
    if signed:
        x = torch.where(q > 127, -x, x)
    return torch.where(e == 255, math.nan, x).view(-1)


# ---------------------------------------------------------------------------
# One pass, plain
# ---------------------------------------------------------------------------
def _plain_layer_norm(st):
    dt = st["x"].dtype
    x, w, b = (st[k].detach().float() for k in ("x", "weight", "bias"))
    xc = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + LN_EPS)
    xhat = xc * rstd
    y = (xhat * w + b).to(dt)
    if "dy" not in st:
        return {"y": y}
    dy = st["dy"].float()
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = rstd * (g - c1 - xhat * c2)
    wd = st["weight"].dtype
    return {"y": y, "dx": dx.to(dt), "dweight": (dy * xhat).sum(0).to(wd),
            "dbias": dy.sum(0).to(wd)}


def _plain_normalize(st):
    x, lens, mode = st["x"].detach().float(), st["lengths"], st["case"]["mode"]
    dt = st["x"].dtype
    norm = torch.sqrt((x * x).sum(2, keepdim=True))
    inv = 1 / norm.clamp(min=NORM_EPS)
    y = x * inv
    real = None
    if lens is not None:
        real = torch.arange(x.shape[1], device=x.device) < lens[:, None]
    out = {}
    if mode == "pack":
        out["documents"] = y[real].to(dt)
        off = torch.zeros(lens.numel() + 1, dtype=torch.int32, device=x.device)
        off[1:] = lens.cumsum(0)
        out["offsets"] = off
        dy = torch.zeros_like(y)
        dy[real] = st["dy"].float()
    else:
        out["y"] = (y if real is None else torch.where(real[..., None], y, 0)).to(dt)
        if mode == "infer":
            return out
        dy = st["dy"].float()
    along = torch.where(norm > NORM_EPS, (y * dy).sum(2, keepdim=True), 0)
    dx = inv * (dy - y * along)
    out["dx"] = (dx if real is None else torch.where(real[..., None], dx, 0)).to(dt)
    return out


def _plain_adamw(st):
    f, case = st["flat"], st["case"]
    eight = case["bits"] == 8
    p = f["master"] if case["master"] else f["param"].float()
    g = f["grad"].float()
    m, v = f["exp_avg"], f["exp_avg_sq"]
    if eight:
        m, v = _decode(m, f["scales"][:, 0], True), _decode(v, f["scales"][:, 1], False)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    c1, c2 = 1 - BETA1 ** STEP, 1 - BETA2 ** STEP
    p = p * (1 - LR * DECAY) - (LR / c1) * (m / (torch.sqrt(v) / math.sqrt(c2) + EPS))
    f["param"].copy_(p)
    if case["master"]:
        f["master"].copy_(p)
    if eight:
        dm, dv = _dither(m.numel(), STEP, st["seed"], m.device)
        m8, em = _encode(m, True, dm)
        v8, ev = _encode(v, False, dv)
        f["exp_avg"].copy_(m8)
        f["exp_avg_sq"].copy_(v8)
        f["scales"].copy_(torch.stack([em, ev], 1))
        m = _decode(m8, em, True).to(torch.bfloat16)  # 4 significant bits: exact in bf16
        v = _decode(v8, ev, False).to(torch.bfloat16)
    else:
        f["exp_avg"].copy_(m)
        f["exp_avg_sq"].copy_(v)
        m, v = f["exp_avg"], f["exp_avg_sq"]
    return _adamw_outputs(st, m, v)


def _adamw_outputs(st, m, v):
    out = {"param": st["flat"]["param"], "exp_avg": m, "exp_avg_sq": v}
    if st["case"]["master"]:
        out["master"] = st["flat"]["master"]
    return out


# ---------------------------------------------------------------------------
# One pass, by the package
# ---------------------------------------------------------------------------
def _own_layer_norm(st):
    import maxsim_amd

    y = maxsim_amd.layer_norm(st["x"], st["weight"], st["bias"], eps=LN_EPS)
    if "dy" not in st:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_normalize(st):
    import maxsim_amd

    mode = st["case"]["mode"]
    if mode == "pack":
        d, off = maxsim_amd.pack_normalized_documents(st["x"], st["lengths"], eps=NORM_EPS)
        (dx,) = torch.autograd.grad(d, st["x"], st["dy"])
        return {"documents": d.detach(), "offsets": off, "dx": dx}
    y = maxsim_amd.normalize_embeddings(st["x"], st["lengths"], eps=NORM_EPS)
    if mode == "infer":
        return {"y": y}
    (dx,) = torch.autograd.grad(y, st["x"], st["dy"])
    return {"y": y.detach(), "dx": dx}


def _own_adamw(st):
    import maxsim_amd

    maxsim_amd.adamw_step(st["param"], st["grad"], st["exp_avg"], st["exp_avg_sq"], step=STEP,
                          lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                          masters=st["master"], scales=st["scales"], seed=st["seed"])
    f = st["flat"]
    m, v = f["exp_avg"], f["exp_avg_sq"]
    if st["scales"] is not None:
        m, v = maxsim_amd.adamw_state_values(m, v, f["scales"])
    return _adamw_outputs(st, m, v)


def run(state):
    kind = state["case"]["kind"]
    if kind == "layer_norm":
        return _own_layer_norm(state) if own else _plain_layer_norm(state)
    if kind == "normalize":
        return _own_normalize(state) if own else _plain_normalize(state)
    return _own_adamw(state) if own else _plain_adamw(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs written once; tokens behind a sequence's
    length are written, never read."""
    s, kind = BYTES[case["dtype"]], case["kind"]
    if kind == "layer_norm":
        n, w = case["rows"] * case["dim"], case["dim"] * BYTES[case["wdtype"]]
        if case["mode"] == "infer":
            return {"bytes": 2 * n * s + 2 * w, "flops": 7 * n}
        return {"bytes": 4 * n * s + 4 * w, "flops": 19 * n}
    if kind == "normalize":
        padded = case["n"] * case["length"] * case["dim"]
        real = padded * (case["lo"] + case["length"]) / (2 * case["length"]) if case["lo"] else padded
        if case["mode"] == "infer":
            return {"bytes": (real + padded) * s, "flops": 3 * real}
        out = real if case["mode"] == "pack" else padded
        return {"bytes": (2 * real + out + padded) * s, "flops": 9 * real}
    n = sum(math.prod(x) for x in _shapes(case))
    # the gradient in; the parameter and its states in and out
    moved = BYTES[case["gdtype"]] + 2 * s + (4 * 2 if case["bits"] == 32 else 2 * 2)
    if case["master"]:
        moved += 4 * 2 - s  # the parameter itself is written only
    if case["bits"] == 8:
        moved += 2 * 2 + 4 / BLOCK  # the states' values out, and the scales
    return {"bytes": n * moved, "flops": 15 * n}


# ---------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_layer_norm(st):
    x, w, b = (st[k].detach().double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    xhat = (x - mean) / (var + LN_EPS).sqrt()
    out = {"y": xhat * w + b}
    if "dy" in st:
        dy = st["dy"].double()
        n = x.shape[1]
        g = dy * w
        out["dweight"], out["dbias"] = (dy * xhat).sum(0), dy.sum(0)
        along = (g * xhat).sum(1, keepdim=True)
        out["dx"] = (g - (g.sum(1, keepdim=True) + xhat * along) / n) / (var + LN_EPS).sqrt()
    return out


def _exact_normalize(st):
    """Document by document: row by row of a document, y = x / |x| and
    dx = (dy - y <y, dy>) / |x|, in the real tokens alone."""
    x, case = st["x"].detach(), st["case"]
    n, length, dim = x.shape
    lens = [length] * n if st["lengths"] is None else st["lengths"].tolist()
    out = {}
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for i, k in enumerate(lens):
        row = x[i, :k].double()
        y[i, :k] = row / torch.linalg.vector_norm(row, dim=1, keepdim=True).clamp_min(NORM_EPS)
    if case["mode"] == "pack":
        out["documents"] = torch.cat([y[i, :k] for i, k in enumerate(lens)])
        out["offsets"] = None
    else:
        out["y"] = y
    if case["mode"] != "infer":
        dx = torch.zeros_like(y)
        at = 0
        for i, k in enumerate(lens):
            dy = st["dy"][at:at + k] if case["mode"] == "pack" else st["dy"][i, :k]
            at += k
            u, d = y[i, :k], dy.double()
            size = torch.linalg.vector_norm(x[i, :k].double(), dim=1, keepdim=True)
            dx[i, :k] = (d - u * (u * d).sum(1, keepdim=True)) / size
        out["dx"] = dx
    return out


def _exact_codes(x, signed, dither):
    """The values of the 8-bit states in 64 bits: the two grid neighbours of
    each magnitude, and the upper one where the dither reaches past the rest."""
    a = x.abs().view(-1, BLOCK)
    top = a.amax(1, keepdim=True)
    e = torch.frexp(top.clamp_min(1e-300)).exponent - 1  # top in [2^e, 2^(e + 1))
    e = e.clamp(min=LOWEST[signed] - 127)
    low = e - (TOP[signed] - 1)  # exponent of the smallest normal magnitude
    own_e = torch.maximum(torch.frexp(a.clamp_min(1e-300)).exponent - 1, low.expand_as(a))
    grid = ((own_e.to(torch.int64) - 3 + 1023) << 52).view(torch.float64)  # 2^(own_e - 3)
    down = torch.floor(a / grid)
    up = (a / grid - down) * 2 ** 20 + dither.view(-1, BLOCK) >= 2 ** 20
    value = (down + up) * grid
    if not signed:
        value = torch.where((a > 0) & (value == 0), grid, value)
    return (torch.sign(x).view(-1, BLOCK) * value).view(-1)


def _exact_adamw(st):
    f, case = st["flat"], st["case"]
    p = (f["master"] if case["master"] else f["param"]).double()
    g = f["grad"].double()
    m, v = f["exp_avg"], f["exp_avg_sq"]
    if case["bits"] == 8:  # exact: a few bits moved by a power of two
        m, v = _decode(m, f["scales"][:, 0], True), _decode(v, f["scales"][:, 1], False)
    m = torch.lerp(g, m.double(), BETA1)
    v = torch.lerp(g.square(), v.double(), BETA2)
    mhat, vhat = m / (1 - BETA1 ** STEP), v / (1 - BETA2 ** STEP)
    p = p - LR * (mhat / (vhat.sqrt() + EPS) + DECAY * p)
    if case["bits"] == 8:
        dm, dv = _dither(m.numel(), STEP, st["seed"], m.device)
        m, v = _exact_codes(m, True, dm), _exact_codes(v, False, dv)
    out = {"param": p, "exp_avg": m, "exp_avg_sq": v}
    if case["master"]:
        out["master"] = p
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "layer_norm":
            return _exact_layer_norm(st)
        if case["kind"] == "normalize":
            return _exact_normalize(st)
        return _exact_adamw(st)
