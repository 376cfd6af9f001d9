"""What lies around the scores in training and indexing: from an encoder's
hidden states to scored token embeddings, and the step that trains both.

* :func:`layer_norm` -- layer norm over the last axis, differentiable.
* :func:`normalize_embeddings` -- token embeddings of unit length, those of
  padding 0; :func:`pack_normalized_documents` -- the same, packed into the
  inputs of the contrastive functions.  Differentiable.
* :func:`adamw_step` and :class:`AdamW` -- the AdamW step over many tensors in
  a few launches, with states in 32 or 8 bits.

The reference leaves these to torch (its training example, README.md:160-205).
Here they are hand-written HIP kernels behind ``include/maxsim_amd_training.h``:
one pass over memory each, sums in fp32, 16-bit results rounded once.
Differentiable means first derivatives in reverse mode: the gradients have no
derivatives of their own and forward-mode tangents are not carried (both raise).
All are exported from :mod:`maxsim_amd`.
"""

from __future__ import annotations

import math
from typing import Tuple

import torch

from ._ops import ops

#: Elements of a parameter that share the scales of their 8-bit states.
STATE_BLOCK = 256


def _require_hip(name: str, t: torch.Tensor) -> None:
    # the operators are registered for HIP tensors alone, and without one the
    # dispatcher's error names no argument
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a HIP (torch 'cuda') tensor; got {t.device}")


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last axis.

    Args:
        x: ``[..., dim]`` fp32 / fp16 / bf16, dim up to 16384.  Leading axes
            that are not one run of rows are copied first.
        weight, bias: ``[dim]`` in x's dtype or fp32 (both alike); None: 1, 0.
        eps: added to the variance (over ``dim``), >= 0.

    Returns:
        ``x.shape`` in x's dtype.  Differentiable with respect to x, weight
        and bias, each gradient in its tensor's dtype (fp32 sums rounded
        once, in an order that the sizes alone decide).  Squares are fp32
        numbers: rows with elements past 1e19 have an infinite variance.
    """
    _require_hip("x", x)
    return ops.maxsim_layer_norm(x, weight, bias, eps)


# ---------------------------------------------------------------------------
# Token embeddings of unit length
# ---------------------------------------------------------------------------
def normalize_embeddings(x, lengths=None, *, eps: float = 1e-12) -> torch.Tensor:
    """``x / max(|x|, eps)`` for each token embedding.

    Args:
        x: ``[..., dim]`` fp32 / fp16 / bf16, dim up to 16384.
        lengths: ``[N]`` int32/int64 for x ``[N, L, dim]``: tokens at or past
            a sequence's length become 0 and are never read (they may hold
            NaN).  A length of 0 leaves the sequence without a token; lengths
            outside ``[0, L]`` are clamped.
        eps: at least 2^-126; a token no longer than it is divided by it.

    Returns:
        ``x.shape`` in x's dtype, differentiable with respect to x (padding
        gets a gradient of 0, whatever comes down for it).  Tokens of any
        finite length: the squares of long and short ones stay in range.
    """
    _require_hip("x", x)
    return ops.maxsim_normalize_embeddings(x, lengths, eps)


# The host waits in it; torch.compile runs it at a graph break.
@torch.compiler.disable
def _packed_layout(lengths, max_len: int):
    return ops.maxsim_length_offsets(lengths, max_len)


def pack_normalized_documents(doc_emb, doc_lengths, *,
                              eps: float = 1e-12) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`maxsim_amd.pack_documents` of :func:`normalize_embeddings` in one
    pass, differentiable: padded documents ``[Nb, Ld, D]`` with lengths
    ``[Nb]`` become ``(documents [total, D], document_offsets [Nb + 1] int32)``
    for the contrastive functions, with every row at unit length.

    Lengths are clamped to ``[0, Ld]``; the host waits for the total row count
    (the output's size).  Padding is never read and gets a gradient of 0."""
    if doc_emb.dim() != 3:
        raise ValueError(f"doc_emb must be 3-D [Nb, Ld, D]; got shape {tuple(doc_emb.shape)}")
    Nb, Ld, _ = doc_emb.shape
    if tuple(doc_lengths.shape) != (Nb,):
        raise ValueError(
            f"doc_lengths must have shape [Nb={Nb}]; got {tuple(doc_lengths.shape)}")
    _require_hip("doc_emb", doc_emb)
    lengths, offsets, total = _packed_layout(
        doc_lengths.to(doc_emb.device, non_blocking=True), Ld)
    return ops.maxsim_pack_normalized(doc_emb, lengths, offsets, total, eps), offsets


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, scales=None, masters=None,
               seed: int = 0) -> None:
    """One AdamW step (decoupled weight decay) over lists of tensors, in place::

        m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay)
            - lr / (1 - beta1^step) m / (sqrt(v) / sqrt(1 - beta2^step) + eps)

    Args:
        params: fp32 / fp16 / bf16 tensors on one device, each dense in memory
            in any order of its axes.  Nothing that the step updates may
            share memory with another tensor of the lists (ValueError).
        grads: their gradients, in the parameter's dtype or fp32.
        exp_avgs, exp_avg_sqs: the states, in the parameters' order in memory:
            fp32, or uint8 codes with ``scales``.
        step: number of this step, from 1; or an int64 tensor of one element
            on the device, read when the kernels run (for a captured graph).
        lr: a number, or an fp32 tensor of one element on the device.
        scales: for 8-bit states, a uint8 ``[ceil(numel / 256), 2]`` per
            parameter.  All states start as zeros.
        masters: fp32 tensors that 16-bit parameters are the rounding of; the
            step is taken on them.  Without them a 16-bit parameter is read,
            moved in fp32 and rounded to nearest, which loses steps smaller
            than half its spacing.  (What a step takes off an fp32 value,
            update and decay together, is rounded once, to the value's
            spacing.)
        seed: of the random rounding of 8-bit states, which depends on
            (seed, step, position of the element in the lists) alone; its low
            32 bits count.

    8-bit states keep 4 significant bits per element and a power-of-two scale
    per 256; they are rounded up or down at random in proportion, so that the
    moving averages keep moving by less than their spacing.  The step itself
    uses them unrounded.  A value that is not finite makes its block NaN."""
    params = list(params)
    grads, exp_avgs, exp_avg_sqs = list(grads), list(exp_avgs), list(exp_avg_sqs)
    scales, masters = list(scales or ()), list(masters or ())
    lr_tensor = lr if isinstance(lr, torch.Tensor) else None
    step_tensor = step if isinstance(step, torch.Tensor) else None
    if not params:
        if grads or exp_avgs or exp_avg_sqs or scales or masters:
            raise ValueError("adamw_step needs lists of one length; got no params")
        return
    _require_hip("params", params[0])
    ops.maxsim_adamw_step(
        params, grads, exp_avgs, exp_avg_sqs, scales, masters,
        0.0 if lr_tensor is not None else lr, lr_tensor, betas[0], betas[1], eps, weight_decay,
        1 if step_tensor is not None else step, step_tensor, seed)


def adamw_state_values(exp_avg, exp_avg_sq, scales) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the 8-bit states of a parameter stand for: the first and second
    moment in bf16, which holds them exactly."""
    _require_hip("exp_avg", exp_avg)
    return ops.maxsim_adamw_state_values(exp_avg, exp_avg_sq, scales)


def _check_options(group) -> None:
    if group["state_bits"] not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32; got {group['state_bits']}")
    for name in ("lr", "eps", "weight_decay"):
        value = group[name]
        if name == "lr" and isinstance(value, torch.Tensor):
            continue  # on the device; checked where it is used, but for its value
        if not (value >= 0.0 and math.isfinite(value)):
            raise ValueError(f"{name} must be finite and >= 0; got {value}")
    if len(group["betas"]) != 2 or not all(0.0 <= b < 1.0 for b in group["betas"]):
        raise ValueError(f"betas must be two numbers in [0, 1); got {tuple(group['betas'])}")


class AdamW(torch.optim.Optimizer):
    """AdamW on :func:`adamw_step`: every parameter of a group in a few
    launches, states in 32 or 8 bits.

    Args:
        params, lr, betas, eps, weight_decay: as ``torch.optim.AdamW``; lr may
            be an fp32 tensor of one element on the parameters' device.
        state_bits: 32, or 8 for parameters of at least ``min_8bit_size``
            elements (below it 8 bits save nothing that counts).
        master_weights: keep an fp32 copy of each 16-bit parameter and step on
            that (made at the parameter's first step; the parameter itself is
            then only written).
        seed: of the random rounding of 8-bit states.

    State of a parameter: ``step`` (an int), ``exp_avg``, ``exp_avg_sq``, and
    ``scales`` / ``master`` where they apply.  ``state_dict`` round trips keep
    the states' own dtypes, and ``load_state_dict`` takes
    ``torch.optim.AdamW``'s too.  The step count lives on the host: a captured
    graph would replay one step's, so ``step()`` refuses to be captured
    (:func:`adamw_step` takes it as a tensor)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, min_8bit_size: int = 4096,
                 master_weights: bool = False, seed: int = 0):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size,
                                      master_weights=master_weights, seed=seed))

    def add_param_group(self, param_group) -> None:
        """As torch's; a group's own options are checked like the defaults."""
        _check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _new_state(self, p, group) -> dict:
        eight = group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]
        dtype = torch.uint8 if eight else torch.float32
        state = {"step": 0, "exp_avg": torch.zeros_like(p, dtype=dtype),
                 "exp_avg_sq": torch.zeros_like(p, dtype=dtype)}
        if eight:
            blocks = (p.numel() + STATE_BLOCK - 1) // STATE_BLOCK
            state["scales"] = torch.zeros(blocks, 2, dtype=torch.uint8, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        """Step every parameter that has a gradient; returns the closure's loss."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step() counts its steps on the host and cannot be captured; "
                               "use adamw_step with a step tensor")
        for at, group in enumerate(self.param_groups):
            # one call per device, step count and kind of state
            calls: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                elif group["master_weights"] and "master" not in state and p.dtype != torch.float32:
                    state["master"] = p.detach().to(torch.float32)  # loaded from elsewhere
                key = (p.device, state["step"], "scales" in state, "master" in state)
                calls.setdefault(key, []).append((p, state))
            for (_, step, eight, master), found in calls.items():
                states = [s for _, s in found]
                adamw_step([p for p, _ in found], [p.grad for p, _ in found],
                           [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                           step=step + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"],
                           scales=[s["scales"] for s in states] if eight else None,
                           masters=[s["master"] for s in states] if master else None,
                           seed=group["seed"] + at)
                for s in states:
                    s["step"] = step + 1
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch's, which casts a state to its parameter's dtype; here each
        keeps its own (8-bit codes, fp32 moments and masters).

        A ``torch.optim.AdamW``'s state dict is taken as well: its moments as
        fp32 states, whatever ``state_bits`` says of new ones, and a master is
        made at the next step where ``master_weights`` asks for one.  Options of
        this class that the dict does not have stay as they are.  ValueError for
        what this optimizer would step otherwise: ``amsgrad``, ``maximize``, a
        decay that is not decoupled, another optimizer's states."""
        # the last hook before torch's cast, which leaves what is no tensor
        handle = self.register_load_state_dict_pre_hook(_hold_states)
        try:
            super().load_state_dict(state_dict)
        finally:
            handle.remove()

    def __setstate__(self, state) -> None:
        # called with what is loaded, before the hooks that come after it
        for p, held in state["state"].items():
            if isinstance(p, torch.Tensor):
                for name, value in held.items():
                    if isinstance(value, _Held):
                        held[name] = value.tensor.to(device=p.device, copy=True)
        super().__setstate__(state)


class _Held:
    """A state's tensor on its way through torch's load_state_dict."""

    def __init__(self, tensor: torch.Tensor):
        self.tensor = tensor


def _hold_states(optimizer, state_dict) -> dict:
    """state_dict as this optimizer has it, its states' tensors held."""
    groups, owner = [], {}
    for saved, group in zip(state_dict["param_groups"], optimizer.param_groups):
        if saved.get("amsgrad") or saved.get("maximize"):
            raise ValueError("AdamW has no amsgrad and no maximize")
        if not saved.get("decoupled_weight_decay", True) and saved.get("weight_decay"):
            raise ValueError("AdamW's weight decay is decoupled; the loaded one is not")
        groups.append({**{k: v for k, v in group.items() if k != "params"}, **saved})
        _check_options(groups[-1])
        owner.update(zip(saved["params"], group["params"]))
    groups += state_dict["param_groups"][len(groups):]  # torch refuses another number of them
    states = {i: _hold_state(i, state, owner[i]) if i in owner else state
              for i, state in state_dict["state"].items()}
    return {**state_dict, "param_groups": groups, "state": states}


def _hold_state(i, state, p) -> dict:
    held = {}
    for name, value in state.items():
        if not isinstance(value, torch.Tensor):
            held[name] = value
        elif name == "step":
            held[name] = int(value)
        else:
            if name in ("exp_avg", "exp_avg_sq", "master") and value.shape == p.shape:
                if value.is_floating_point() and (value.dtype != torch.float32
                                                  or value.stride() != p.stride()):
                    value = torch.empty_like(p, dtype=torch.float32).copy_(value)
            held[name] = _Held(value)
    if held and not {"step", "exp_avg", "exp_avg_sq"} <= held.keys():
        raise ValueError(f"the state of parameter {i} has no step, exp_avg and exp_avg_sq: "
                         f"{sorted(held)}")
    if held and held["exp_avg"].tensor.dtype == torch.uint8 and "scales" not in held:
        raise ValueError(f"the state of parameter {i} has 8-bit codes without their scales")
    return held
