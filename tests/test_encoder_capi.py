"""The C ABI of token embeddings, the gradients' norm and the clipped step (CPU
only: exports and argument checks, nothing is launched)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LIB = ROOT / "maxsim_amd" / "libmaxsim_amd.so"
OK, INVALID, UNSUPPORTED = 0, 1, 2
F32, F16, BF16 = 0, 1, 2
I64, P, F, D, SIZE = (ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_double,
                      ctypes.c_size_t)
INT = ctypes.c_int
ONE = P(16)


class Grad(ctypes.Structure):
    _fields_ = [("grad", P), ("numel", I64), ("dtype", INT)]


@pytest.fixture(scope="module")
def lib():
    handle = ctypes.CDLL(str(LIB))
    handle.maxsim_amd_last_error.restype = ctypes.c_char_p
    return handle


def test_every_declared_symbol_is_exported(lib):
    text = (ROOT / "include" / "maxsim_amd_encoder.h").read_text()
    names = re.findall(r"^\s*(?:int|size_t)\s+(maxsim_amd_\w+)\s*\(", text, re.M)
    assert len(set(names)) == 7
    for name in names:
        assert hasattr(lib, name), name


def test_embed_forward_refusals(lib):
    fn = lib.maxsim_amd_embed_forward
    fn.argtypes = [INT, INT, P, I64, I64, I64, P, INT, I64, I64, P, INT, F, I64, P, P, P]

    def call(wdtype=F32, dtype=BF16, weight=ONE, vocab=9, dim=64, stride=64, ids=ONE, n=2, length=3,
             y=ONE, rows=None):
        return fn(wdtype, dtype, weight, vocab, dim, stride, ids, 1, n, length, None, 0, 1.0, -1, y,
                  rows, None)

    assert call(n=0, ids=None, y=None) == OK and call(length=0, ids=None, y=None) == OK
    for kw, text in ((dict(dtype=5), b"dtype"), (dict(wdtype=5), b"dtype"),
                     (dict(wdtype=F16), b"weight_dtype"), (dict(wdtype=BF16, dtype=F32), b"weight_dtype"),
                     (dict(dim=0), b"dim"), (dict(vocab=-1), b"negative"), (dict(n=-1), b"negative"),
                     (dict(length=-1), b"negative"), (dict(stride=-1), b"stride"),
                     (dict(weight=None), b"null"), (dict(ids=None), b"null"), (dict(y=None), b"null")):
        assert call(**kw) == INVALID, kw
        assert text in lib.maxsim_amd_last_error()
    for kw in (dict(dim=16385), dict(vocab=2 ** 31), dict(length=2 ** 31),
               dict(n=2 ** 21, length=2 ** 10, rows=ONE)):
        assert call(**kw) == UNSUPPORTED, kw


def test_embed_backward_refusals(lib):
    size = lib.maxsim_amd_embed_backward_workspace_size
    size.restype, size.argtypes = SIZE, [INT, I64, I64, I64]
    assert size(BF16, 100, 9, 16385) == 0 and size(BF16, -1, 9, 64) == 0
    assert size(BF16, 2 ** 31, 9, 64) == 0 and size(9, 100, 9, 64) == 0
    need = size(BF16, 10000, 9, 64)
    assert need >= 10000 * 16
    assert size(BF16, 600, 9, 64) == 0 == size(BF16, 2048, 96, 64)  # few tokens need none
    fn = lib.maxsim_amd_embed_backward
    fn.argtypes = [INT, INT, P, I64, P, I64, I64, I64, F, P, P, SIZE, P]

    def call(wdtype=F32, dtype=BF16, dy=ONE, stride=64, rows=ONE, tokens=10000, vocab=9, dim=64,
             dw=ONE, ws=ONE, ws_bytes=need):
        return fn(wdtype, dtype, dy, stride, rows, tokens, vocab, dim, 1.0, dw, ws, ws_bytes, None)

    assert call(vocab=0, dw=None, ws=None) == OK
    for kw, text in ((dict(dtype=5), b"dtype"), (dict(wdtype=F16), b"weight_dtype"),
                     (dict(tokens=-1), b"negative"), (dict(stride=-1), b"stride"),
                     (dict(dy=None), b"null"), (dict(rows=None), b"null"), (dict(dw=None), b"null"),
                     (dict(ws=None), b"workspace"), (dict(ws_bytes=need - 1), b"workspace")):
        assert call(**kw) == INVALID, kw
        assert text in lib.maxsim_amd_last_error()
    assert call(tokens=2 ** 31) == UNSUPPORTED


def test_gradient_list_refusals(lib):
    size = lib.maxsim_amd_grad_norm_workspace_size
    size.restype, size.argtypes = SIZE, [P, I64]
    norm = lib.maxsim_amd_grad_norm
    norm.argtypes = [P, I64, D, D, P, P, P, SIZE, P]
    clip = lib.maxsim_amd_clip_grads
    clip.argtypes = norm.argtypes
    good = (Grad * 2)(Grad(ONE, 5, F32), Grad(ONE, 10 ** 6, BF16))
    need = size(good, 2)
    assert need % 8 == 0 and 8 * 2 <= need <= 8 * 1000
    assert size(None, 0) == 0 and size((Grad * 1)(Grad(ONE, 5, 7)), 1) == 0
    for bad, text in ((Grad(ONE, 5, 7), b"dtype"), (Grad(ONE, -1, F32), b"negative"),
                      (Grad(None, 1, F32), b"null")):
        one = (Grad * 1)(bad)
        for fn in (norm, clip):
            assert fn(one, 1, 1.0, 0.0, ONE, ONE, ONE, 64, None) == INVALID
            assert text in lib.maxsim_amd_last_error()
    for args, text in (((None, 2, 1.0, 0.0, ONE, ONE, ONE, need), b"no tensors"),
                       ((good, -1, 1.0, 0.0, ONE, ONE, ONE, need), b"no tensors"),
                       ((good, 2, 1.0, 0.0, None, ONE, ONE, need), b"null"),
                       ((good, 2, -1.0, 0.0, ONE, ONE, ONE, need), b"max_norm"),
                       ((good, 2, float("nan"), 0.0, ONE, ONE, ONE, need), b"max_norm"),
                       ((good, 2, 1.0, -1.0, ONE, ONE, ONE, need), b"max_norm"),
                       ((good, 2, 1.0, 0.0, ONE, ONE, None, need), b"workspace"),
                       ((good, 2, 1.0, 0.0, ONE, ONE, ONE, need - 1), b"workspace")):
        for fn in (norm, clip):
            assert fn(*args, None) == INVALID, text
            assert text in lib.maxsim_amd_last_error()
    assert clip(good, 2, 1.0, 0.0, ONE, None, ONE, need, None) == INVALID
    large = (Grad * 1)(Grad(ONE, 2 ** 50, F32))
    assert clip(large, 1, 1.0, 0.0, ONE, ONE, ONE, need, None) == UNSUPPORTED


def test_scaled_step_refusals(lib):
    fn = lib.maxsim_amd_adamw_step_scaled
    fn.argtypes = [INT, INT, INT, P, I64, P, D, P, D, D, D, D, I64, P, ctypes.c_uint64, P]
    assert fn(F32, F32, 32, None, 0, ONE, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 1, None, 0, None) == OK
    assert fn(F32, F32, 16, None, 0, ONE, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 1, None, 0,
              None) == INVALID
    assert b"state_bits" in lib.maxsim_amd_last_error()


def test_the_operators_are_exported():
    import maxsim
    import maxsim_amd
    from maxsim_amd import training

    for name in ("embed_tokens", "grad_norm", "clip_factor", "clip_grad_norm"):
        assert getattr(maxsim, name) is getattr(maxsim_amd, name) is getattr(training, name)
        assert name not in maxsim_amd.__all__  # which stays the reference's list


def test_host_tensors_are_refused():
    import torch

    import maxsim_amd

    table, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: maxsim_amd.embed_tokens(table, ids), lambda: maxsim_amd.grad_norm([table]),
                 lambda: maxsim_amd.clip_grad_norm(table, 1.0),
                 lambda: maxsim_amd.clip_factor([table], 1.0)):
        with pytest.raises(RuntimeError, match="HIP"):
            call()
    for padding in (4, -5):
        with pytest.raises((RuntimeError, ValueError)):
            maxsim_amd.embed_tokens(table, ids, padding_idx=padding)
    assert float(maxsim_amd.grad_norm([])) == 0.0
    for value in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            maxsim_amd.AdamW([torch.nn.Parameter(table)], max_norm=value)
