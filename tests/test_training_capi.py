"""The C ABI of the operators around the scores (CPU only: exports and argument
checks, nothing is launched)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LIB = ROOT / "maxsim_amd" / "libmaxsim_amd.so"
OK, INVALID, UNSUPPORTED = 0, 1, 2
F32, F16, BF16 = 0, 1, 2
I64, P, F, D = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_double
ONE = P(16)


class Tensor(ctypes.Structure):
    _fields_ = [("param", P), ("grad", P), ("exp_avg", P), ("exp_avg_sq", P), ("scales", P),
                ("master", P), ("numel", I64), ("position", ctypes.c_uint64)]


@pytest.fixture(scope="module")
def lib():
    handle = ctypes.CDLL(str(LIB))
    handle.maxsim_amd_last_error.restype = ctypes.c_char_p
    return handle


def test_every_declared_symbol_is_exported(lib):
    text = (ROOT / "include" / "maxsim_amd_training.h").read_text()
    names = re.findall(r"^\s*(?:int|size_t)\s+(maxsim_amd_\w+)\s*\(", text, re.M)
    assert len(set(names)) == 8
    for name in names:
        assert hasattr(lib, name), name


def _norm(lib, dtype=BF16, wdtype=BF16, x=ONE, rows=4, dim=64, stride=64, eps=1e-5, y=ONE, mean=None,
          rstd=None):
    fn = lib.maxsim_amd_layer_norm_forward
    fn.argtypes = [ctypes.c_int, ctypes.c_int, P, I64, I64, I64, P, P, F, P, P, P, P]
    return fn(dtype, wdtype, x, rows, dim, stride, ONE, ONE, eps, y, mean, rstd, None)


def test_layer_norm_forward_refusals(lib):
    assert _norm(lib, rows=0, x=None, y=None) == OK
    for kw, text in ((dict(dtype=5), b"dtype"), (dict(wdtype=F16), b"weight_dtype"),
                     (dict(rows=-1), b"negative"), (dict(dim=0), b"dim"),
                     (dict(stride=-1), b"stride"), (dict(eps=-1.0), b"eps"),
                     (dict(eps=float("nan")), b"eps"), (dict(x=None), b"null"),
                     (dict(y=None), b"null"), (dict(mean=ONE), b"null")):
        assert _norm(lib, **kw) == INVALID, kw
        assert text in lib.maxsim_amd_last_error()
    assert _norm(lib, dim=16385) == UNSUPPORTED


def test_layer_norm_backward_refusals(lib):
    size = lib.maxsim_amd_layer_norm_backward_workspace_size
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_int, I64, I64]
    assert size(BF16, 0, 64) == 0 and size(BF16, 5, 0) == 0 and size(BF16, 5, 16385) == 0
    assert size(BF16, 1, 64) == 2 * 64 * 4
    assert size(F32, 10 ** 9, 768) <= 1024 * 2 * 768 * 4
    fn = lib.maxsim_amd_layer_norm_backward
    fn.argtypes = [ctypes.c_int, ctypes.c_int, P, I64, P, I64, P, P, P, I64, I64, P, P, P, P,
                   ctypes.c_size_t, P]

    def call(dy=ONE, rows=4, dim=64, dx=ONE, dw=ONE, ws=ONE, ws_bytes=1 << 20, stride=64):
        return fn(BF16, BF16, dy, stride, ONE, stride, ONE, ONE, ONE, rows, dim, dx, dw, dw, ws,
                  ws_bytes, None)

    assert call(dx=None, dw=None) == OK  # nothing is wanted
    for kw, text in ((dict(dy=None), b"null"), (dict(ws=None), b"workspace"),
                     (dict(ws_bytes=511), b"workspace"), (dict(rows=-1), b"negative"),
                     (dict(stride=-1), b"stride"), (dict(dim=0), b"dim")):
        assert call(**kw) == INVALID, kw
        assert text in lib.maxsim_amd_last_error()


def test_unit_rows_refusals(lib):
    fn = lib.maxsim_amd_unit_rows_forward
    fn.argtypes = [ctypes.c_int, P, I64, I64, I64, I64, I64, P, ctypes.c_int, P, I64, F, P, P]

    def call(dtype=F16, x=ONE, n=2, length=3, dim=64, stride=64, lengths=ONE, offsets=None, rows=0,
             eps=1e-12, y=ONE):
        return fn(dtype, x, n, length, dim, stride, stride, lengths, 0, offsets, rows, eps, y, None)

    assert call(n=0, x=None, y=None) == OK and call(length=0, x=None, y=None) == OK
    assert call(offsets=ONE, rows=0, y=None) == OK
    for kw, text in ((dict(dtype=9), b"dtype"), (dict(n=-1), b"negative"),
                     (dict(length=-1), b"negative"), (dict(dim=0), b"dim"),
                     (dict(stride=-4), b"stride"), (dict(eps=0.0), b"eps"),
                     (dict(eps=float("nan")), b"eps"), (dict(x=None), b"null"),
                     (dict(y=None), b"null"), (dict(lengths=None, offsets=ONE, rows=5), b"lengths"),
                     (dict(offsets=ONE, rows=-1), b"negative")):
        assert call(**kw) == INVALID, kw
        assert text in lib.maxsim_amd_last_error()
    assert call(dim=16385) == UNSUPPORTED and call(length=2 ** 31) == UNSUPPORTED
    back = lib.maxsim_amd_unit_rows_backward
    back.argtypes = [ctypes.c_int, P, I64, I64, P, I64, I64, I64, I64, I64, P, ctypes.c_int, P, I64,
                     F, P, P]
    assert back(F16, None, 64, 64, ONE, 2, 3, 64, 64, 64, ONE, 0, None, 0, 1e-12, ONE,
                None) == INVALID
    assert back(F16, ONE, -1, 64, ONE, 2, 3, 64, 64, 64, ONE, 0, None, 0, 1e-12, ONE,
                None) == INVALID
    scan = lib.maxsim_amd_length_offsets
    scan.argtypes = [P, ctypes.c_int, I64, I64, P, P, P, P]
    assert scan(ONE, 0, -1, 5, ONE, ONE, None, None) == INVALID
    assert scan(None, 0, 4, 5, ONE, ONE, None, None) == INVALID
    assert scan(ONE, 0, 1 << 16, 1 << 15, ONE, ONE, None, None) == UNSUPPORTED  # offsets past int32


def test_adamw_refusals(lib):
    fn = lib.maxsim_amd_adamw_step
    fn.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.POINTER(Tensor), I64, D, P, D, D,
                   D, D, I64, P, ctypes.c_uint64, P]

    def call(dtype=BF16, gdtype=BF16, bits=32, tensors=(), lr=1e-3, b1=0.9, b2=0.999, eps=1e-8,
             decay=0.0, step=1, step_at=None):
        arr = (Tensor * max(1, len(tensors)))(*tensors)
        return fn(dtype, gdtype, bits, arr, len(tensors), lr, None, b1, b2, eps, decay, step, step_at,
                  0, None)

    def tensor(numel=8, master=None, scales=None, grad=16):
        return Tensor(16, grad, 16, 16, scales, master, numel, 0)

    assert call() == OK and call(tensors=[tensor(0, grad=None)]) == OK
    assert call(step=0, step_at=ONE) == OK  # the device's step counts
    for kw, text in ((dict(dtype=7), b"dtype"), (dict(gdtype=F16), b"grad_dtype"),
                     (dict(bits=16), b"state_bits"), (dict(b1=1.0), b"betas"),
                     (dict(b2=-0.1), b"betas"), (dict(eps=-1.0), b"eps"),
                     (dict(lr=float("nan")), b"lr"), (dict(decay=-1.0), b"weight_decay"),
                     (dict(step=0), b"step"), (dict(tensors=[tensor(-1)]), b"negative"),
                     (dict(tensors=[tensor(grad=None)]), b"null"),
                     (dict(tensors=[tensor()], bits=8), b"null"),
                     (dict(tensors=[tensor(), tensor(master=16)]), b"master"),
                     (dict(dtype=F32, gdtype=F32, tensors=[tensor(master=16)]), b"master")):
        assert call(**kw) == INVALID, kw
        assert text in lib.maxsim_amd_last_error()
    assert call(tensors=[tensor(2 ** 50)]) == UNSUPPORTED
    values = lib.maxsim_amd_adamw_state_values
    values.argtypes = [P, P, P, I64, P, P, P]
    assert values(ONE, ONE, ONE, -1, ONE, ONE, None) == INVALID
    assert values(ONE, None, ONE, 4, ONE, ONE, None) == INVALID
    assert values(None, None, None, 0, None, None, None) == OK


def test_unit_rows_refuse_an_eps_below_the_normal_numbers(lib):
    # its reciprocal is past fp32's largest number
    fn = lib.maxsim_amd_unit_rows_forward
    fn.argtypes = [ctypes.c_int, P, I64, I64, I64, I64, I64, P, ctypes.c_int, P, I64, F, P, P]
    for eps in (1e-39, 1e-45, -1.0):
        assert fn(F32, ONE, 2, 3, 64, 192, 64, None, 0, None, 0, eps, ONE, None) == INVALID
        assert b"eps" in lib.maxsim_amd_last_error()
    assert fn(F32, ONE, 0, 3, 64, 192, 64, None, 0, None, 0, 2.0 ** -126, ONE, None) == OK
