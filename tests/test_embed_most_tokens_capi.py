"""The C ABI of the embedding table's gradient for the most tokens that it is
documented to take (CPU only: a child process that sees no GPU)."""

from __future__ import annotations

import ctypes
import os

import pytest

from .test_embed_no_tokens_capi import BF16, F16, F32, INVALID, LIB, UNSUPPORTED, run_without_a_gpu

MOST = 2 ** 31 - 1


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="the pointers are made up: needs a machine without a GPU")
@pytest.mark.parametrize("types,dim", [((F32, F32), 1), ((F16, F16), 1), ((F32, BF16), 64), ((F32, F32), 128)],
                         ids=str)
@pytest.mark.parametrize("vocab", [1, 1000003, MOST])
def test_the_most_tokens_are_not_refused(types, dim, vocab):
    size = ctypes.CDLL(str(LIB)).maxsim_amd_embed_backward_workspace_size
    size.restype = ctypes.c_size_t
    size.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64]
    need = size(types[1], MOST, vocab, dim)
    assert need > 16 * MOST
    status = run_without_a_gpu(*types, MOST, vocab, dim, need)
    if vocab * dim * 4 > 2 ** 39:  # a table of a TB (no GPU holds it) has more rows to clear than a launch takes
        assert status == UNSUPPORTED
    else:
        assert status not in (INVALID, UNSUPPORTED), status
