"""The C ABI of the embedding table's gradient where there are no tokens (CPU
only: a child process that sees no GPU, so that a crash on the host is its own
and nothing is launched)."""

from __future__ import annotations

import ctypes
import os
import subprocess
import sys
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parent.parent / "maxsim_amd" / "libmaxsim_amd.so"
INVALID, UNSUPPORTED = 1, 2
F32, F16, BF16 = 0, 1, 2

# arguments: weight type, type, tokens, vocab, dim, bytes of workspace; prints the status
CALL = f"""
import ctypes, sys
lib = ctypes.CDLL({str(LIB)!r})
I64, P, F, SIZE = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t
fn = lib.maxsim_amd_embed_backward
fn.argtypes = [ctypes.c_int, ctypes.c_int, P, I64, P, I64, I64, I64, F, P, P, SIZE, P]
wt, t, tokens, vocab, dim, size = map(int, sys.argv[1:])
none = None if tokens == 0 else P(16)
print(fn(wt, t, none, dim, none, tokens, vocab, dim, 1.0, P(16), P(16) if size else None, size, None))
"""


def run_without_a_gpu(*args):
    """Status of maxsim_amd_embed_backward; the launch itself fails."""
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="")
    done = subprocess.run([sys.executable, "-c", CALL, *map(str, args)], env=env, text=True,
                          capture_output=True, timeout=100)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])  # negative: a signal
    return int(done.stdout)


# on both sides of the widths that the one launch takes, and of its numbers of rows
@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="the pointers are made up: needs a machine without a GPU")
@pytest.mark.parametrize("types,dim", [((F32, F32), 1024), ((F32, F32), 1025), ((F32, F32), 16384),
                                       ((BF16, BF16), 2048), ((BF16, BF16), 2560), ((F16, F16), 2049),
                                       ((F32, BF16), 16384), ((F32, F16), 4096)], ids=str)
@pytest.mark.parametrize("vocab", [1, 100, 2 ** 29 + 1, 2 ** 31 - 1])
def test_no_tokens_end_with_a_status(types, dim, vocab):
    status = run_without_a_gpu(*types, 0, vocab, dim, 0)
    assert status not in (INVALID, UNSUPPORTED), status


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [8, 1024, 1025, 2048, 2049, 16384])
@pytest.mark.parametrize("vocab", [0, 1, 100, 2 ** 31 - 1])
def test_no_tokens_need_no_workspace(vocab, dim, dtype):
    size = ctypes.CDLL(str(LIB)).maxsim_amd_embed_backward_workspace_size
    size.restype = ctypes.c_size_t
    size.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64]
    assert size(dtype, 0, vocab, dim) == 0
