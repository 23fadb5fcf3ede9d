"""The C entries of masked attention refuse sizes that are none, in a process of its own: what they compute from them must not end it."""
import subprocess
import sys

import pytest

from mlperf_training_b200.ops import _lib
from mlperf_training_b200.ops import functional as F

CALLS = """
import ctypes
from mlperf_training_b200.ops import _lib
lib = _lib.load()
for B, Sq, Skv, Hq, Hkv, D in [(1, 4, 4, 0, 1, 64), (1, 4, 4, 0, 0, 64), (1, 4, 4, 2, 0, 64), (0, 4, 4, 2, 1, 64), (1, 0, 4, 2, 1, 64), (1, 4, 0, 2, 1, 64),
                               (1, 4, 4, -2, 1, 64), (1, 4, 4, -2, -1, 64), (1, 4, 4, 1, 2, 64), (-1, 4, 4, 2, 1, 64), (1, 8, 4, 2, 1, 64)]:
    print(lib.b200_attn_masked_fwd_workspace(B, Sq, Skv, Hq, D), lib.b200_attn_masked_rows_workspace(B, Sq, Skv, Hq, Hkv, D),
          lib.b200_attn_masked_bwd_workspace(B, Sq, Skv, Hq, Hkv, D), lib.b200_attn_masked_few_rows(B, Sq, Hq, Hkv))
    sizes, tail = [B, Sq, Skv, Hq, Hkv, D], [ctypes.c_float(1.0), ctypes.c_float(0.0), None, ctypes.c_longlong(0), None]
    pitch = [ctypes.c_longlong(64)] * 10
    assert lib.b200_attn_masked_fwd(*[None] * 9, *sizes, *pitch[:6], *tail) != 0
    assert lib.b200_attn_masked_rows(*[None] * 8, *sizes, *pitch[:6], *tail) != 0
    assert lib.b200_attn_masked_bwd(*[None] * 13, *sizes, *pitch, *tail) != 0
print("done")
"""


def test_sequences_that_32_bits_do_not_count():
    with pytest.raises(ValueError):
        F.attention_mask(2 ** 32 + 1, 1, 1)


@pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="the kernel library is not built")
def test_sizes_that_are_none():
    r = subprocess.run([sys.executable, "-c", CALLS], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split()[-1] == "done", (r.returncode, r.stdout[-500:], r.stderr[-2000:])
    for line in r.stdout.split("\n")[:-2]:
        # (the forward's workspace does not know of key heads, nor whether rows are few of the keys: the others see all that is wrong)
        assert line.split()[1:3] == ["0", "0"]
