"""The tree decode's C entry points at sizes that its 32-bit counts do not hold: refused on the host.  Each call runs in a
process of its own, so that one that ends its process is seen."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys
sys.path.insert(0, {root!r})
from co_alibi_attn import _native
lib, P = _native.lib(), 4096
dtype, B, Hq, Hkv, T, L, D, page = {shape!r}
print(lib.co_alibi_decode_tree_workspace_bytes(dtype, B, Hq, Hkv, T, L, D))
table, blocks, pages = (P, 1 << 10, 1) if page else (None, 0, 0)
print(lib.co_alibi_decode_tree(dtype, P, P, P, P, P, None, P, P, None, 0, table, blocks, pages, page or 1 << 30, P, None, P,
                               1 << 60, B, Hq, Hkv, T, L, D, 0.125, None))
print(lib.co_alibi_last_error().decode())
"""


@pytest.mark.parametrize("shape,code,message", [
    # (dtype, B, Hq, Hkv, T, L, D, page): the rows of a kv head would be 2^32, 2^31 and -2^31 + 64 ...
    ((1, 1, 1 << 27, 1, 32, 100, 64, 0), 1, "problem too large for one launch"),
    ((1, 1, 1 << 26, 1, 32, 100, 64, 0), 1, "problem too large for one launch"),
    ((1, 1, (1 << 25) + 1, 1, 64, 100, 64, 0), 1, "problem too large for one launch"),
    ((1, 1, 65536, 1, 65536, 100, 64, 0), 2, "at most 64 new tokens per sequence, got 65536"),
    ((1, 1, 8, 8, 65, 100, 64, 0), 2, "at most 64 new tokens per sequence, got 65"),
    # ... and the chunks of all sequences 2^31, through a table whose sequences share one page of 2^20 rows.
    ((2, 128, 1, 1, 1, 1 << 30, 16, 1 << 20), 1, "problem too large for one launch"),
    ((1, 1, 6, 4, 3, 100, 64, 0), 1, "heads_q must be a multiple of heads_kv"),
    ((1, 1, 1, 1, 1, (1 << 31) - 1, 64, 0), 1, "problem too large for one launch"),
], ids=str)
def test_uncountable_shapes_are_refused(shape, code, message):
    done = subprocess.run([sys.executable, "-c", CODE.format(root=ROOT, shape=shape)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    size, got, text = done.stdout.strip().split("\n")
    assert got == str(code) and message in text
    # (A size that only the launch's grid refuses still has a workspace.)
    assert size == "0" or shape[5] == (1 << 31) - 1
