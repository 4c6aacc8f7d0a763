"""Limits of the run-of-tokens operators that are decided on the host."""

import ctypes as C

import pytest

from hackathon_b200 import _lib


def workspace(lengths, heads, size, state, dtype):
    args = _lib.ScanArgsC(rows=sum(lengths), heads=heads, size=size, state=state, ldx=heads * size, ldy=heads * size, dtype=dtype)
    plan = _lib.SequencesC(1 << 20, None, None, len(lengths), sum(lengths), len(lengths), max(lengths))
    out = C.c_int64(-1)
    _lib.check(_lib.lib().b2e_mamba2_scan_workspace(C.byref(plan), C.byref(args), C.byref(out)))
    return out.value


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("long,short,heads", [(2000, 2000, 64), (3000, 4000, 8), (100000, 1, 8), (5000, 30000, 1)])
def test_scan_workspace_goes_by_split_tokens(dtype, long, short, heads):
    """One long sequence among many single tokens: at most two states a segment of 128 tokens, whatever
    the number of sequences."""
    need = workspace([long] + [1] * short, heads, 64, 128, dtype)
    places = 2 * ((long + short) // 128)
    assert need <= places * heads * (64 * 128 + 1) * 4 + 256
    alone = workspace([long], heads, 64, 128, dtype)
    assert alone <= (long // 128 + 1) * heads * (64 * 128 + 1) * 4 + 256
