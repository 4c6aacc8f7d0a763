"""Limits of the run-of-tokens operators that are decided on the host."""

import ctypes as C

import numpy as np
import pytest
import torch

from hackathon_b200 import _lib
from hackathon_b200 import kernels as K


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


BIG = 2 ** 31  # one more than a 32-bit index can hold; views of one value, no memory


def many(*shape, dtype=torch.float32):
    return torch.zeros(*[min(n, 1) for n in shape], dtype=dtype).expand(*shape)


F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("call", [
    lambda n: K.rms_norm_fp8(many(n, 1)), lambda n: K.rms_norm_fp8(many(1, n)),
    lambda n: K.quantize_fp8(many(n, 1)), lambda n: K.quantize_fp8(many(1, n)),
    lambda n: K.quantize_fp8_weight(many(n, 1)), lambda n: K.quantize_fp8_weight(many(1, n)),
    lambda n: K.fp8_linear(many(n, 16, dtype=F8), many(n, 1), many(8, 16, dtype=F8), many(1, 1)),
    lambda n: K.fp8_linear(many(1, 16, dtype=F8), many(1, 1), many(n, 16, dtype=F8), many(-(-n // 128), 1)),
    lambda n: K.fp8_linear(many(1, n, dtype=F8), many(1, -(-n // 128)), many(1, n, dtype=F8), many(1, -(-n // 128))),
    lambda n: K.causal_conv(torch.zeros(2, 8, 3), many(n, 8), many(8, 4), None, K.SequenceBatch([1, 2], device="cpu")),
    lambda n: K.causal_conv(torch.zeros(0, n, 3), many(0, n), many(n, 4)),
    lambda n: K.mamba2_scan(torch.zeros(1, 1, 1, 1), many(n, 1, 1), many(n, 1), many(n, 1), many(n, 1), torch.zeros(1), K.SequenceBatch([2], device="cpu")),
    lambda n: K.SequenceBatch([n], device="cpu"),
    lambda n: K.SequenceBatch([1, n - 1], device="cpu"),
])
@pytest.mark.parametrize("n", [BIG, BIG - 1, BIG - 1023, 2 * BIG + 5])
def test_sizes_beyond_32_bit_indices_are_refused(call, n):
    with pytest.raises(AssertionError, match="2\\^31 - 1024"):
        call(n)


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 1023])
def test_c_abi_refuses_sizes_beyond_32_bit_indices(n):
    P, lib = 1 << 20, _lib.lib()
    plan = C.byref(_lib.SequencesC(P, None, None, 1, n, 1, n))
    scan = dict(ssm=P, x=P, b=P, c=P, dt=P, a=P, y=P, ldx=1, ldb=1, ldc=1, lddt=1, ldy=1, rows=n, heads=1, size=1, state=1)
    wide = dict(scan, rows=1, size=n, ldx=n, ldy=n)
    need = C.c_int64()
    for rc in [
        lambda: lib.b2e_rms_norm_fp8(P, 0, 1, None, 0, 0, None, 1e-5, n, 1, P, 16, P, None, None, None),
        lambda: lib.b2e_rms_norm_fp8(P, 0, n, None, 0, 0, None, 1e-5, 1, n, P, 1 << 31, P, None, None, None),
        lambda: lib.b2e_quantize_fp8(P, 0, 1, n, 1, P, 16, P, None),
        lambda: lib.b2e_quantize_fp8_weight(P, 0, n, 1, n, P, 1 << 31, P, None),
        lambda: lib.b2e_fp8_linear(P, 16, P, n, 16, P, 16, P, 1, None, 0, P, 0, 1, None),
        lambda: lib.b2e_fp8_linear(P, 16, P, 1, 16, P, 16, P, n, None, 0, P, 0, n, None),
        lambda: lib.b2e_causal_conv(plan, P, P, 0, 1, n, 1, P, None, 4, 0, P, 1, None),
        lambda: lib.b2e_causal_conv(None, P, P, 0, n, 1, n, P, None, 4, 0, P, n, None),
        lambda: lib.b2e_mamba2_scan_workspace(plan, C.byref(_lib.ScanArgsC(**scan)), C.byref(need)),
        lambda: lib.b2e_mamba2_scan(None, C.byref(_lib.ScanArgsC(**scan)), None, 0, None),
    ]:
        assert rc() == -1 and "2^31 - 1024" in lib.b2e_last_error().decode()
    assert lib.b2e_mamba2_scan(None, C.byref(_lib.ScanArgsC(**wide)), None, 0, None) == -1
    assert "too many channels" in lib.b2e_last_error().decode()
    many_seqs = C.byref(_lib.SequencesC(P, None, None, 2 ** 30 + 1, 5, 2 ** 31 - 1, 5))
    assert lib.b2e_causal_conv(many_seqs, P, P, 0, 1, 5, 1, P, None, 4, 0, P, 1, None) == -1
    assert "2^30" in lib.b2e_last_error().decode()


@pytest.mark.parametrize("kw", [
    dict(lengths=[2.9, 1]), dict(lengths=torch.tensor([2.0, 1.0])), dict(lengths=[2, 1], slots=[0, 1.5]),
    dict(lengths=[2, 1], state_rows=2.5), dict(lengths=["2"]),
])
def test_plan_refuses_what_is_not_a_whole_number(kw):
    with pytest.raises(AssertionError, match="must be integers"):
        K.SequenceBatch(**kw, device="cpu")


def test_plan_takes_integers_of_other_kinds():
    b = K.SequenceBatch(torch.tensor([3, 0, 2]), np.array([4, 0, 1]), state_rows=np.int64(5), device="cpu")
    assert (b.lengths, b.slots, b.state_rows, b.tokens) == ((3, 0, 2), (4, 0, 1), 5, 5)
