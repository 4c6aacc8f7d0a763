"""What the run-of-tokens operators refuse, on the host: no call here reaches a kernel.
Every case is a valid call (refused last, for its CPU tensors) with one thing wrong."""

import ctypes as C

import pytest
import torch

from hackathon_b200 import _lib
from hackathon_b200 import kernels as K

F8 = torch.float8_e4m3fn


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def batch(lengths, slots=None, **kw):
    return K.SequenceBatch(lengths, slots, device="cpu", **kw)


def norm_args(**kw):
    return {**dict(x=z(3, 256), weight=z(256), residual=z(3, 256)), **kw}


def linear_args(**kw):
    return {**dict(q=z(3, 256, dtype=F8), scale=z(3, 2), wq=z(130, 256, dtype=F8), wscale=z(2, 2), bias=z(130)), **kw}


def conv_args(**kw):
    return {**dict(window=z(2, 8, 3), x=z(5, 8), weight=z(8, 4), bias=z(8), seqs=batch([2, 3])), **kw}


def scan_args(**kw):
    return {**dict(ssm=z(2, 4, 8, 16), x=z(5, 4, 8), b=z(5, 16), c=z(5, 16), dt=z(5, 4), a=z(4), seqs=batch([2, 3]), d=z(4),
                   z=z(5, 4, 8)), **kw}


CASES = [
    (K.rms_norm_fp8, norm_args, {}, "no CPU path"),
    (K.rms_norm_fp8, norm_args, dict(x=z(256)), "rows, cols"),
    (K.rms_norm_fp8, norm_args, dict(x=z(3, 0)), "rows, cols"),
    (K.rms_norm_fp8, norm_args, dict(x=z(3, 256, dtype=torch.float64)), "x must be float32"),
    (K.rms_norm_fp8, norm_args, dict(residual=z(2, 256)), "residual must be"),
    (K.rms_norm_fp8, norm_args, dict(residual=z(3, 256, dtype=torch.bfloat16)), "residual must be"),
    (K.rms_norm_fp8, norm_args, dict(weight=z(255)), "weight must be"),
    (K.rms_norm_fp8, norm_args, dict(weight=z(256, dtype=torch.bfloat16)), "weight must be"),
    (K.fp8_linear, linear_args, {}, "no CPU path"),
    (K.fp8_linear, linear_args, dict(q=z(3, 256)), "float8_e4m3fn"),
    (K.fp8_linear, linear_args, dict(wq=z(130, 128, dtype=F8)), "expected"),
    (K.fp8_linear, linear_args, dict(scale=z(3, 1)), "scale must be"),
    (K.fp8_linear, linear_args, dict(scale=z(3, 2, dtype=torch.float64)), "scale must be"),
    (K.fp8_linear, linear_args, dict(wscale=z(1, 2)), "wscale must be"),
    (K.fp8_linear, linear_args, dict(bias=z(129)), "bias must be"),
    (K.fp8_linear, linear_args, dict(out_dtype=torch.float64), "out_dtype"),
    (K.causal_conv, conv_args, {}, "no CPU path"),
    (K.causal_conv, conv_args, dict(window=z(2, 8, 4), weight=z(8, 5)), "window must be"),
    (K.causal_conv, conv_args, dict(window=z(2, 8, 3, dtype=torch.bfloat16)), "window must be fp32"),
    (K.causal_conv, conv_args, dict(window=z(2, 3, 8).transpose(1, 2)), "contiguous"),
    (K.causal_conv, conv_args, dict(x=z(5, 9)), "x must be"),
    (K.causal_conv, conv_args, dict(weight=z(8, 3)), "weight must be"),
    (K.causal_conv, conv_args, dict(bias=z(9)), "bias must be"),
    (K.causal_conv, conv_args, dict(x=z(4, 8)), "5 tokens"),
    (K.causal_conv, conv_args, dict(seqs=batch([2, 3], [0, 2])), "need 3 state rows"),
    (K.causal_conv, conv_args, dict(seqs=None), "without a SequenceBatch"),
    (K.mamba2_scan, scan_args, {}, "no CPU path"),
    (K.mamba2_scan, scan_args, dict(ssm=z(2, 4, 8, 16, dtype=torch.bfloat16)), "ssm must be fp32"),
    (K.mamba2_scan, scan_args, dict(ssm=z(2, 4, 16, 8).transpose(2, 3)), "contiguous"),
    (K.mamba2_scan, scan_args, dict(ssm=z(2, 4, 8, 257), b=z(5, 257), c=z(5, 257)), "at most 256"),
    (K.mamba2_scan, scan_args, dict(x=z(5, 4, 9)), "x must be"),
    (K.mamba2_scan, scan_args, dict(b=z(5, 16, dtype=torch.bfloat16)), "b must be"),
    (K.mamba2_scan, scan_args, dict(c=z(5, 15)), "c must be"),
    (K.mamba2_scan, scan_args, dict(z=z(4, 4, 8)), "z must be"),
    (K.mamba2_scan, scan_args, dict(dt=z(5, 4, dtype=torch.bfloat16)), "dt must be"),
    (K.mamba2_scan, scan_args, dict(dt=z(5, 3)), "dt must be"),
    (K.mamba2_scan, scan_args, dict(a=z(3)), "a must be"),
    (K.mamba2_scan, scan_args, dict(a=None), "a must be"),
    (K.mamba2_scan, scan_args, dict(d=z(5)), "d must be"),
    (K.mamba2_scan, scan_args, dict(seqs=batch([2, 4])), "6 tokens"),
    (K.mamba2_scan, scan_args, dict(seqs=None), "without a SequenceBatch"),
]


@pytest.mark.parametrize("fn,base,wrong,match", CASES, ids=[f"{c[0].__name__}-{i}" for i, c in enumerate(CASES)])
def test_refused(fn, base, wrong, match):
    with pytest.raises(AssertionError, match=match):
        fn(**base(**wrong))


def test_quantisers_refuse():
    with pytest.raises(AssertionError, match="rows, cols"):
        K.quantize_fp8(z(3))
    with pytest.raises(AssertionError, match="float32"):
        K.quantize_fp8(z(3, 4, dtype=torch.int32))
    with pytest.raises(AssertionError, match="out, in"):
        K.quantize_fp8_weight(z(0, 4))
    for fn in (K.quantize_fp8, K.quantize_fp8_weight):
        with pytest.raises(AssertionError, match="no CPU path"):
            fn(z(3, 4))


@pytest.mark.parametrize("lengths,slots,kw,match", [
    ([1, -1], None, {}, "negative"),
    ([1, 2], [3, 3], {}, "distinct"),
    ([1, 2], [0], {}, "1 slots for 2"),
    ([1, 2], [0, -1], {}, "negative"),
    ([1, 2], [0, 5], dict(state_rows=5), "row 5 of 5"),
    ([1, 2, 3], None, dict(state_rows=2), "row 2 of 2"),
    ([2 ** 30, 2 ** 30], None, {}, "2\\^31"),
])
def test_sequence_batch_refuses(lengths, slots, kw, match):
    with pytest.raises(AssertionError, match=match):
        batch(lengths, slots, **kw)


def test_sequence_batch_layout():
    b = batch([3, 0, 2], [4, 0, 1])
    assert (b.tokens, b.state_rows, len(b)) == (5, 5, 3)
    assert b._arrays.tolist() == [0, 3, 3, 5, 0, 2, 1, 4, 0, 1]
    assert (b._c.seqs, b._c.tokens, b._c.longest) == (3, 5, 3)
    assert (b._c.order - b._c.starts, b._c.slots - b._c.starts) == (16, 28)
    steps = batch([1, 1], [1, 0])  # one token a sequence: no starts
    assert steps._c.starts is None and steps._arrays.tolist() == [1, 0]
    assert batch([]).tokens == 0


def call(name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    return rc, _lib.lib().b2e_last_error().decode()


def test_c_abi_refuses_before_any_device_call():
    """Sizes, types, strides and plans are checked on the host; P stands for a device pointer nobody reads."""
    P = 1 << 20
    for args, match in [
        ((P, 9, 64, None, 0, 0, None, 1e-5, 2, 64, P, 64, P, None, None, None), "unknown dtype"),
        ((P, 0, 63, None, 0, 0, None, 1e-5, 2, 64, P, 64, P, None, None, None), "row stride"),
        ((P, 1, 64, P, 2, 64, None, 1e-5, 2, 64, P, 64, P, P, None, None), "residual"),
        ((P, 1, 64, None, 0, 0, None, 1e-5, 2, 64, P, 64, P, P, None, None), "total needs"),
        ((None, 0, 64, None, 0, 0, None, 1e-5, 2, 64, P, 64, P, None, None, None), "null"),
        ((P, 0, 64, None, 0, 0, None, 1e-5, -1, 64, P, 64, P, None, None, None), "bad sizes"),
    ]:
        rc, msg = call("b2e_rms_norm_fp8", *args)
        assert rc == -1 and match in msg
    for args, match in [
        ((P, 64, P, 2, 64, P, 64, P, 8, None, 2, P, 0, 8, None), "activation"),
        ((P, 72, P, 2, 64, P, 64, P, 8, None, 0, P, 0, 8, None), "16-byte"),
        ((P + 8, 64, P, 2, 64, P, 64, P, 8, None, 0, P, 0, 8, None), "16-byte"),
        ((P, 64, P, 2, 64, P, 48, P, 8, None, 0, P, 0, 8, None), "row stride"),
        ((P, 64, P, 2, 64, P, 64, P, 8, None, 0, P, 7, 8, None), "unknown dtype"),
        ((P, 64, P, 2, 0, P, 64, P, 8, None, 0, P, 0, 8, None), "bad sizes"),
    ]:
        rc, msg = call("b2e_fp8_linear", *args)
        assert rc == -1 and match in msg
    plan = lambda starts=P, slots=None, seqs=2, tokens=5, rows=2, longest=3: C.byref(  # noqa: E731
        _lib.SequencesC(starts, slots, None, seqs, tokens, rows, longest))
    for p, rows, taps, match in [
        (plan(tokens=6), 5, 4, "more tokens"), (plan(seqs=3), 5, 4, "more sequences"), (plan(starts=None), 5, 4, "without starts"),
        (plan(seqs=-1), 5, 4, "negative"), (plan(longest=6), 5, 4, "longest"), (plan(), 5, 5, "2 to 4 taps"),
    ]:
        rc, msg = call("b2e_causal_conv", p, P, P, 0, 8, rows, 8, P, None, taps, 0, P, 8, None)
        assert rc == -1 and match in msg
    def scan(p=None, work=0, at=None, **kw):
        a = dict(ssm=P, x=P, b=P, c=P, dt=P, a=P, d=None, z=None, y=P, ldx=32, ldb=16, ldc=16, lddt=4, ldz=0, ldy=32, rows=5,
                 heads=4, size=8, state=16, dtype=0, softplus=1)
        return call("b2e_mamba2_scan", p or plan(), C.byref(_lib.ScanArgsC(**{**a, **kw})), at, work, None)
    for kw, match in [
        (dict(state=257), "1..256"), (dict(heads=0), "positive"), (dict(dtype=3), "unknown dtype"), (dict(x=None), "null"),
        (dict(ldx=31), "row stride"), (dict(ssm=P + 4), "16-byte"), (dict(rows=4), "more tokens"),
        (dict(p=plan(tokens=5000, longest=5000, seqs=1), rows=5000), "workspace"),
        (dict(p=plan(tokens=5000, longest=5000, seqs=1), rows=5000, at=P + 8, work=1 << 40), "workspace starts"),
    ]:
        rc, msg = scan(**kw)
        assert rc == -1 and match in msg, (kw, rc, msg)
    rc, msg = call("b2e_mamba2_scan", plan(), None, None, 0, None)
    assert rc == -1 and "null" in msg
    assert call("b2e_seqops_device_error", None)[0] == -1


def test_scan_workspace_follows_the_plan():
    """Whole sequences where they fill the device, segments of a multiple of 128 tokens where they do not."""
    args = _lib.ScanArgsC(rows=1 << 20, heads=8, size=64, state=128, ldx=512, ldy=512)
    def need(seqs, tokens, longest):
        out = C.c_int64(-1)
        plan = _lib.SequencesC(1 << 20, None, None, seqs, tokens, seqs, longest)
        _lib.check(_lib.lib().b2e_mamba2_scan_workspace(C.byref(plan), C.byref(args), C.byref(out)))
        return out.value
    assert need(1, 100, 100) == 0 and need(2000, 200000, 1000) == 0
    one = need(1, 16384, 16384)
    assert one > 0 and one % 256 == 0
    assert _lib.lib().b2e_mamba2_scan_workspace(None, C.byref(args), None) == -1
