"""The run-of-tokens operators where their contract is easily broken: sequence ends inside a
chunk, plans and extents at their limits, values at the ends of their types."""

import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from hackathon_b200 import _lib as L
from hackathon_b200 import kernels as K
from tests import seqops_ref as R
from tests.test_gpu_seqops import DEV, PAIRS, TYPES, check_q, gen, ids, norm_ref, rnd, scan_inputs

pytestmark = pytest.mark.gpu


def need_memory(gib):
    if torch.cuda.mem_get_info(DEV)[0] < gib << 30:
        pytest.skip(f"needs {gib} GB of device memory")


def scan(inp, seqs, **kw):
    return K.mamba2_scan(inp["ssm"], inp["x"], inp["b"], inp["c"], inp["dt"], inp["a"], seqs, d=inp["d"], z=inp["z"], **kw)


def against_recurrence(inp, before, y, lengths, pairs):
    """y and the states of sequences in rows 0, 1, ... against the recurrence in 64 bits."""
    want, ssm, ymag, smag = R.scan(before, inp["x"], inp["b"], inp["c"], inp["dt"], inp["a"], lengths, range(len(lengths)), inp["d"], inp["z"])
    steps = max(lengths) + 1
    R.close(y, want, R.scan_tol(want, ymag, steps, y.dtype, pairs) + 4 * 2.0 ** -22 * want.abs(), "y")
    R.close(inp["ssm"], ssm, R.scan_tol(ssm, smag, steps, torch.float32), "ssm")


# ------------------------------------------------- ends inside a chunk


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("h,n,gate", [(8, 128, True), (7, 64, False)])
def test_scan_ends_inside_a_chunk(dt, h, n, gate):
    """Sequences that end in the second and third chunk of 128 tokens, more of them than run at once, each
    followed by one whose values are all NaN: bit for bit what they are without those neighbours, every
    time, and the recurrence's values."""
    lengths = [130, 257, 300, 383, 129, 255, 258, 200] * 8
    total, p = sum(lengths), 64
    clean = scan_inputs(50, len(lengths), total, h, p, n, dt, gate)
    before = clean["ssm"].clone()
    y = scan(clean, K.SequenceBatch(lengths, device=DEV))

    names = [k for k in ("x", "b", "c", "dt", "z") if clean[k] is not None]
    wide = {k: torch.full((2 * total, *clean[k].shape[1:]), float("nan"), dtype=clean[k].dtype, device=DEV) for k in names}
    at = []  # rows of the clean tokens between the others
    for s, e in R.seq_rows(lengths):
        at += range(2 * s, 2 * s + e - s)
    at = torch.tensor(at, device=DEV)
    for k in names:
        wide[k][at] = clean[k]
    both = K.SequenceBatch([n for n in lengths for _ in range(2)], device=DEV)
    slots = 2 * torch.arange(len(lengths), device=DEV)
    for _ in range(5):
        inp = {**clean, **wide, "ssm": torch.zeros(2 * len(lengths), h, p, n, device=DEV)}
        inp["ssm"][slots] = before
        got = scan(inp, both)
        assert torch.equal(got[at], y) and torch.equal(inp["ssm"][slots], clean["ssm"])
    assert K.device_error() == 0

    few = sum(lengths[:8])
    cut = {k: clean[k][:few] if k in names else clean[k] for k in clean}
    cut["ssm"] = clean["ssm"][:8]
    against_recurrence(cut, before[:8], y[:few], lengths[:8], PAIRS[dt])


# ------------------------------------------------- plans that leave their operands


def c_plan(starts, slots, order, tokens, state_rows, longest):
    """A plan as a C host makes it (it keeps the device arrays that it points into)."""
    arrays = [None if v is None else torch.tensor(v, dtype=torch.int32, device=DEV) for v in (starts, slots, order)]
    seqs = len(starts) - 1 if starts is not None else len(slots)
    plan = L.SequencesC(*[None if a is None else a.data_ptr() for a in arrays], seqs, tokens, state_rows, longest)
    plan.arrays = arrays
    return plan


def c_scan(inp, plan):
    _, h, p, n = inp["ssm"].shape
    y = torch.zeros_like(inp["x"])
    at = {k: inp[k].data_ptr() for k in ("ssm", "x", "b", "c", "dt", "a")}
    args = L.ScanArgsC(**at, y=y.data_ptr(), ldx=h * p, ldb=n, ldc=n, lddt=h, ldy=h * p, rows=len(y), heads=h, size=p, state=n,
                       dtype=K._TORCH_DTYPES[y.dtype], softplus=1)
    need = C.c_int64()
    L.check(L.lib().b2e_mamba2_scan_workspace(C.byref(plan), C.byref(args), C.byref(need)))
    work = torch.empty(max(need.value, 1), dtype=torch.uint8, device=DEV)
    L.check(L.lib().b2e_mamba2_scan(C.byref(plan), C.byref(args), work.data_ptr(), need.value, None))
    torch.cuda.synchronize()
    return y


def c_conv(window, x, w, plan):
    y = torch.zeros_like(x)
    L.check(L.lib().b2e_causal_conv(C.byref(plan), window.data_ptr(), x.data_ptr(), K._TORCH_DTYPES[x.dtype], x.shape[1], len(x),
                                    x.shape[1], w.data_ptr(), None, 4, 0, y.data_ptr(), x.shape[1], None))
    torch.cuda.synchronize()
    return y


def reported():
    """The error word says that a plan was out of range, once: reading clears it."""
    return K.device_error() == 1 and K.device_error() == 0


# three sequences: what is wrong, and those that are still stepped
BAD_PLANS = [
    (dict(starts=[0, 40, 70, 140]), [0, 1]), (dict(starts=[-8, 40, 70, 100]), [1, 2]), (dict(starts=[0, 40, 30, 100]), []),
    (dict(starts=[0, 40, 2 ** 31 - 1, 100]), [0]), (dict(starts=[0, -2 ** 31, 70, 100]), [2]),
    (dict(slots=[0, 3, 2]), [0, 2]), (dict(slots=[0, 1, -1]), [0, 1]), (dict(slots=[-2 ** 31, 2 ** 31 - 1, 2]), [2]),
    (dict(order=[2, 1, 3]), [1, 2]), (dict(order=[-1, 0, 1]), [0, 1]),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("wrong,good", BAD_PLANS, ids=[f"{next(iter(w))}-{i}" for i, (w, _) in enumerate(BAD_PLANS)])
def test_scan_and_conv_report_a_bad_plan(dt, wrong, good):
    """The sequence that leaves the operands or the table is not stepped, the others are, and the word says so."""
    assert K.device_error() == 0
    spec = dict(starts=[0, 40, 70, 100], slots=[0, 1, 2], order=[2, 0, 1])
    at = list(zip(spec["starts"], spec["starts"][1:]))
    inp = scan_inputs(60, 3, 100, 4, 64, 128, dt, False)
    before, same = inp["ssm"].clone(), {**inp, "ssm": inp["ssm"].clone()}
    want = c_scan(same, c_plan(**spec, tokens=100, state_rows=3, longest=40))
    assert K.device_error() == 0
    plan = c_plan(**{**spec, **wrong}, tokens=100, state_rows=3, longest=40)
    y = c_scan(inp, plan)
    assert reported()
    for i, (s, e) in enumerate(at):
        if i in good:
            assert torch.equal(y[s:e], want[s:e]) and torch.equal(inp["ssm"][i], same["ssm"][i])
        elif "starts" not in wrong:  # (a shared border moves a neighbour's rows too)
            assert not y[s:e].any() and torch.equal(inp["ssm"][i], before[i])

    if "order" in wrong:  # the convolution does not go by it
        return
    x, w = rnd(gen(61), 100, 64).to(dt), rnd(gen(62), 64, 4)
    win = rnd(gen(63), 3, 64, 3)
    before, clean = win.clone(), win.clone()
    want = c_conv(clean, x, w, c_plan(**spec, tokens=100, state_rows=3, longest=40))
    y = c_conv(win, x, w, plan)
    assert reported()
    for i, (s, e) in enumerate(at):
        if i in good:
            assert torch.equal(y[s:e], want[s:e]) and torch.equal(win[i], clean[i])
        elif "starts" not in wrong:
            assert not y[s:e].any() and torch.equal(win[i], before[i])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("wrong", [dict(starts=[0, 3000, 3060]), dict(starts=[-5, 2960, 3000]), dict(slots=[2, 1]), dict(starts=[0, 2960, 2000]),
                                   dict(starts=[0, 2960, -2 ** 31])])
def test_split_scan_reports_a_bad_plan(dt, wrong):
    """The same where sequences are split into segments."""
    inp = scan_inputs(64, 2, 3000, 2, 64, 128, dt, False)
    before = inp["ssm"].clone()
    plan = c_plan(**{**dict(starts=[0, 2960, 3000], slots=[0, 1], order=[0, 1]), **wrong}, tokens=3000, state_rows=2, longest=2960)
    assert K.device_error() == 0
    c_scan(inp, plan)
    assert reported()
    bad = 0 if "slots" in wrong or wrong["starts"][0] < 0 else 1
    assert torch.equal(inp["ssm"][bad], before[bad]) and not torch.equal(inp["ssm"][1 - bad], before[1 - bad])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("n", [128, 30])
def test_single_tokens_report_a_bad_plan(dt, n):
    inp = scan_inputs(65, 3, 3, 2, 64, n, dt, False)
    before = inp["ssm"].clone()
    plan = c_plan(None, [0, 3, 2], None, tokens=3, state_rows=3, longest=1)
    assert K.device_error() == 0
    y = c_scan(inp, plan)
    assert reported()
    assert torch.equal(inp["ssm"][1], before[1]) and not torch.equal(inp["ssm"][2], before[2]) and not y[1].any() and y[2].any()
    x, w, win = rnd(gen(66), 3, 64).to(dt), rnd(gen(67), 64, 4), rnd(gen(68), 3, 64, 3)
    before = win.clone()
    y = c_conv(win, x, w, plan)
    assert reported()
    assert torch.equal(win[1], before[1]) and not torch.equal(win[2], before[2]) and not y[1].any() and y[2].any()


# ------------------------------------------------- split sequences among others


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("lengths", [
    [1] * 600 + [1500] + [3] * 400 + [0] * 50 + [2300] + [2] * 300,  # far more sequences than segments
    [384, 384, 129, 300, 257, 1, 128, 640, 256, 1000],               # borders on segments' borders
    [127] + [1] * 129 + [384, 384, 640, 129, 257, 300] + [0, 1] * 40,
], ids=["many", "borders", "both"])
def test_split_sequences_among_others(dt, lengths):
    """Segments of several split sequences and short ones beside them: each finds its own states."""
    h = 2
    slots = torch.randperm(len(lengths), generator=torch.Generator().manual_seed(7)).tolist()
    inp = scan_inputs(70, len(lengths), sum(lengths), h, 64, 128, dt, True)
    before = inp["ssm"].clone()
    plan = K.SequenceBatch(lengths, slots, device=DEV)
    assert max(lengths) > 256  # where sequences of this batch are split
    y = scan(inp, plan)
    want, ssm, ymag, smag = R.scan(before, inp["x"], inp["b"], inp["c"], inp["dt"], inp["a"], lengths, slots, inp["d"], inp["z"])
    steps = max(lengths) + 1
    R.close(y, want, R.scan_tol(want, ymag, steps, dt, PAIRS[dt]) + 4 * 2.0 ** -22 * want.abs(), "y")
    R.close(inp["ssm"], ssm, R.scan_tol(ssm, smag, steps, torch.float32), "ssm")
    assert K.device_error() == 0


# ------------------------------------------------- values at the ends of their types


def normed_rows(x, eps, out):
    """The rows' norm and its 8 bits against 64 bits."""
    v, n, scale = norm_ref(x, None, None, eps)
    check_q(out.q, out.scale, n, scale)
    R.close(out.normed, n, R.rounding(n, x.dtype) + 2.0 ** -18 * n.abs(), "normed")


@pytest.mark.parametrize("dt", TYPES[:2], ids=ids[:2])
@pytest.mark.parametrize("cols", [256, 250, 1000, 1024, 4096, 8192, 9000])
def test_rms_norm_squares_beyond_float32(dt, cols):
    """Rows whose squares overflow or vanish, alone and beside ordinary ones."""
    x = rnd(gen(80), 9, cols)
    x *= torch.tensor([1.0, 1e19, 1e25, 2.0 ** 124 / 8, 1e-19, 1e-25, 1e-37, 1.0, 1.0], device=DEV)[:, None]
    x[7, 3] = 3e38   # one value's square overflows
    x[8, 5:] = 1e-30  # five values' squares outweigh the rest
    x = x.clamp(-3.3e38, 3.3e38).to(dt)
    for rows in (x, x[3:4].contiguous(), x[:0]):
        normed_rows(rows, 0.0, K.rms_norm_fp8(rows, eps=0.0, keep_norm=True))
        normed_rows(rows, 1e-5, K.rms_norm_fp8(rows, eps=1e-5, keep_norm=True))


def test_rms_norm_of_one_value_in_a_very_long_row():
    """Its square, 2^-72, vanishes in the mean of 2^29, and is far from it when scaled for that mean."""
    need_memory(16)
    x = torch.zeros(1, 2 ** 29, dtype=torch.bfloat16, device=DEV)
    x[0, 5] = 2.0 ** -36
    out = K.rms_norm_fp8(x, eps=0.0, keep_norm=True)
    want = 2.0 ** 14.5  # 2^-36 / sqrt(2^-72 / 2^29)
    assert abs(float(out.normed[0, 5]) / want - 1) < R.half(torch.bfloat16) + 2.0 ** -18
    assert abs(float(out.scale[0, 0]) * 448 / want - 1) < 2.0 ** -18 and float(out.q[0, 5]) == 448.0
    assert int(out.normed.count_nonzero()) == 1


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("cols", [256, 250, 1024, 4096])
def test_rms_norm_rows_that_are_not_finite(dt, cols):
    """A NaN makes its row NaN; an infinity its group, and the rest of its row zero; other rows keep their bits."""
    x = rnd(gen(81), 6, cols).to(dt)
    x[1, 5] = float("nan")
    x[2, 7], x[3, cols - 1], x[4, 0], x[4, 1] = float("inf"), float("-inf"), float("inf"), float("nan")
    out = K.rms_norm_fp8(x, keep_norm=True)
    q, groups = out.q.float(), -(-cols // 128)
    for row in (1, 4):
        assert q[row].isnan().all() and out.scale[row].isnan().all() and out.normed[row].isnan().all()
    for row, at in ((2, 7), (3, cols - 1)):
        g = at // 128
        assert q[row, g * 128:(g + 1) * 128].isnan().all() and out.scale[row, g].isnan()
        assert out.normed[row, at].isnan() and int(out.normed[row].isnan().sum()) == 1
        others = [i for i in range(groups) if i != g]
        rest = [i for i in range(cols) if i // 128 != g]
        assert not q[row, rest].any() and (out.scale[row, others] == 2.0 ** -100).all() and not out.normed[row, rest].any()
    clean = K.rms_norm_fp8(x[[0, 5]].contiguous(), keep_norm=True)
    assert torch.equal(q[[0, 5]], clean.q.float()) and torch.equal(out.scale[[0, 5]], clean.scale) and torch.equal(out.normed[[0, 5]], clean.normed)


# ------------------------------------------------- decay rates at the ends of float32


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("lengths", [[1, 1, 1], [300, 200, 40], [1500], [2, 1300, 700]], ids=["steps", "whole", "one split", "split"])
def test_scan_with_extreme_rates(dt, lengths):
    """Rates of minus infinity, of 1e30 and of zero: a state that is set anew with every token, or only added to."""
    inp = scan_inputs(90, len(lengths), sum(lengths), 5, 64, 128, dt, True)
    inp["a"] = torch.tensor([float("-inf"), -1e30, -3e38, -1.0, 0.0], device=DEV)
    before = inp["ssm"].clone()
    y = scan(inp, K.SequenceBatch(lengths, device=DEV))
    against_recurrence(inp, before, y, lengths, PAIRS[dt])


# ------------------------------------------------- offsets beyond 2^31 elements


ROWS, STRIDE = 40, 2 ** 26 + 128  # the last rows start beyond 2^31 elements


def far(base, like, at):
    """The rows of `like` in rows STRIDE elements apart."""
    flat = like.reshape(ROWS, -1)
    view = base.as_strided(flat.shape, (STRIDE, 1), at)
    view.copy_(flat)
    return view.unflatten(1, like.shape[1:])


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("lengths", [[ROWS], [1] * ROWS, [9, 0, 31]], ids=["whole", "steps", "two"])
def test_rows_far_apart(dt, lengths):
    """Row strides that put the last rows beyond 2^31 elements: the packed operands' bits."""
    need_memory(48)
    h, p, n = 4, 64, 128
    base = torch.empty(ROWS * STRIDE, dtype=dt, device=DEV)
    steps = base if dt == torch.float32 else torch.empty(ROWS * STRIDE, dtype=torch.float32, device=DEV)
    inp = scan_inputs(100, len(lengths), ROWS, h, p, n, dt, True)
    wide = {k: far(base, inp[k], 512 * i) for i, k in enumerate(("x", "b", "c", "z"))}
    wide["dt"] = far(steps, inp["dt"], 4096)
    wide = {**inp, **wide, "ssm": inp["ssm"].clone()}
    plan = K.SequenceBatch(lengths, device=DEV)
    assert torch.equal(scan(wide, plan), scan(inp, plan)) and torch.equal(wide["ssm"], inp["ssm"])

    x, flat = wide["x"].flatten(1), inp["x"].flatten(1)
    assert x.stride(0) == STRIDE
    for a, b in zip(K.rms_norm_fp8(x, residual=x), K.rms_norm_fp8(flat, residual=flat)):
        assert a is b is None or torch.equal(a.float(), b.float())
    for at in (x, x[:, 1:]):
        for a, b in zip(K.quantize_fp8(at) + K.quantize_fp8_weight(at), K.quantize_fp8(at.contiguous()) + K.quantize_fp8_weight(at.contiguous())):
            assert torch.equal(a.float(), b.float())
    w = rnd(gen(101), h * p, 4)
    win = rnd(gen(102), len(lengths), h * p, 3)
    other = win.clone()
    assert torch.equal(K.causal_conv(win, x, w, None, plan, silu=True), K.causal_conv(other, flat, w, None, plan, silu=True))
    assert torch.equal(win, other) and K.device_error() == 0


@pytest.mark.parametrize("m", [ROWS, 3])
def test_projection_rows_far_apart(m):
    need_memory(16)
    g = gen(103)
    q, scale = K.quantize_fp8(rnd(g, ROWS, 512))
    wq, wscale = K.quantize_fp8_weight(rnd(g, ROWS, 512))
    base = torch.empty(ROWS * STRIDE, dtype=torch.uint8, device=DEV)
    fq, fw = (far(base, t.view(torch.uint8), at).view(torch.float8_e4m3fn) for t, at in ((q, 0), (wq, 1024)))
    assert torch.equal(K.fp8_linear(fq[-m:], scale[-m:], fw, wscale), K.fp8_linear(q[-m:], scale[-m:], wq, wscale))
    assert K.device_error() == 0


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("lengths", [[20, 30], [1, 1], [700, 2]], ids=["whole", "steps", "split"])
@pytest.mark.parametrize("rows,n", [(40000, 128), (160000, 30)])
def test_state_tables_beyond_32_bits(dt, lengths, rows, n):
    """States behind 2^31 values of their table."""
    need_memory(24)
    h, p = 8, 64
    inp = scan_inputs(104, 2, sum(lengths), h, p, n, dt, False)
    table = torch.zeros(rows, h, p, n, device=DEV)
    slots = [rows - 1, rows - 3]
    table[slots] = inp["ssm"]
    want = scan(inp, K.SequenceBatch(lengths, device=DEV))
    y = scan({**inp, "ssm": table}, K.SequenceBatch(lengths, slots, device=DEV))
    assert torch.equal(y, want) and torch.equal(table[slots], inp["ssm"])
    assert not table[0].any() and not table[rows - 2].any()
    assert K.device_error() == 0


@pytest.mark.parametrize("lengths", [[20, 30], [1, 1]], ids=["prompt", "steps"])
@pytest.mark.parametrize("ch", [4352, 4351])
def test_windows_beyond_32_bits(lengths, ch):
    need_memory(24)
    rows = 170000
    g = gen(105)
    x, w, small = rnd(g, sum(lengths), ch), rnd(g, ch, 4), rnd(g, 2, ch, 3)
    table = torch.zeros(rows, ch, 3, device=DEV)
    slots = [rows - 1, rows - 3]
    table[slots] = small
    want = K.causal_conv(small, x, w, None, K.SequenceBatch(lengths, device=DEV))
    y = K.causal_conv(table, x, w, None, K.SequenceBatch(lengths, slots, device=DEV))
    assert torch.equal(y, want) and torch.equal(table[slots], small)
    assert not table[0].any() and not table[rows - 2].any()


# ------------------------------------------------- the integration guide's example


@pytest.mark.parametrize("dt", TYPES, ids=ids)
def test_example_of_the_guide_runs(dt):
    """The layer in INTEGRATION.md, as it stands there."""
    text = (Path(__file__).resolve().parent.parent / "INTEGRATION.md").read_text()
    code = next(b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "mamba2_scan(" in b)
    g, heads, size, bc, hid, tokens, rows = gen(110), 4, 64, 128, 256, 666, 16
    inner = heads * size
    env = dict(torch=torch, inner=inner, bc=bc, heads=heads, size=size, u=rnd(g, tokens, hid).to(dt), residual=rnd(g, tokens, hid).to(dt),
               norm_weight=torch.ones(hid, device=DEV), weight=rnd(g, 2 * inner + 2 * bc, hid) * hid ** -0.5,
               window=torch.zeros(rows, inner + 2 * bc, 3, device=DEV), conv_weight=rnd(g, inner + 2 * bc, 4), conv_bias=rnd(g, inner + 2 * bc),
               dt_weight=rnd(g, heads, hid) * hid ** -0.5, dt_bias=rnd(g, heads), ssm=torch.zeros(rows, heads, size, bc, device=DEV),
               a=-torch.ones(heads, device=DEV), d=torch.ones(heads, device=DEV))
    exec(code, env)
    assert env["y"].shape == (tokens, heads, size) and env["y"].dtype == dt and env["y"].isfinite().all() and env["y"].any()
    stepped = [7, 3, 12]
    assert all(env["ssm"][r].any() and env["window"][r].any() for r in stepped)
    assert not any(env["ssm"][r].any() for r in range(rows) if r not in stepped)
    assert K.device_error() == 0
