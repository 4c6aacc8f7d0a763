"""The run-of-tokens operators on the GPU (rms_norm_fp8, fp8_linear, causal_conv,
mamba2_scan) against float64 restatements of their formulas, at the sizes, types,
strides and masks where they can go wrong."""

import pytest
import torch

from hackathon_b200 import kernels as K
from tests import seqops_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = [str(t).split(".")[1] for t in TYPES]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rnd(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


# ------------------------------------------------------------------ norm


def norm_ref(x, w, r, eps, norm=True):
    v = x.double() if r is None else x.double() + r.double()
    n = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() if norm else v
    if w is not None:
        n = n * w.double()
    pad = torch.nn.functional.pad(n.abs(), (0, -n.shape[1] % 128))
    scale = (pad.unflatten(1, (-1, 128)).amax(-1) / 448).clamp(min=2.0 ** -100)
    return v, n, scale


def check_q(q, scale, n, want_scale, rel=2.0 ** -18):
    """float32 statistics are within 2^-18 (at most 2^6 roundings of 2^-24); e4m3 values within half a
    step: 2^-4 of a normal value, 2^-10 below 2^-6."""
    R.close(scale, want_scale, rel * want_scale, "scale")
    exact = n / want_scale.repeat_interleave(128, 1)[:, :n.shape[1]]
    tol = exact.abs().clamp(min=2.0 ** -6) * (2.0 ** -4 + 4 * rel)
    R.close(q.float(), exact, tol, "q")


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols,res", [
    (1, 2048, True), (3, 1, False), (5, 79, True), (7, 128, True), (130, 264, True), (2, 1000, False),
    (1300, 512, True), (33, 4096, True), (700, 4096, False), (4, 8192, True), (3, 8200, True), (2, 9001, True),
])
def test_rms_norm_fp8(dt, rows, cols, res):
    g = gen(rows * 31 + cols)
    x = (rnd(g, rows, cols) * 3).to(dt)
    w = torch.rand(cols, device=DEV, generator=g) + 0.5
    r = rnd(g, rows, cols).to(dt) if res else None
    out = K.rms_norm_fp8(x, w, residual=r, eps=1e-5, keep_norm=True)
    v, n, scale = norm_ref(x, w, r, 1e-5)
    assert out.q.dtype == torch.float8_e4m3fn and out.q.data_ptr() % 16 == 0
    check_q(out.q, out.scale, n, scale)
    R.close(out.normed, n, R.rounding(n, dt) + 2.0 ** -18 * n.abs(), "normed")
    if res:
        assert out.total.dtype == dt
        R.close(out.total, v, R.rounding(v, dt) + 2.0 ** -23 * (v.abs() + r.double().abs()), "total")
    else:
        assert out.total is None


@pytest.mark.parametrize("dt", TYPES[1:], ids=ids[1:])
def test_rms_norm_fp8_float32_residual_and_no_weight(dt):
    g = gen(4)
    x, r = rnd(g, 300, 256).to(dt), rnd(g, 300, 256)
    out = K.rms_norm_fp8(x, residual=r, eps=1e-6)
    v, n, scale = norm_ref(x, None, r, 1e-6)
    assert out.total.dtype == torch.float32 and out.normed is None
    check_q(out.q, out.scale, n, scale)
    R.close(out.total, v, 2.0 ** -23 * (v.abs() + r.double().abs()), "total")


@pytest.mark.parametrize("cols", [256, 250])
def test_rms_norm_fp8_strided_and_unaligned_rows(cols):
    g = gen(5)
    wide = rnd(g, 9, 3 * cols + 5)
    x, r = wide[:, 3:3 + cols], wide[:, 2 * cols:3 * cols]
    a = K.rms_norm_fp8(x, residual=r)
    b = K.rms_norm_fp8(x.contiguous(), residual=r.contiguous())
    v, n, scale = norm_ref(x, None, r, 1e-5)
    check_q(a.q, a.scale, n, scale)
    check_q(b.q, b.scale, n, scale)
    t = K.rms_norm_fp8(x.T.contiguous().T, residual=r)  # columns not contiguous: copied
    assert torch.equal(t.q.view(torch.uint8), a.q.view(torch.uint8))


@pytest.mark.parametrize("cols", [256, 250])
def test_rms_norm_fp8_special_rows(cols):
    """An all-zero row keeps a finite scale; a NaN or an infinity spoils its own row alone."""
    x = rnd(gen(6), 6, cols)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 1e-30
    out = K.rms_norm_fp8(x)
    assert not out.q[1].float().any() and (out.scale[1] == 2.0 ** -100).all()
    assert out.q[2].float().isnan().all()
    assert out.q[3, 7].float().isnan()
    clean = K.rms_norm_fp8(x[[0, 5]].contiguous())
    assert torch.equal(out.q[[0, 5]].view(torch.uint8) if cols % 16 == 0 else out.q[[0, 5]].float(),
                       clean.q.view(torch.uint8) if cols % 16 == 0 else clean.q.float())
    assert out.q[4].float().isfinite().all()


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(1, 16), (6, 79), (257, 384), (40, 4096)])
def test_quantize_fp8(dt, rows, cols):
    x = (rnd(gen(rows + cols), rows, cols) * 20).to(dt)
    q, scale = K.quantize_fp8(x)
    _, n, want = norm_ref(x, None, None, 0, norm=False)
    check_q(q, scale, n, want, rel=2.0 ** -22)


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 79), (300, 1000)])
def test_quantize_fp8_weight(dt, n, k):
    w = rnd(gen(n + k), n, k).to(dt)
    q, scale = K.quantize_fp8_weight(w)
    pad = torch.nn.functional.pad(w.double().abs(), (0, -k % 128, 0, -n % 128))
    want = (pad.unflatten(1, (-1, 128)).amax(-1).T.unflatten(1, (-1, 128)).amax(-1).T / 448).clamp(min=2.0 ** -100)
    R.close(scale, want, 2.0 ** -22 * want, "scale")
    full = want.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    exact = w.double() / full
    R.close(q.float(), exact, exact.abs().clamp(min=2.0 ** -6) * (2.0 ** -4 + 2.0 ** -20), "q")


# ---------------------------------------------------------------- linear


def linear_ref(q, scale, wq, wscale, bias, relu):
    k, n = q.shape[1], wq.shape[0]
    x = q.double() * scale.double().repeat_interleave(128, 1)[:, :k]
    w = wq.double() * wscale.double().repeat_interleave(128, 1)[:, :k].repeat_interleave(128, 0)[:n]
    y, mag = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return (y.relu() if relu else y), mag


@pytest.mark.parametrize("m,k,n,bias,relu,out", [
    (1, 2048, 8448, False, False, torch.bfloat16), (1, 1, 1, True, False, torch.float32),
    (3, 79, 130, True, True, torch.float32), (16, 128, 128, False, False, torch.float16),
    (17, 640, 200, True, False, torch.float32), (33, 4096, 300, False, False, torch.bfloat16),
    (64, 1000, 1280, True, True, torch.float16), (65, 256, 1280, True, False, torch.float32),
    (129, 384, 77, False, True, torch.float32), (1000, 2048, 528, True, False, torch.bfloat16),
    (4096, 256, 1280, False, False, torch.float32), (300, 17000, 136, False, False, torch.float32),
    (5, 17000, 136, False, False, torch.float32), (40, 40000, 20000, False, False, torch.bfloat16), (2500, 512, 2050, True, False, torch.float16),
    # whole tiles and halves in one launch, the last half empty or whole; whole tiles only
    (3845, 200, 1290, True, False, torch.float32), (4200, 300, 1280, True, True, torch.bfloat16), (3845, 2100, 1000, False, False, torch.float16),
    # blocks of 64 rows with the groups shared out over a cluster
    (65, 2048, 1280, True, False, torch.bfloat16), (400, 4100, 250, True, True, torch.float32), (200, 8192, 128, False, False, torch.float16),
])
def test_fp8_linear(m, k, n, bias, relu, out):
    """A product's terms are exact in float32; a group's 128 are summed in 4 steps and the groups one
    by one, each step rounding by at most 2^-23 of the terms' magnitudes."""
    g = gen(m * 3 + k + n)
    q, scale = K.quantize_fp8(rnd(g, m, k) * (0.5 + torch.rand(m, 1, device=DEV, generator=g)))
    wq, wscale = K.quantize_fp8_weight(rnd(g, n, k) * k ** -0.5)
    b = rnd(g, n) if bias else None
    y = K.fp8_linear(q, scale, wq, wscale, bias=b, relu=relu, out_dtype=out)
    want, mag = linear_ref(q, scale, wq, wscale, b, relu)
    assert y.dtype == out
    R.close(y, want, R.rounding(want, out) + (-(-k // 128) + 12) * 2.0 ** -23 * mag + 1e-30, "y")
    again = K.fp8_linear(q, scale, wq, wscale, bias=b, relu=relu, out_dtype=out)
    assert torch.equal(y, again), "the same operands give the same bits"
    assert K.device_error() == 0


@pytest.mark.parametrize("m,k", [(4, 300), (200, 300), (4, 1500), (100, 1500)])
def test_fp8_linear_rows_keep_to_themselves(m, k):
    """A row with a NaN, an infinite scale or a zero scale leaves the other rows' bits alone; strided and
    unaligned operands give the packed ones' bits."""
    g = gen(m)
    q, scale = K.quantize_fp8(rnd(g, m, k))
    wq, wscale = K.quantize_fp8_weight(rnd(g, 140, k))
    y = K.fp8_linear(q, scale, wq, wscale)
    bad_q, bad_s = q.clone(), scale.clone()
    bad_q.view(torch.uint8)[1, 5] = 0x7F  # e4m3 NaN
    bad_s[2, 1] = float("inf")
    z = K.fp8_linear(bad_q, bad_s, wq, wscale)
    assert z[1].isnan().all() and not z[2].isfinite().any()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(z[keep], y[keep])
    odd = torch.empty(m, k + 1, dtype=torch.uint8, device=DEV)[:, 1:]
    odd.copy_(q.view(torch.uint8) if q.is_contiguous() else q.contiguous().view(torch.uint8))
    assert torch.equal(K.fp8_linear(odd.view(torch.float8_e4m3fn), scale, wq, wscale), y)
    assert torch.equal(K.fp8_linear(q, scale.T.contiguous().T, wq, wscale), y)


# ------------------------------------------------------------------ conv


def conv_tol(want, mag, dtype):
    """Five float32 roundings of the sum; the activation's exponential and reciprocal are within 2^-20
    over the arguments here (below 16), all relative to at most the sum's magnitudes."""
    return R.rounding(want, dtype) + 2.0 ** -19 * mag + 1e-30


LENGTHS = [
    [1], [0], [5], [0, 1, 2, 3, 4, 7, 8, 9], [31, 0, 33, 1, 64, 100, 0], [1, 1, 1, 1], [1, 0, 1], [700], [3] * 70,
]


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("lengths", LENGTHS, ids=[str(i) for i in range(len(LENGTHS))])
@pytest.mark.parametrize("ch,taps,silu", [(64, 4, True), (7, 4, False), (264, 3, True), (40, 2, False)])
def test_causal_conv(dt, lengths, ch, taps, silu):
    g = gen(ch + sum(lengths))
    n, total = len(lengths), sum(lengths)
    rows = n + 2
    slots = torch.randperm(rows, generator=torch.Generator().manual_seed(n))[:n].tolist()
    window = rnd(g, rows, ch, taps - 1)
    x = rnd(g, total + 3, ch + 8).to(dt)[:, :ch]
    x[total:] = float("nan")  # rows behind the batch are not read
    w, b = rnd(g, ch, taps), rnd(g, ch) if silu else None
    before = window.clone()
    y = K.causal_conv(window, x, w, b, K.SequenceBatch(lengths, slots, state_rows=rows, device=DEV), silu=silu)
    want, win, mag = R.conv(before, x[:total], w, b, lengths, slots, silu)
    assert y.dtype == dt and y.is_contiguous() and y.shape == (total + 3, ch)
    assert not y[total:].any()
    R.close(y[:total], want, conv_tol(want, mag, dt), "y")
    assert torch.equal(window.double(), win), "a window holds the inputs themselves"


def test_causal_conv_long_prompt_and_steps_agree():
    """A prompt in one call, in two, and token by token leave the same window and the same values."""
    g = gen(1)
    ch, n = 4352, 900
    x, w, b = rnd(g, n, ch).bfloat16(), rnd(g, ch, 4), rnd(g, ch)
    win = [rnd(g, 1, ch, 3)] * 3
    win = [v.clone() for v in win]
    whole = K.causal_conv(win[0], x, w, b, K.SequenceBatch([n], device=DEV), silu=True)
    parts = torch.cat([K.causal_conv(win[1], x[s], w, b, K.SequenceBatch([len(x[s])], device=DEV), silu=True)
                       for s in (slice(0, 401), slice(401, n))])
    assert torch.equal(whole, parts) and torch.equal(win[0], win[1])
    for i in range(20):
        assert torch.equal(K.causal_conv(win[2], x[i:i + 1], w, b, silu=True), whole[i:i + 1])


def test_causal_conv_neighbours_do_not_leak():
    g = gen(2)
    x, w = rnd(g, 90, 32), rnd(g, 32, 4)
    win = rnd(g, 3, 32, 3)
    clean_win, bad_win = win.clone(), win.clone()
    clean = K.causal_conv(clean_win, x, w, None, K.SequenceBatch([30, 30, 30], device=DEV))
    bad = x.clone()
    bad[30:60] = float("nan")
    bad_win[1] = float("inf")
    y = K.causal_conv(bad_win, bad, w, None, K.SequenceBatch([30, 30, 30], device=DEV))
    for s in (slice(0, 30), slice(60, 90)):
        assert torch.equal(y[s], clean[s])
    assert torch.equal(bad_win[[0, 2]], clean_win[[0, 2]])


# ------------------------------------------------------------------ scan


def scan_inputs(seed, rows, tokens, h, p, n, dt, gate):
    g = gen(seed)
    return dict(ssm=rnd(g, rows, h, p, n), x=rnd(g, tokens, h, p).to(dt), b=rnd(g, tokens, n).to(dt), c=rnd(g, tokens, n).to(dt),
                dt=rnd(g, tokens, h) - 2, a=-torch.exp(2 * torch.rand(h, device=DEV, generator=g)),
                d=rnd(g, h) if gate else None, z=rnd(g, tokens, h, p).to(dt) if gate else None)


PAIRS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 0.0}


def check_scan(inp, lengths, slots, rows, total, pairs=None, softplus=True, extra=0):
    dt = inp["x"].dtype
    before = inp["ssm"].clone()
    seqs = None if lengths is None else K.SequenceBatch(lengths, slots, state_rows=rows, device=DEV)
    y = K.mamba2_scan(inp["ssm"], inp["x"], inp["b"], inp["c"], inp["dt"], inp["a"], seqs, d=inp["d"], z=inp["z"], softplus=softplus)
    lens = [1] * rows if lengths is None else lengths
    slts = list(range(rows)) if slots is None else slots
    cut = {k: v[:total] if k in ("x", "b", "c", "dt", "z") and v is not None else v for k, v in inp.items()}
    want, ssm, ymag, smag = R.scan(before, cut["x"], cut["b"], cut["c"], cut["dt"], cut["a"], lens, slts, cut["d"], cut["z"], softplus)
    steps = max(lens, default=0) + 1
    pairs = PAIRS[dt] if pairs is None else pairs
    assert y.dtype == dt and y.is_contiguous()
    assert not y[total:].any()
    gate = 4 * 2.0 ** -22 * want.abs()  # the gate's exponential and division
    R.close(y[:total], want, R.scan_tol(want, ymag, steps, dt, pairs) + gate, "y")
    R.close(inp["ssm"], ssm, R.scan_tol(ssm, smag, steps, torch.float32), "ssm")
    idle = [r for r in range(rows) if r not in [s for s, k in zip(slts, lens) if k]]
    assert torch.equal(inp["ssm"][idle], before[idle]), "idle rows stay bit for bit"
    assert K.device_error() == 0
    return y


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("rows,h,p,n,gate", [
    (1, 64, 64, 128, True), (5, 8, 64, 64, False), (300, 8, 64, 128, True), (3, 2, 17, 40, True), (4, 3, 100, 256, False),
    (3, 2, 33, 30, True), (2, 1, 1, 1, False), (7, 5, 64, 4, True), (0, 4, 64, 128, False),
])
def test_mamba2_scan_single_tokens(dt, rows, h, p, n, gate):
    check_scan(scan_inputs(rows + h + p + n, rows, rows, h, p, n, dt, gate), None, None, rows, rows, pairs=0.0)


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("lengths", LENGTHS + [[127, 128, 129, 0, 1, 255]], ids=[str(i) for i in range(len(LENGTHS) + 1)])
@pytest.mark.parametrize("h,p,n,gate", [(4, 64, 128, True), (3, 64, 64, False), (2, 48, 40, True), (1, 65, 130, False), (5, 64, 128, False)])
def test_mamba2_scan_prompts(dt, lengths, h, p, n, gate):
    count, total = len(lengths), sum(lengths)
    rows = count + 2
    slots = torch.randperm(rows, generator=torch.Generator().manual_seed(count))[:count].tolist()
    inp = scan_inputs(total + h + p + n, rows, total + 3, h, p, n, dt, gate)
    for k in ("x", "b", "c", "dt", "z"):
        if inp[k] is not None:
            inp[k][total:] = float("nan")  # rows behind the batch are not read
    check_scan(inp, lengths, slots, rows, total)


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("h,lengths", [(8, [5000]), (2, [1, 3000, 0, 2000]), (1, [385, 1500])])
def test_mamba2_scan_long_sequences_are_split(dt, h, lengths):
    rows = len(lengths)
    check_scan(scan_inputs(h, rows, sum(lengths), h, 64, 128, dt, False), lengths, None, rows, sum(lengths))


@pytest.mark.parametrize("dt", TYPES, ids=ids)
def test_mamba2_scan_prompt_equals_single_tokens(dt):
    """A prompt leaves the state that as many single steps leave, and gives their outputs."""
    inp = scan_inputs(3, 2, 60, 4, 64, 128, dt, True)
    ssm = inp["ssm"].clone()
    y = check_scan(inp, [40, 20], None, 2, 60)
    for i in range(20):
        at = torch.tensor([i, 40 + i], device=DEV)
        one = K.mamba2_scan(ssm, inp["x"][at], inp["b"][at], inp["c"][at], inp["dt"][at], inp["a"], d=inp["d"], z=inp["z"][at])
        tol = (2 * R.half(dt) + PAIRS[dt] + 2.0 ** -18) * one.double().abs() + (PAIRS[dt] + 2.0 ** -18) * 40
        R.close(y[at], one.double(), tol, f"token {i}")


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("h", [1, 40])
def test_mamba2_scan_strides(dt, h):
    """Operands as slices of a joined projection's rows."""
    g = gen(8)
    p, n, t = 64, 128, 300
    wide = rnd(g, t, 2 * h * p + 2 * n + 8).to(dt)
    inp = scan_inputs(9, 2, t, h, p, n, dt, True)
    inp["x"] = wide[:, :h * p].unflatten(1, (h, p))
    inp["z"] = wide[:, h * p:2 * h * p].unflatten(1, (h, p))
    inp["b"], inp["c"] = wide[:, 2 * h * p:2 * h * p + n], wide[:, 2 * h * p + n:2 * h * p + 2 * n]
    inp["dt"] = torch.cat([inp["dt"], inp["dt"]], 1)[:, :h]
    assert not inp["x"].is_contiguous()
    check_scan(inp, [130, 170], [1, 0], 2, t)


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("kind", ["reset", "hold", "grow", "zero", "mixed"])
def test_mamba2_scan_decays(dt, kind):
    """Steps that reset the state (decay 0), hold it (decay 1), let it grow, add nothing."""
    inp = scan_inputs(11, 2, 400, 4, 64, 128, dt, False)
    if kind == "reset":
        inp["dt"][::37] = 500.0
    elif kind == "hold":
        inp["dt"][:] = -30.0
    elif kind == "grow":
        inp["a"] = inp["a"].abs() * 0.01
    elif kind == "zero":
        inp["dt"][:] = 0.0
    else:
        inp["dt"] = inp["dt"] * 4
        inp["dt"][::50] = 80.0
    check_scan(inp, [250, 150], None, 2, 400, softplus=kind != "zero")


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("n", [40, 100, 200])
def test_mamba2_scan_products_of_decays(dt, n):
    """Products of a sequence's decays far above and far below one, in small steps and in large ones."""
    inp = scan_inputs(12, 3, 160, 2, 48, n, dt, False)
    steps = torch.full((160, 2), 0.6, device=DEV)
    steps[:40] = -0.6                # up by e^24 and down again, then as far below
    steps[80:100] = 9.0              # each decay below the range that is kept on
    steps[100:120] = -1.0
    inp["dt"], inp["a"] = steps, torch.tensor([-1.0, -0.3], device=DEV)
    check_scan(inp, [100, 20, 40], None, 3, 160, pairs=0.0, softplus=False)


@pytest.mark.parametrize("dt", TYPES, ids=ids)
@pytest.mark.parametrize("name", ["x", "b", "c", "dt"])
def test_mamba2_scan_values_that_are_not_finite_stay_behind(dt, name):
    """A NaN or an infinity in a token reaches neither earlier tokens nor other sequences or heads' rows."""
    lengths = [200, 200, 200]
    inp = scan_inputs(13, 3, 600, 4, 64, 128, dt, False)
    clean = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in inp.items()}
    seqs = K.SequenceBatch(lengths, device=DEV)
    args = ("x", "b", "c", "dt", "a")
    want = K.mamba2_scan(clean["ssm"], *[clean[k] for k in args], seqs)
    inp[name][260] = float("inf") if name == "x" else float("nan")
    got = K.mamba2_scan(inp["ssm"], *[inp[k] for k in args], seqs)
    assert torch.equal(got[:260], want[:260]) and torch.equal(got[400:], want[400:])
    assert not got[260].isfinite().any()
    assert torch.equal(inp["ssm"][[0, 2]], clean["ssm"][[0, 2]])
    if name != "c":  # the state carries it on
        assert not got[399].isfinite().any() and not inp["ssm"][1].isfinite().all()


def test_plans_of_other_batches_and_streams():
    """Two streams, each with its own batch and tables, and the work's own buffers."""
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    cases = [scan_inputs(20 + i, 2, 3000, 2, 64, 128, torch.bfloat16, True) for i in range(2)]
    want = []
    for c in cases:
        ssm = c["ssm"].clone()
        want.append((K.mamba2_scan(ssm, c["x"], c["b"], c["c"], c["dt"], c["a"], K.SequenceBatch([1000, 2000], device=DEV), d=c["d"], z=c["z"]), ssm))
    torch.cuda.synchronize()
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got.append(K.mamba2_scan(c["ssm"], c["x"], c["b"], c["c"], c["dt"], c["a"], K.SequenceBatch([1000, 2000], device=DEV), d=c["d"], z=c["z"]))
    torch.cuda.synchronize()
    for c, g, (y, ssm) in zip(cases, got, want):
        assert torch.equal(g, y) and torch.equal(c["ssm"], ssm)


def test_operators_in_a_captured_graph():
    """Norm, projection, convolution and scan captured once and replayed on new inputs."""
    g = gen(30)
    h, p, n, hid, t = 8, 64, 128, 256, 700
    ch = h * p + 2 * n
    wq, ws = K.quantize_fp8_weight(rnd(g, ch, hid) * hid ** -0.5)
    seqs = K.SequenceBatch([300, 400], device=DEV)
    x, conv_w, dt, a = rnd(g, t, hid).bfloat16(), rnd(g, ch, 4), rnd(g, t, h) - 2, -torch.rand(h, device=DEV, generator=g)
    window, ssm = torch.zeros(2, ch, 3, device=DEV), torch.zeros(2, h, p, n, device=DEV)

    def step():
        q = K.rms_norm_fp8(x)
        xbc = K.causal_conv(window, K.fp8_linear(q.q, q.scale, wq, ws, out_dtype=torch.bfloat16), conv_w, None, seqs, silu=True)
        return K.mamba2_scan(ssm, xbc[:, :h * p].unflatten(1, (h, p)), xbc[:, h * p:h * p + n], xbc[:, h * p + n:], dt, a, seqs)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for seed in (31, 32):
        x.copy_(rnd(gen(seed), t, hid).bfloat16())
        window.zero_(), ssm.zero_()
        want, state = step().clone(), ssm.clone()
        window.zero_(), ssm.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(ssm, state)
    del graph


def test_large_offsets():
    """A state table beyond 2^31 values and rows beyond 2^31 elements."""
    rows, h, p, n = 40000, 8, 64, 128  # 2.6e9 floats
    free, _ = torch.cuda.mem_get_info(DEV)
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    ssm = torch.zeros(rows, h, p, n, device=DEV)
    inp = scan_inputs(40, 2, 50, h, p, n, torch.bfloat16, False)
    slots = [rows - 1, rows - 3]
    small = inp["ssm"].zero_()
    seqs = K.SequenceBatch([20, 30], slots, state_rows=rows, device=DEV)
    y = K.mamba2_scan(ssm, inp["x"], inp["b"], inp["c"], inp["dt"], inp["a"], seqs)
    want = K.mamba2_scan(small, inp["x"], inp["b"], inp["c"], inp["dt"], inp["a"], K.SequenceBatch([20, 30], device=DEV))
    assert torch.equal(y, want) and torch.equal(ssm[slots], small)
    assert not ssm[0].any() and not ssm[rows - 2].any()
