"""Cases of the sequence and 8-bit operators, each with a plain form and an exact one.

Four operators that a Mamba2 layer is made of when a whole run of tokens goes through it at
once: the RMS norm that adds the residual and writes 8 bits with scales, the 8-bit projection,
the short causal convolution and the selective scan, the last two for prompts and for single
tokens. Where ``own`` is false ``run`` computes them with elementary torch operations; where it
is true it calls ``hackathon_b200.kernels``.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
GROUP = 128  # values of a row, and rows and columns of a weight's block, that share a scale
F8_MAX = 448.0  # largest e4m3 value
MIN_SCALE = 2.0 ** -100  # keeps the quotient of an all-zero group finite
CHUNK = 64  # tokens that the plain scan takes together


def listed():
    return [
        # one request's row at the default model's hidden size: latency
        dict(name="norm 1x2048 bf16", op="norm", rows=1, cols=2048, dtype="bf16", residual=True),
        # a long backlog at the default model's inner size: bandwidth
        dict(name="norm 16384x4096 bf16", op="norm", rows=16384, cols=4096, dtype="bf16", residual=True),
        # one token through the default model's joined x|z|b|c projection: the weights' bytes count
        dict(name="linear 1x2048x8448", op="linear", rows=1, inner=2048, cols=8448, bias=False, relu=False, out="bf16"),
        # a 4096-symbol step's joined projection at hidden 256: short inner size, few tiles
        dict(name="linear 4096x256x1280", op="linear", rows=4096, inner=256, cols=1280, bias=True, relu=False, out="fp32"),
        # a 10,000-request stream through the default model's output projection: rate
        dict(name="linear 10000x4096x2048", op="linear", rows=10000, inner=4096, cols=2048, bias=False, relu=False, out="bf16"),
        # a 4096-symbol step at hidden 256: x, b and c channels, one token a sequence
        dict(name="conv step 4096x768 fp32", op="conv", seqs=4096, tokens=4096, channels=768, dtype="fp32", step=True),
        # a 10,000-request stream of 16 symbols, x|b|c columns of the default model's projection
        dict(name="conv prompt 10000x4352 bf16", op="conv", seqs=16, tokens=10000, channels=4352, dtype="bf16", step=False),
        # one request's state update at the default model: latency
        dict(name="scan step 1x64 fp32", op="scan", seqs=1, tokens=1, heads=64, size=64, state=128, dtype="fp32", gate=False, step=True),
        # a 4096-symbol step at hidden 256: the state's bytes count
        dict(name="scan step 4096x8 fp32", op="scan", seqs=4096, tokens=4096, heads=8, size=64, state=128, dtype="fp32", gate=True, step=True),
        # the histories of 64 symbols at the default model, ragged
        dict(name="scan prompt 64/32768x64 bf16", op="scan", seqs=64, tokens=32768, heads=64, size=64, state=128, dtype="bf16", gate=True, step=False),
        # the histories of 64 symbols at hidden 256 in 32 bits, as the layer runs with fp32 weights
        dict(name="scan prompt 64/10000x8 fp32", op="scan", seqs=64, tokens=10000, heads=8, size=64, state=128, dtype="fp32", gate=False, step=False),
        # one symbol's long history at hidden 256: few rows, a long axis
        dict(name="scan prompt 1/16384x8 bf16", op="scan", seqs=1, tokens=16384, heads=8, size=64, state=128, dtype="bf16", gate=False, step=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "conv", "scan", "scan"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "norm":
        return dict(op=op, rows=_log(rng, 1, 12000), cols=_log(rng, 64, 4096), dtype=dtype, residual=rng.random() < 0.7)
    if op == "linear":
        return dict(op=op, rows=_log(rng, 1, 10000), inner=_log(rng, 79, 4096), cols=_log(rng, 16, 2048),
                    bias=rng.random() < 0.5, relu=rng.random() < 0.3, out=dtype)
    step = rng.random() < 0.4
    seqs = _log(rng, 1, 4096) if step else _log(rng, 1, 64)
    if op == "conv":
        return dict(op=op, seqs=seqs, tokens=seqs if step else _log(rng, seqs, 10000), channels=_log(rng, 8, 2048), dtype=dtype, step=step)
    return dict(op=op, seqs=seqs, tokens=seqs if step else _log(rng, seqs, 10000), heads=_log(rng, 1, 8 if step else 24),
                size=rng.choice([64, 64, 64, 32, 48, 96]), state=rng.choice([128, 128, 64, 40]), dtype=dtype,
                gate=rng.random() < 0.5, step=step)


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """Ragged lengths that sum to the tokens, the same for every seed (zero among them at times)."""
    if case["step"]:
        return [1] * case["seqs"]
    rng = random.Random(case["seqs"] * 1000003 + case["tokens"])
    cuts = sorted(rng.randrange(case["tokens"] + 1) for _ in range(case["seqs"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]


def _rand(g, *shape, lo=None, hi=None):
    if lo is None:
        return torch.randn(*shape, device=DEV, generator=g)
    return torch.rand(*shape, device=DEV, generator=g) * (hi - lo) + lo


def _round8(v, scale):
    return (v / scale).to(torch.float8_e4m3fn)


def _groups(x, size=GROUP):
    """Largest magnitude of each group of `size` columns (the last one may be short)."""
    pad = -x.shape[-1] % size
    return torch.nn.functional.pad(x.abs(), (0, pad)).unflatten(-1, (-1, size)).amax(-1)


def _spread(scale, cols):
    return scale.repeat_interleave(GROUP, -1)[..., :cols]


def _rows16(q):
    """The same values in rows that start on 16 bytes, as a quantiser lays them out for the projection."""
    wide = torch.zeros(q.shape[0], q.shape[1] + -q.shape[1] % 16, device=DEV, dtype=torch.float8_e4m3fn)
    wide[:, :q.shape[1]] = q
    return wide[:, :q.shape[1]]


def _weight8(w):
    """(out, in) weights in 8 bits with a scale for each 128 x 128 block."""
    scale = (_groups(_groups(w).T).T / F8_MAX).clamp(min=MIN_SCALE).contiguous()
    full = _spread(_spread(scale, w.shape[1]).T, w.shape[0]).T
    return _rows16(_round8(w, full)), scale


def _sequences(case, g):
    """Lengths, starts and state rows: a program's symbols sit anywhere in its state table."""
    n = case["seqs"]
    rows = n if case["step"] else n + 3
    slots = torch.randperm(rows, device=DEV, generator=g)[:n]
    return _lengths(case), slots.tolist(), rows


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES.get(case.get("dtype"))
    s = dict(case=case)
    if case["op"] == "norm":
        m, k = case["rows"], case["cols"]
        s["x"] = _rand(g, m, k).to(dt)
        s["residual"] = (_rand(g, m, k) * 2).to(dt) if case["residual"] else None
        s["weight"] = _rand(g, k, lo=0.5, hi=1.5)
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["cols"]
        x = _rand(g, m, k) * _rand(g, m, 1, lo=0.5, hi=2.0)
        s["scale"] = (_groups(x) / F8_MAX).clamp(min=MIN_SCALE)
        s["q"] = _rows16(_round8(x, _spread(s["scale"], k)))
        s["wq"], s["wscale"] = _weight8(_rand(g, n, k, lo=-1.0, hi=1.0) * k ** -0.5)
        s["bias"] = _rand(g, n, lo=-0.5, hi=0.5) if case["bias"] else None
    elif case["op"] == "conv":
        lengths, slots, rows = _sequences(case, g)
        c = case["channels"]
        # columns of a wider projection's output, as the layer has them
        s["x"] = _rand(g, case["tokens"], c + 32).to(dt)[:, :c]
        s["window"] = _rand(g, rows, c, 3)
        s["weight"] = _rand(g, c, 4, lo=-0.5, hi=0.5)
        s["bias"] = _rand(g, c, lo=-0.5, hi=0.5)
        _plan(s, case, lengths, slots, rows)
    else:
        lengths, slots, rows = _sequences(case, g)
        t, h, p, n = case["tokens"], case["heads"], case["size"], case["state"]
        s["x"] = _rand(g, t, h, p).to(dt)
        s["b"] = _rand(g, t, n).to(dt)
        s["c"] = _rand(g, t, n).to(dt)
        # steps between 0.001 and 0.1 around the layer's bias, decay rates between 1 and 16
        target = torch.exp(_rand(g, h, lo=math.log(1e-3), hi=math.log(0.1)))
        s["dt"] = _rand(g, t, h) * 0.5 + torch.log(torch.expm1(target))
        s["a"] = -torch.exp(_rand(g, h, lo=0.0, hi=math.log(16.0)))
        s["d"] = _rand(g, h, lo=0.5, hi=1.5) if case["gate"] else None
        s["z"] = _rand(g, t, h, p).to(dt) if case["gate"] else None
        s["ssm"] = _rand(g, rows, h, p, n) * 0.5
        _plan(s, case, lengths, slots, rows)
    return s


def _plan(s, case, lengths, slots, rows):
    """What a program keeps for a batch of sequences: index tensors for the plain form, and the
    framework's plan. A step over the whole table (row i is state row i) needs neither."""
    s["slots"] = None
    if case["step"]:
        s["seqs"] = None
        return
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    s["lengths"] = torch.tensor(lengths, device=DEV)
    s["starts"] = torch.tensor(starts[:-1], device=DEV)
    s["longest"] = max(lengths)
    s["slots"] = torch.tensor(slots, device=DEV)
    s["owner"] = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), s["lengths"])
    if own:
        from hackathon_b200 import kernels

        s["seqs"] = kernels.SequenceBatch(lengths, slots, state_rows=rows, device=torch.device(DEV, 0))


# ------------------------------------------------------------------ one pass


def run(state):
    return {"norm": _norm, "linear": _linear, "conv": _conv, "scan": _scan}[state["case"]["op"]](state)


def _norm(s):
    if own:
        from hackathon_b200 import kernels

        r = kernels.rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=1e-5)
        return [r.q, r.scale] + ([] if r.total is None else [r.total])
    v = s["x"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    n = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-5) * s["weight"]
    scale = (_groups(n) / F8_MAX).clamp(min=MIN_SCALE)
    q = _round8(n, _spread(scale, n.shape[1]))
    return [q, scale] + ([] if s["residual"] is None else [v.to(s["x"].dtype)])


def _linear(s):
    case = s["case"]
    if own:
        from hackathon_b200 import kernels

        return kernels.fp8_linear(s["q"], s["scale"], s["wq"], s["wscale"], bias=s["bias"], relu=case["relu"],
                                  out_dtype=DTYPES[case["out"]])
    k, n = case["inner"], case["cols"]
    x = s["q"].float() * _spread(s["scale"], k)
    w = s["wq"].float() * _spread(_spread(s["wscale"], k).T, n).T
    y = x @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["relu"]:
        y = y.clamp(min=0)
    return y.to(DTYPES[case["out"]])


def _conv(s):
    x, window = s["x"], s["window"]
    if own:
        from hackathon_b200 import kernels

        return [kernels.causal_conv(window, x, s["weight"], s["bias"], s["seqs"], silu=True), window]
    w = s["weight"]
    if s["slots"] is None:
        taps = torch.cat([window, x.float()[:, :, None]], -1)
        y = (taps * w).sum(-1) + s["bias"]
        window.copy_(taps[:, :, 1:])
    else:
        # the windows ahead of their sequences, in one run of rows: token t of sequence i is row t + 3 (i + 1)
        n = len(s["lengths"])
        rows = torch.empty(x.shape[0] + 3 * n, x.shape[1], device=x.device)
        at = torch.arange(x.shape[0], device=x.device) + 3 * (s["owner"] + 1)
        head = (s["starts"] + 3 * torch.arange(n, device=x.device))[:, None] + torch.arange(3, device=x.device)
        rows[at] = x.float()
        rows[head] = window[s["slots"]].transpose(1, 2)
        y = rows[at - 3] * w[:, 0] + rows[at - 2] * w[:, 1] + rows[at - 1] * w[:, 2] + rows[at] * w[:, 3] + s["bias"]
        window[s["slots"]] = rows[head + s["lengths"][:, None]].transpose(1, 2)
    return [(y * torch.sigmoid(y)).to(x.dtype), window]


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _scan(s):
    x, ssm = s["x"], s["ssm"]
    if own:
        from hackathon_b200 import kernels

        return [kernels.mamba2_scan(ssm, x, s["b"], s["c"], s["dt"], s["a"], s["seqs"], d=s["d"], z=s["z"]), ssm]
    y = _scan_step(s) if s["slots"] is None else _scan_chunks(s)
    if s["d"] is not None:
        y = y + s["d"][:, None] * x.float()
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z * torch.sigmoid(z))
    return [y.to(x.dtype), ssm]


def _scan_step(s):
    dt = _softplus(s["dt"])
    ssm = s["ssm"]
    ssm.mul_(torch.exp(s["a"] * dt)[:, :, None, None])
    ssm.add_((dt[:, :, None] * s["x"].float())[..., None] * s["b"].float()[:, None, None, :])
    return (ssm * s["c"].float()[:, None, None, :]).sum(-1)


def _scan_chunks(s):
    """Chunks of CHUNK tokens: inside a chunk every pair of tokens by its decay, between chunks by
    the chunks' states. Decays are summed in 64 bits, where far tokens' sums cancel."""
    n, q = len(s["lengths"]), CHUNK
    chunks = max(1, -(-s["longest"] // q))
    offset = torch.arange(chunks * q, device=DEV)
    valid = offset < s["lengths"][:, None]
    at = torch.where(valid, s["starts"][:, None] + offset, 0)

    def take(v):  # (tokens, ...) -> (sequences, chunks, q, ...), zeros behind a sequence
        w = v.float()[at]
        w = torch.where(valid.reshape(valid.shape + (1,) * (w.dim() - 2)), w, 0.0)
        return w.unflatten(1, (chunks, q))

    x, b, c = take(s["x"]), take(s["b"]), take(s["c"])
    dt = take(_softplus(s["dt"]))
    log = (s["a"].double() * dt.double()).cumsum(2)  # (n, chunks, q, heads)
    log_t = log.permute(0, 1, 3, 2)
    pair = (log_t[..., :, None] - log_t[..., None, :]).float()
    causal = torch.ones(q, q, dtype=torch.bool, device=DEV).tril()
    pair = torch.where(causal, torch.exp(pair), 0.0)
    pair = pair * (c @ b.transpose(-1, -2))[:, :, None] * dt.permute(0, 1, 3, 2)[..., None, :]
    xh = x.permute(0, 1, 3, 2, 4)  # (n, chunks, heads, q, size)
    y = pair @ xh
    total = log[:, :, -1]  # (n, chunks, heads)
    left = torch.exp((total[:, :, None] - log).float()) * dt
    own_state = (left.permute(0, 1, 3, 2)[..., None] * xh).transpose(-1, -2) @ b[:, :, None]  # (n, chunks, heads, size, state)
    ends = torch.nn.functional.pad(total.cumsum(1), (0, 0, 1, 0)).permute(0, 2, 1)  # log decay before chunk i, and in all
    far = (ends[:, :, :, None] - ends[:, :, None, 1:]).float()
    before = torch.ones(chunks + 1, chunks, dtype=torch.bool, device=DEV).tril(-1)
    far = torch.where(before, torch.exp(far), 0.0)  # (n, heads, chunks + 1, chunks)
    first = s["ssm"][s["slots"]]  # (n, heads, size, state)
    size = first.shape[-2:]
    states = (far @ own_state.transpose(1, 2).flatten(3)).unflatten(-1, size)
    states = states + torch.exp(ends.float())[..., None, None] * first[:, :, None]
    s["ssm"][s["slots"]] = states[:, :, -1]
    carried = states[:, :, :-1].transpose(1, 2)  # (n, chunks, heads, size, state)
    y = y + (c[:, :, None] @ carried.transpose(-1, -2)) * torch.exp(log_t.float())[..., None]
    y = y.permute(0, 1, 3, 2, 4).flatten(1, 2)  # (n, chunks * q, heads, size)
    token = torch.arange(s["x"].shape[0], device=DEV)
    return y[s["owner"], token - s["starts"][s["owner"]]]


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "norm":
        m, k, e = case["rows"], case["cols"], SIZE[case["dtype"]]
        return dict(bytes=m * k * (1 + e * (3 if case["residual"] else 1)) + m * -(-k // GROUP) * 4 + k * 4, flops=6 * m * k)
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["cols"]
        g = -(-k // GROUP)
        return dict(bytes=m * k + n * k + m * g * 4 + -(-n // GROUP) * g * 4 + m * n * SIZE[case["out"]] + (4 * n if case["bias"] else 0),
                    flops=2 * m * n * k)
    e, t = SIZE[case["dtype"]], case["tokens"]
    if case["op"] == "conv":
        c = case["channels"]
        touched = sum(1 for n in _lengths(case) if n)
        return dict(bytes=2 * t * c * e + touched * c * 3 * 8 + c * 20, flops=12 * t * c)
    h, p, n = case["heads"], case["size"], case["state"]
    touched = sum(1 for k in _lengths(case) if k)
    return dict(bytes=t * h * p * e * (3 if case["gate"] else 2) + 2 * t * n * e + t * h * 4 + touched * h * p * n * 8 + h * 8,
                flops=5 * t * h * p * n)


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        v = s["x"].double()
        if s["residual"] is not None:
            v = v + s["residual"].double()
        k = v.shape[1]
        n = v / (v.square().sum(1, keepdim=True) / k + 1e-5).sqrt() * s["weight"].double()
        scale = torch.stack([n[:, i:i + GROUP].abs().max(1).values for i in range(0, k, GROUP)], 1) / F8_MAX
        scale = scale.clamp(min=MIN_SCALE)
        q = n / scale[:, torch.arange(k, device=DEV) // GROUP]
        return [q, scale] + ([] if s["residual"] is None else [v])
    if case["op"] == "linear":
        k, n = case["inner"], case["cols"]
        by_k, by_n = torch.arange(k, device=DEV) // GROUP, torch.arange(n, device=DEV) // GROUP
        x = s["q"].double() * s["scale"].double()[:, by_k]
        w = s["wq"].double() * s["wscale"].double()[by_n][:, by_k]
        y = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
        return y.relu() if case["relu"] else y
    if case["op"] == "conv":
        return _exact_conv(s, case)
    return _exact_scan(s, case)


def _rows_of(s, case):
    lengths = _lengths(case)
    slots = list(range(case["seqs"])) if s["slots"] is None else s["slots"].tolist()
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return lengths, slots, starts


def _exact_conv(s, case):
    x, w, window = s["x"].double(), s["weight"].double(), s["window"].double()
    if case["step"]:
        full = torch.cat([window, x[:, :, None]], 2)
        y = torch.einsum("scj,cj->sc", full, w) + s["bias"].double()
        return [y / (1 + torch.exp(-y)), full[:, :, 1:]]
    y = torch.zeros_like(x)
    for n, row, at in zip(*_rows_of(s, case)):
        full = torch.cat([window[row].T, x[at:at + n]])  # (3 + n, channels)
        for j in range(4):
            y[at:at + n] += full[j:j + n] * w[:, j]
        window[row] = full[n:].T
    y = y + s["bias"].double()
    return [y / (1 + torch.exp(-y)), window]


def _exact_scan(s, case):
    x, b, c = s["x"].double(), s["b"].double(), s["c"].double()
    dt = torch.nn.functional.softplus(s["dt"].double())
    decay = torch.exp(s["a"].double() * dt)
    ssm = s["ssm"].double()
    y = torch.zeros_like(x)
    lengths, slots, starts = _rows_of(s, case)
    order = sorted(range(len(lengths)), key=lambda i: -lengths[i])  # the longest first, so that those that go on stay in front
    rows = torch.tensor([slots[i] for i in order], device=DEV)
    first = torch.tensor([starts[i] for i in order], device=DEV)
    h = ssm[rows]
    for t in range(max(lengths)):
        live = sum(1 for i in order if lengths[i] > t)
        at = first[:live] + t
        u = (dt[at][..., None] * x[at])[..., None] * b[at][:, None, None, :]
        h[:live] = torch.addcmul(u, h[:live], decay[at][..., None, None])
        y[at] = torch.einsum("shpn,sn->shp", h[:live], c[at])
    ssm[rows] = h
    if s["d"] is not None:
        y = y + s["d"].double()[:, None] * x
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z / (1 + torch.exp(-z))
    return [y, ssm]
