"""Float64 restatements of the run-of-tokens operators, with the sums of absolute
values that bound a float32 evaluation's rounding. Test infrastructure only."""

import math

import torch


def half(dtype):
    """Half a step of a type, relative to the value."""
    return torch.finfo(dtype).eps / 2


def rounding(value, dtype):
    """What one rounding to `dtype` may be off: half a step, which is eps / 2 relative to the value (and
    1% for a value that float32 has already moved across a power of two), and below the smallest normal
    number, where steps no longer shrink, eps / 2 of that number (2^-25 for float16)."""
    return half(dtype) * (1.01 * value.abs() + torch.finfo(dtype).smallest_normal)


def seq_rows(lengths):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return list(zip(starts, starts[1:]))


def conv(window, x, w, bias, lengths, slots, silu):
    """(y, new window, sum of magnitudes ahead of the activation)."""
    x, w, window = x.double(), w.double(), window.double().clone()
    b = torch.zeros(x.shape[1], dtype=torch.float64, device=x.device) if bias is None else bias.double()
    taps = w.shape[1]
    y, mag = torch.zeros_like(x), torch.zeros_like(x)
    for (s, e), slot in zip(seq_rows(lengths), slots):
        v = torch.cat([window[slot].T, x[s:e]])
        for j in range(taps):
            y[s:e] += v[j:j + e - s] * w[:, j]
            mag[s:e] += v[j:j + e - s].abs() * w[:, j].abs()
        y[s:e] += b
        mag[s:e] += b.abs()
        window[slot] = v[v.shape[0] - taps + 1:].T
    if silu:
        y = y * torch.sigmoid(y)
    return y, window, mag


def scan(ssm, x, b, c, dt, a, lengths, slots, d=None, z=None, softplus=True):
    """(y, new ssm, magnitudes of y's sum ahead of the gate, of the state's): the recurrence token by token."""
    x, b, c = x.double(), b.double(), c.double()
    t = torch.nn.functional.softplus(dt.double()) if softplus else dt.double()
    decay = torch.exp(a.double() * t)
    ssm = ssm.double().clone()
    mag = ssm.abs()
    y, ymag = torch.zeros_like(x), torch.zeros_like(x)
    for (s, e), slot in zip(seq_rows(lengths), slots):
        h, m = ssm[slot].clone(), mag[slot].clone()
        for i in range(s, e):
            u = (t[i][:, None] * x[i])[:, :, None] * b[i]
            h = decay[i][:, None, None] * h + u
            m = decay[i][:, None, None] * m + u.abs()
            y[i] = (h * c[i]).sum(-1)
            ymag[i] = (m * c[i].abs()).sum(-1)
        ssm[slot], mag[slot] = h, m
    gate = 1.0
    if d is not None:
        y = y + d.double()[:, None] * x
        ymag = ymag + d.double().abs()[:, None] * x.abs()
    if z is not None:
        gate = z.double() * torch.sigmoid(z.double())
        y = y * gate
        ymag = ymag * gate.abs()
    return y, ssm, ymag, mag


def overflow(dtype):
    """From here on a value rounds to an infinity: the largest number and half its step, which is
    eps 2^e for a number in [2^e, 2^(e + 1)). float16: 65504 + 2^-10 2^15 / 2 = 65520."""
    f = torch.finfo(dtype)
    return f.max + f.eps / 2 * 2.0 ** math.floor(math.log2(f.max))


def close(got, want, tol, what):
    """Within `tol` of `want`, or the infinity that a value within `tol` of it rounds to."""
    edge, got = overflow(got.dtype), got.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    over = (got - want).abs() - tol
    bad = ~((over <= 0) | (got.isinf() & (got.sign() == want.sign()) & (want.abs() + tol >= edge)))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off; worst by {float((got - want).abs().nan_to_num(9e9).max()):.3g}, "
                           f"tolerance there up to {float(tol.max()) if torch.is_tensor(tol) else tol:.3g}")


def scan_tol(want, mag, steps, dtype, pairs=0.0):
    """y or a state against the recurrence: a rounding to the output's type, and float32 sums whose
    roundings (a few a step over `steps` steps) add up like their square root; `pairs`: relative
    rounding of the terms themselves, where a kernel rounds them."""
    return rounding(want, dtype) + ((4 * steps ** 0.5 + 24) * 2.0 ** -23 + pairs) * mag + 1e-30
