"""The fused state steps, with the reference's operator API.

Drop-in for model/kernels.py's ``mlstm_step``, ``retnet_step`` and
``mamba2_step`` (model/kernels.py:346-401): same arguments, same semantics, same
refusals. The state is updated IN PLACE on active rows (idle rows stay bit
for bit), the returned output is a fresh contiguous float32 tensor with zeros on
idle rows, and ``mask=None`` means every row is active. Operands may be strided
views (they are made contiguous); the state may not, because it is written in
place. Errors raise AssertionError, like the reference's wrappers
(model/kernels.py:85-122). The computation is libb2e.so's CUDA kernels on the
current torch stream; there is no CPU path.

Beside them, the operators of a Mamba2 layer over a whole run of tokens (a
symbol's history in one call instead of one call a token), which the reference
does not have: ``rms_norm_fp8``, ``fp8_linear`` with its quantisers,
``causal_conv`` and ``mamba2_scan``, the last two over the packed sequences of a
``SequenceBatch``. They serve: nothing here has a gradient.
"""

from __future__ import annotations

import ctypes as C
import operator
import struct
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib


def _small(t: torch.Tensor, shape: tuple, name: str, device) -> torch.Tensor:
    # model/kernels.py:85-98: fp32 asserted, never cast; shape and device checked.
    assert t.dtype == torch.float32, f"{name} must be fp32, got {t.dtype}"
    assert tuple(t.shape) == shape, f"{name} must be {shape}, got {tuple(t.shape)}"
    assert t.device == device, f"{name} must be on {device}, it is on {t.device}"
    return t.contiguous()


def _mask_u8(mask, batch: int, device):
    # model/kernels.py:101-113; the contiguous copy also packs a strided mask.
    if mask is None:
        return None
    assert mask.dtype == torch.bool, f"mask must be bool, got {mask.dtype}"
    assert tuple(mask.shape) == (batch,), f"mask must be ({batch},), got {tuple(mask.shape)}"
    assert mask.device == device, f"mask must be on {device}, it is on {mask.device}"
    return mask.to(torch.uint8).contiguous()


def _state_ok(state: torch.Tensor, name: str) -> None:
    # model/kernels.py:116-121: written in place, so never copied.
    assert state.dtype == torch.float32, f"{name} must be fp32, got {state.dtype}"
    assert state.is_contiguous(), f"{name} must be contiguous, it is written in place"
    assert state.dim() == 4, f"{name} must be 4-D, got {tuple(state.shape)}"
    assert state.is_cuda, f"{name} must be a CUDA tensor (there is no CPU path)"


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream(device) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def mlstm_step(cell, q, k, v, i_gate, f_gate, mask):
    """cell <- f*cell + i*(k outer v) on active rows; return sum_h q*cell_new."""
    _state_ok(cell, "cell")
    b, n, sh, sk = cell.shape
    dev = cell.device
    q = _small(q, (b, n, sh), "q", dev)
    k = _small(k, (b, n, sh), "k", dev)
    v = _small(v, (b, n, sk), "v", dev)
    i_gate = _small(i_gate, (b, n), "i_gate", dev)
    f_gate = _small(f_gate, (b, n), "f_gate", dev)
    m = _mask_u8(mask, b, dev)
    out = torch.empty(b, n, sk, dtype=torch.float32, device=dev)
    if b:
        _lib.check(_lib.lib().b2e_mlstm_step(_ptr(cell), _ptr(q), _ptr(k), _ptr(v), _ptr(i_gate), _ptr(f_gate),
                                             _ptr(m), b, n, sh, sk, _ptr(out), _stream(dev)))
    return out


def retnet_step(state, k_rope, v, q_scaled, decay, mask):
    """state <- decay*state + (k outer v) on active rows; return sum_h q_scaled*state_new."""
    _state_ok(state, "state")
    b, n, sh, sk = state.shape
    dev = state.device
    k_rope = _small(k_rope, (b, n, sh), "k_rope", dev)
    v = _small(v, (b, n, sk), "v", dev)
    q_scaled = _small(q_scaled, (b, n, sh), "q_scaled", dev)
    decay = _small(decay, (n,), "decay", dev)
    m = _mask_u8(mask, b, dev)
    out = torch.empty(b, n, sk, dtype=torch.float32, device=dev)
    if b:
        _lib.check(_lib.lib().b2e_retnet_step(_ptr(state), _ptr(k_rope), _ptr(v), _ptr(q_scaled), _ptr(decay),
                                              _ptr(m), b, n, sh, sk, _ptr(out), _stream(dev)))
    return out


def mamba2_step(ssm, x, b, c, dt, decay, mask):
    """ssm <- decay*ssm + dt*(b outer x) on active rows; return sum_c c*ssm_new."""
    _state_ok(ssm, "ssm")
    bs, n, sh, sc = ssm.shape
    dev = ssm.device
    x = _small(x, (bs, n, sh), "x", dev)
    b = _small(b, (bs, sc), "b", dev)
    c = _small(c, (bs, sc), "c", dev)
    dt = _small(dt, (bs, n), "dt", dev)
    decay = _small(decay, (bs, n), "decay", dev)
    m = _mask_u8(mask, bs, dev)
    out = torch.empty(bs, n, sh, dtype=torch.float32, device=dev)
    if bs:
        _lib.check(_lib.lib().b2e_mamba2_step(_ptr(ssm), _ptr(x), _ptr(b), _ptr(c), _ptr(dt), _ptr(decay),
                                              _ptr(m), bs, n, sh, sc, _ptr(out), _stream(dev)))
    return out


_TORCH_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def set_state_kernel_waves(waves: int) -> int:
    """Grid of the state kernels when they stream alone (this module's three steps
    and the layer engine): waves > 0 short CTAs of a few items, ~waves waves of two
    CTAs per SM (default 8, the fastest alone); 0 one persistent CTA per SM, the
    grid the ensemble engine's step uses. Results are identical bit for bit.
    Process-wide; returns the previous value (b2e_set_state_kernel_waves)."""
    prev = C.c_int32()
    _lib.check(_lib.lib().b2e_set_state_kernel_waves(int(waves), C.byref(prev)))
    return prev.value


def cast_linear(x, weight, bias=None, relu: bool = False, err=None):
    """CastLinear.forward (example_model.py:92-95) / nn.Linear on the GPU.

    ``weight`` (out, in) is float32, bfloat16 or float16. With a low-precision
    weight, x is rounded to its type, products accumulate in float32, the bias
    (same type as the weight) is added and the result is rounded to the weight's
    type before widening: exactly CastLinear. Returns a new float32 tensor.
    ``err`` is an optional int32 CUDA tensor of one element that receives an error
    code if the tensor-core kernel times out; without it the tensor-core kernel
    is not used.
    """
    assert weight.is_cuda and weight.dim() == 2 and weight.is_contiguous()
    wt = _TORCH_DTYPES[weight.dtype]
    assert x.dtype in (torch.float32, weight.dtype), f"x must be fp32 or {weight.dtype}, got {x.dtype}"
    assert x.device == weight.device and x.dim() == 2 and x.shape[1] == weight.shape[1]
    x = x.contiguous()
    if bias is not None:
        assert bias.dtype == weight.dtype and bias.shape == (weight.shape[0],)
        bias = bias.contiguous()
    y = torch.empty(x.shape[0], weight.shape[0], dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().b2e_linear(_ptr(x), _TORCH_DTYPES[x.dtype], x.shape[0], x.shape[1], _ptr(weight), wt,
                                     _ptr(bias), weight.shape[0], int(relu), _ptr(y), _ptr(err), _stream(x.device)))
    return y


# ------------------------------------------------------------ runs of tokens

MAX_EXTENT = 2 ** 31 - 1024  # rows, columns, tokens or channels of a call (the kernels' indices are 32-bit, their offsets are not)
FP8_GROUP = 128  # columns of a row (rows and columns of a weight's block) that share a scale


def _integers(values, name: str) -> list:
    try:
        return [operator.index(v) for v in values]
    except TypeError:
        raise AssertionError(f"{name} must be integers") from None


class SequenceBatch:
    """Plan of a packed batch of sequences, kept for every call on that batch.

    Sequence i has ``lengths[i]`` tokens (zero: its state stays as it is), packed
    one after the other in the operands' rows, and lives in row ``slots[i]`` of the
    state tables (default: row i). Everything is checked here, on the host: lengths
    are not negative, slots distinct and inside the ``state_rows`` rows of the
    smallest table the plan is used with (default: up to the highest slot). The
    plan's device arrays belong to ``device``; keep the plan until the work that
    uses it is done.
    """

    def __init__(self, lengths: Sequence[int], slots: Optional[Sequence[int]] = None, *,
                 state_rows: Optional[int] = None, device=None):
        lengths = _integers(lengths, "lengths")
        assert all(n >= 0 for n in lengths), "lengths must not be negative"
        self.tokens = sum(lengths)
        assert self.tokens <= MAX_EXTENT, "a batch has at most 2^31 - 1024 tokens"
        assert len(lengths) <= 2 ** 30, "a batch has at most 2^30 sequences"
        if slots is not None:
            slots = _integers(slots, "slots")
            assert len(slots) == len(lengths), f"{len(slots)} slots for {len(lengths)} sequences"
            assert len(set(slots)) == len(slots), "slots must be distinct"
            assert all(s >= 0 for s in slots), "slots must not be negative"
        need = (max(slots) + 1 if slots else 0) if slots is not None else len(lengths)
        self.state_rows = need if state_rows is None else _integers([state_rows], "state_rows")[0]
        assert need <= self.state_rows < 2 ** 31, f"slots reach row {need - 1} of {self.state_rows} state rows"
        self.lengths = tuple(lengths)
        self.longest = max(lengths, default=0)
        self.slots = tuple(range(len(lengths))) if slots is None else tuple(slots)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        single = all(n == 1 for n in lengths)  # one token a sequence: the step kernels, which need no starts
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        order = [] if single else sorted(range(len(lengths)), key=lambda i: -lengths[i])  # longest first
        host = ([] if single else starts) + order + ([] if slots is None else slots)
        self._arrays = torch.tensor(host, dtype=torch.int32).to(self.device)
        at = self._arrays.data_ptr()
        order_at = at + 4 * len(starts)
        slots_at = at if single else order_at + 4 * len(order)
        self._c = _lib.SequencesC(None if single else at, None if slots is None else slots_at, None if single else order_at,
                                  len(lengths), self.tokens, self.state_rows, self.longest)

    def __len__(self) -> int:
        return len(self.lengths)


class NormFp8(NamedTuple):
    """``rms_norm_fp8``'s results: e4m3 values, their scales (rows, groups of 128
    columns), the sum with the residual and the normed row (None where not asked)."""

    q: torch.Tensor
    scale: torch.Tensor
    total: Optional[torch.Tensor]
    normed: Optional[torch.Tensor]


def _call(name: str, device, *args) -> None:
    """One C-ABI call on `device`'s current stream."""
    fn = getattr(_lib.lib(), name)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _extents(*sizes: int) -> None:
    assert max(sizes) <= MAX_EXTENT, f"sizes are at most 2^31 - 1024, got {max(sizes)}"


def _at(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor):
    """A 2-D operand whose rows are contiguous (copied if they are not) and its row stride."""
    n, c = t.shape
    if (c > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < c):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else c)


def _rows8(t: torch.Tensor):
    """The same for e4m3 rows, which start on 16-byte boundaries."""
    n, k = t.shape
    if (k > 1 and t.stride(1) != 1) or t.data_ptr() % 16 or (n > 1 and (t.stride(0) < k or t.stride(0) % 16)):
        wide = torch.empty(n, -(-k // 16) * 16, dtype=t.dtype, device=t.device)
        wide[:, :k].copy_(t)
        t = wide[:, :k]
    return t, (t.stride(0) if n > 1 else -(-k // 16) * 16)


def _empty8(rows: int, cols: int, device):
    """Empty e4m3 rows, padded so that each starts on a 16-byte boundary, and scales' columns."""
    wide = torch.empty(rows, -(-cols // 16) * 16, dtype=torch.float8_e4m3fn, device=device)
    return wide[:, :cols] if cols % 16 else wide, -(-cols // FP8_GROUP)


def _float(t: torch.Tensor, name: str) -> int:
    assert t.dtype in _TORCH_DTYPES, f"{name} must be float32, bfloat16 or float16, got {t.dtype}"
    return _TORCH_DTYPES[t.dtype]


def _vector(t, n: int, name: str, device):
    """An optional float32 vector of n values."""
    if t is None:
        return None
    assert t.dtype == torch.float32 and t.shape == (n,), f"{name} must be float32 ({n},), got {t.dtype} {tuple(t.shape)}"
    assert t.device == device, f"{name} must be on {device}, it is on {t.device}"
    return t if t.stride(0) == 1 or n == 1 else t.contiguous()


def _operand(t: torch.Tensor, dtype, shape, name: str, device) -> None:
    assert t.dtype == dtype and t.shape == shape, f"{name} must be {dtype} {shape}, got {t.dtype} {tuple(t.shape)}"
    assert t.device == device, f"{name} must be on {device}, it is on {t.device}"


def _head_rows(t: torch.Tensor):
    """A 3-D operand (rows, heads, size) whose rows are contiguous (copied if they are not) and its row stride."""
    n, h, p = t.shape
    a, b, c = t.stride()
    if (c == 1 or p == 1) and (b == p or h == 1) and (a >= h * p or n <= 1):
        return t, (a if n > 1 else h * p)
    return t.contiguous(), h * p


def _on_gpu(t: torch.Tensor, name: str) -> None:
    assert t.is_cuda, f"{name} must be a CUDA tensor (there is no CPU path)"


def rms_norm_fp8(x, weight=None, residual=None, eps: float = 1e-5, keep_norm: bool = False) -> NormFp8:
    """RMS norm of ``x + residual`` (rows, cols) with an 8-bit output for ``fp8_linear``.

    v = x + residual; n = v / sqrt(mean(v^2) + eps) * weight, all in float32; each 128
    columns of a row get scale = max(max|n| / 448, 2^-100) and q = e4m3(n / scale).
    ``total`` is v in the residual's type (x's or float32), the next layer's residual;
    ``keep_norm`` adds n in x's type, for the projections that stay in float32. As the
    formula has it, a NaN makes its whole row NaN; an infinity makes its group of 128 NaN
    and the rest of its row 0. Squares may leave float32's range.
    """
    assert x.dim() == 2 and x.shape[1] > 0, f"x must be (rows, cols), got {tuple(x.shape)}"
    xt = _float(x, "x")
    rows, cols = x.shape
    _extents(rows, cols)
    rt, ldr = xt, 0
    if residual is not None:
        assert residual.shape == x.shape, f"residual must be {tuple(x.shape)}, got {tuple(residual.shape)}"
        assert residual.dtype in (x.dtype, torch.float32), f"residual must be {x.dtype} or float32, got {residual.dtype}"
        assert residual.device == x.device, f"residual must be on {x.device}, it is on {residual.device}"
        rt = _TORCH_DTYPES[residual.dtype]
        residual, ldr = _rows(residual)
    weight = _vector(weight, cols, "weight", x.device)
    _on_gpu(x, "x")
    x, ldx = _rows(x)
    q, groups = _empty8(rows, cols, x.device)
    scale = torch.empty(rows, groups, dtype=torch.float32, device=x.device)
    total = None if residual is None else torch.empty(rows, cols, dtype=residual.dtype, device=x.device)
    normed = torch.empty(rows, cols, dtype=x.dtype, device=x.device) if keep_norm else None
    if rows:
        _call("b2e_rms_norm_fp8", x.device, _at(x), xt, ldx, _at(residual), rt, ldr, _at(weight), eps, rows, cols, _at(q),
              -(-cols // 16) * 16, _at(scale), _at(total), _at(normed))
    return NormFp8(q, scale, total, normed)


def quantize_fp8(x):
    """e4m3 values of x (rows, cols) and the scale of each 128 columns of a row, (rows, ceil(cols / 128)).

    As ``rms_norm_fp8`` has them of n. A NaN makes its group of 128 NaN; so does an infinity."""
    assert x.dim() == 2 and x.shape[1] > 0, f"x must be (rows, cols), got {tuple(x.shape)}"
    xt = _float(x, "x")
    rows, cols = x.shape
    _extents(rows, cols)
    _on_gpu(x, "x")
    x, ldx = _rows(x)
    q, groups = _empty8(rows, cols, x.device)
    scale = torch.empty(rows, groups, dtype=torch.float32, device=x.device)
    if rows:
        _call("b2e_quantize_fp8", x.device, _at(x), xt, ldx, rows, cols, _at(q), -(-cols // 16) * 16, _at(scale))
    return q, scale


def quantize_fp8_weight(weight):
    """e4m3 values of a weight (out, in) and the scale of each 128 x 128 block, (ceil(out / 128), ceil(in / 128))."""
    assert weight.dim() == 2 and weight.numel() > 0, f"weight must be (out, in), got {tuple(weight.shape)}"
    wt = _float(weight, "weight")
    rows, cols = weight.shape
    _extents(rows, cols)
    _on_gpu(weight, "weight")
    weight, ldw = _rows(weight)
    q, groups = _empty8(rows, cols, weight.device)
    scale = torch.empty(-(-rows // FP8_GROUP), groups, dtype=torch.float32, device=weight.device)
    _call("b2e_quantize_fp8_weight", weight.device, _at(weight), wt, ldw, rows, cols, _at(q), -(-cols // 16) * 16, _at(scale))
    return q, scale


def fp8_linear(q, scale, wq, wscale, bias=None, relu: bool = False, out_dtype=torch.float32):
    """The projection of 8-bit rows by an 8-bit weight, beside ``cast_linear``.

    ``q`` (m, k) with ``scale`` (m, ceil(k / 128)) from ``rms_norm_fp8`` or
    ``quantize_fp8``; ``wq`` (n, k) with ``wscale`` (ceil(n / 128), ceil(k / 128)) from
    ``quantize_fp8_weight``; ``bias`` float32 (n,). Each group's 128 products are summed
    and the groups' sums scaled and added in float32; the result is rounded once to
    ``out_dtype``. Operands whose rows do not start on 16-byte boundaries are copied.
    """
    assert q.dim() == 2 and wq.dim() == 2 and q.shape[1] == wq.shape[1] and wq.numel() > 0, \
        f"q (m, k) and wq (n, k) expected, got {tuple(q.shape)} and {tuple(wq.shape)}"
    assert q.dtype == wq.dtype == torch.float8_e4m3fn, f"q and wq must be float8_e4m3fn, got {q.dtype} and {wq.dtype}"
    m, k = q.shape
    n, g = wq.shape[0], -(-k // FP8_GROUP)
    _extents(m, n, k)
    dev = q.device
    _operand(scale, torch.float32, (m, g), "scale", dev)
    _operand(wscale, torch.float32, (-(-n // FP8_GROUP), g), "wscale", dev)
    assert wq.device == dev, f"wq must be on {dev}, it is on {wq.device}"
    assert out_dtype in _TORCH_DTYPES, f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}"
    bias = _vector(bias, n, "bias", dev)
    _on_gpu(q, "q")
    y = torch.empty(m, n, dtype=out_dtype, device=dev)
    if m:
        q, ldq = _rows8(q)
        wq, ldw = _rows8(wq)
        scale, wscale = scale.contiguous(), wscale.contiguous()
        _call("b2e_fp8_linear", dev, _at(q), ldq, _at(scale), m, k, _at(wq), ldw, _at(wscale), n, _at(bias), int(relu), _at(y),
              _TORCH_DTYPES[out_dtype], n)
    return y


def _plan(seqs: Optional[SequenceBatch], rows: int, table: torch.Tensor, name: str):
    """(C plan, tokens) of a call over `rows` operand rows and a state table."""
    if seqs is None:
        assert rows == table.shape[0], f"without a SequenceBatch every row of {name} steps: {rows} rows for {table.shape[0]}"
        return None, rows
    assert seqs.tokens <= rows, f"the batch has {seqs.tokens} tokens, the operands {rows} rows"
    assert seqs.state_rows <= table.shape[0], f"the batch's slots need {seqs.state_rows} state rows, {name} has {table.shape[0]}"
    assert seqs.device == table.device, f"the batch is on {seqs.device}, {name} on {table.device}"
    return C.byref(seqs._c), seqs.tokens


def _out(like, rows: int, tokens: int):
    """An output of the operands' shape; rows of no sequence are zero."""
    y = torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if rows > tokens:
        y[tokens:].zero_()
    return y


def causal_conv(window, x, weight, bias=None, seqs: Optional[SequenceBatch] = None, silu: bool = False):
    """CausalConv1d (model/modules.py:37-41) over every token of packed sequences.

    ``window`` (state rows, channels, taps - 1) float32 holds each sequence's last inputs
    and is updated IN PLACE (rows of no sequence, and of empty ones, stay bit for bit);
    ``x`` (rows, channels); ``weight`` (channels, taps), 2 to 4 taps, and ``bias`` float32.
    y[t] = sum_j weight[j] v[t + j] + bias over v = window ++ sequence, with SiLU if asked,
    rounded once to x's type. Without ``seqs`` each row of x is one token of that row of
    ``window``. Rows of x behind the batch's tokens are not read and give zeros.
    """
    assert window.dim() == 3 and 1 <= window.shape[2] <= 3, f"window must be (rows, channels, 1..3), got {tuple(window.shape)}"
    assert window.dtype == torch.float32, f"window must be fp32, got {window.dtype}"
    assert window.is_contiguous(), "window must be contiguous, it is written in place"
    ch, taps, dev = window.shape[1], window.shape[2] + 1, window.device
    assert ch > 0 and x.dim() == 2 and x.shape[1] == ch, f"x must be (rows, {ch}), got {tuple(x.shape)}"
    xt = _float(x, "x")
    assert x.device == dev, f"x must be on {dev}, it is on {x.device}"
    _operand(weight, torch.float32, (ch, taps), "weight", dev)
    bias = _vector(bias, ch, "bias", dev)
    rows = x.shape[0]
    _extents(rows, ch)
    plan, tokens = _plan(seqs, rows, window, "window")
    _on_gpu(window, "window")
    y = _out(x, rows, tokens)
    if tokens:
        x, ldx = _rows(x)
        weight = weight.contiguous()
        _call("b2e_causal_conv", dev, plan, _at(window), _at(x), xt, ldx, rows, ch, _at(weight), _at(bias), taps, int(silu),
              _at(y), ch)
    return y


_SCAN_ARGS = struct.Struct("9Q6q6i")
assert _SCAN_ARGS.size == C.sizeof(_lib.ScanArgsC)


def mamba2_scan(ssm, x, b, c, dt, a, seqs: Optional[SequenceBatch] = None, d=None, z=None, softplus: bool = True):
    """Mamba2's recurrence (model/mamba2.py:128-165) over every token of packed sequences.

    t = softplus(dt) (dt itself without ``softplus``); ssm <- exp(a t) ssm + t (b outer x);
    y = (sum_c c * ssm + d x) * silu(z). ``ssm`` (state rows, heads, size, state) float32 is
    updated IN PLACE; rows of no sequence, and of empty ones, stay bit for bit. ``x``, ``z``
    (rows, heads, size), ``b``, ``c`` (rows, state), state up to 256, all of one type; ``dt``
    (rows, heads), ``a`` and ``d`` (heads,) float32. Without ``seqs`` each row is one token of
    that row of ``ssm``, as in ``mamba2_step``. Rows behind the batch's tokens are not read and
    give zeros.

    The state and all sums are float32 and y is rounded once to x's type. In bf16 prompts with
    heads of 64 and states of 64 or 128, which run in chunks of 128 tokens on the tensor cores,
    two operands of y are rounded to bf16 as well: the weights of a chunk's pairs of tokens and
    the copy of the state that c multiplies. A term of y is then within 2^-8 of its value, and y
    about 1.35 times as far from the formula as its own rounding takes it; the state is not
    affected.

    A value that is not finite stays in its own sequence and reaches no earlier token; of x, it
    makes its row's y NaN from its token on; bf16 prompts may have NaN where the formula has an
    infinity. ``a`` is meant to be at most zero: with one above, those chunks overflow where the
    sum of a t over one passes 88. Prompts of other types hold the state relative to the product
    of its decays, which leaves t x b a headroom of 2^12 below float32's largest.
    """
    _scan_state_ok(ssm)
    nrows, h, p, n = ssm.shape
    dev = ssm.device
    assert x.dim() == 3, f"x must be (rows, {h}, {p}), got {tuple(x.shape)}"
    rows, dtype = x.shape[0], x.dtype
    _extents(rows, h * p)
    xt = _float(x, "x")
    _operand(x, dtype, (rows, h, p), "x", dev)
    if z is not None:
        _operand(z, dtype, (rows, h, p), "z", dev)
    _operand(b, dtype, (rows, n), "b", dev)
    _operand(c, dtype, (rows, n), "c", dev)
    _operand(dt, torch.float32, (rows, h), "dt", dev)
    assert a is not None, "a must be given"
    a, d = _vector(a, h, "a", dev), _vector(d, h, "d", dev)
    plan, tokens = _plan(seqs, rows, ssm, "ssm")
    _on_gpu(ssm, "ssm")
    y = _out(x, rows, tokens)
    if tokens:
        x, ldx = _head_rows(x)
        z, ldz = (None, 0) if z is None else _head_rows(z)
        (b, ldb), (c, ldc), (dt, lddt) = _rows(b), _rows(c), _rows(dt)
        # b2e_scan_args, packed (a ctypes structure takes as long as the launch)
        args = _SCAN_ARGS.pack(ssm.data_ptr(), x.data_ptr(), b.data_ptr(), c.data_ptr(), dt.data_ptr(), a.data_ptr(),
                               0 if d is None else d.data_ptr(), 0 if z is None else z.data_ptr(), y.data_ptr(),
                               ldx, ldb, ldc, lddt, ldz, h * p, rows, h, p, n, xt, softplus)
        work, size = None, 0
        if seqs is not None and seqs.longest > 1:
            need = C.c_int64()
            _lib.check(_lib.lib().b2e_mamba2_scan_workspace(plan, args, C.byref(need)))
            size = need.value
            work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _call("b2e_mamba2_scan", dev, plan, args, _at(work), size)
    return y


def _scan_state_ok(ssm: torch.Tensor) -> None:
    assert ssm.dtype == torch.float32, f"ssm must be fp32, got {ssm.dtype}"
    assert ssm.dim() == 4 and min(ssm.shape[1:]) > 0, f"ssm must be (rows, heads, size, state), got {tuple(ssm.shape)}"
    assert ssm.is_contiguous(), "ssm must be contiguous, it is written in place"
    assert ssm.shape[3] <= 256, f"a state has at most 256 columns, got {ssm.shape[3]}"
    assert ssm.shape[0] == 0 or not ssm.is_cuda or ssm.data_ptr() % 16 == 0 or ssm.shape[3] % 4, "ssm must start on a 16-byte boundary"


def device_error(device=None) -> int:
    """Error word of this module's run-of-tokens operators on a device (b2e_seqops_device_error):
    0, or the code of a bounded wait that ran out. Waits for the device, reads and clears it."""
    code = C.c_int32()
    with torch.cuda.device(device):
        _lib.check(_lib.lib().b2e_seqops_device_error(C.byref(code)))
    return code.value
