"""A Mamba2 layer over symbols' histories, built from the run-of-tokens operators as a
program uses them, against the layer engine stepped token by token with float32 weights;
then the states are handed to the layer engine, which goes on from them."""

import numpy as np
import pytest
import torch

from hackathon_b200 import config as C
from hackathon_b200 import kernels as K
from hackathon_b200 import weights as Wt
from hackathon_b200.engine import LayerEngine

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


class PromptLayer:
    """The layer's weights in 8 bits and its state tables."""

    def __init__(self, cfg, sd, rows, dtype):
        self.cfg, self.dtype = cfg, dtype
        t = {k: torch.from_numpy(v).to(DEV) for k, v in sd.items()}
        self.inner, self.bc = cfg.mamba_inner, cfg.mamba_bc_size
        order = ("input_proj", "b_proj", "c_proj", "z_proj")
        self.w_in = K.quantize_fp8_weight(torch.cat([t[f"{n}.weight"] for n in order]))
        self.w_out = K.quantize_fp8_weight(t["out_proj.weight"])
        convs = ("input_conv", "b_conv", "c_conv")
        self.conv_w = torch.cat([t[f"{n}.conv.weight"][:, 0] for n in convs]).contiguous()
        self.conv_b = torch.cat([t[f"{n}.conv.bias"] for n in convs])
        self.dt_w, self.dt_b, self.a, self.d, self.norm = t["dt_proj.weight"], t["dt_proj.bias"], t["a"], t["d"], t["norm.weight"]
        ch = self.inner + 2 * self.bc
        self.window = torch.zeros(rows, ch, 3, device=DEV)
        self.ssm = torch.zeros(rows, cfg.mamba_heads, cfg.mamba_head_size, self.bc, device=DEV)

    def run(self, u, norm_w, batch):
        """norm -> projection -> convolution -> scan -> norm -> projection."""
        h = K.rms_norm_fp8(u.to(self.dtype), norm_w, eps=1e-6, keep_norm=True)
        p = K.fp8_linear(h.q, h.scale, *self.w_in, out_dtype=self.dtype)
        ch = self.inner + 2 * self.bc
        xbc = K.causal_conv(self.window, p[:, :ch], self.conv_w, self.conv_b, batch, silu=True)
        dt = K.cast_linear(h.normed.float(), self.dt_w, self.dt_b)
        heads = (self.cfg.mamba_heads, self.cfg.mamba_head_size)
        y = K.mamba2_scan(self.ssm, xbc[:, :self.inner].unflatten(1, heads), xbc[:, self.inner:self.inner + self.bc],
                          xbc[:, self.inner + self.bc:], dt, self.a, batch, d=self.d, z=p[:, ch:].unflatten(1, heads))
        o = K.rms_norm_fp8(y.flatten(1), self.norm, eps=1e-5)
        return K.fp8_linear(o.q, o.scale, *self.w_out), h.normed

    def leaves(self, row):
        i, b = self.inner, self.inner + self.bc
        w = self.window[row].cpu().numpy()
        return [w[:i], w[i:b], w[b:], self.ssm[row].cpu().numpy()]


def off(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.linalg.norm(a - b) / np.linalg.norm(b)


# Ten e4m3 roundings meet in an output: activation and weight of x, b, c, z and of the output
# projection. Each is within 2^-4 of its value, about 2^-4 / sqrt(3) in the mean square, and they are
# independent: sqrt(10) 2^-4 / sqrt(3) = 0.114. Twice that bounds the 2-norm; a state holds x and b (four).
OUT, STATE = 0.23, 0.15


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
def test_prompt_layer_against_single_steps_and_handover(dtype):
    cfg = C.D2
    sd = Wt.generate(Wt.mamba2_specs("", cfg.hidden_size), seed=3)
    sd["a"] = (sd["a"] * 0.1).astype(np.float32)  # memories of tens of tokens
    lengths, slots, rows = [150, 37, 0, 260], [5, 0, 2, 3], 6
    batch = K.SequenceBatch(lengths, slots, state_rows=rows, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    u = torch.randn(sum(lengths), cfg.hidden_size, device=DEV, generator=g)
    norm_w = torch.rand(cfg.hidden_size, device=DEV, generator=g) + 0.5
    layer = PromptLayer(cfg, sd, rows, dtype)
    got, normed = layer.run(u, norm_w, batch)
    assert K.device_error() == 0

    eng = LayerEngine("mamba2", cfg, sd, linear_dtype="fp32", capacity=rows, max_batch=1)
    want = torch.empty_like(got)
    at = 0
    for n, slot in zip(lengths, slots):
        st = torch.tensor([slot], dtype=torch.int32, device=DEV)
        for i in range(at, at + n):
            eng.step_device(st, normed[i:i + 1].float().contiguous(), want[i:i + 1])
        at += n
    torch.cuda.synchronize()
    assert off(got.cpu(), want.cpu()) < OUT
    for slot in (5, 0, 3):
        mine, theirs = layer.leaves(slot), eng.read_slot(slot)
        for a, b in zip(mine, theirs):
            assert a.shape == b.shape and off(a, b) < STATE
    assert not layer.ssm[[1, 2, 4]].any() and not layer.window[[1, 2, 4]].any(), "rows of no token stay as they were"

    # handover: the layer engine goes on from the prompts' states, and so do single tokens here
    x = torch.randn(3, cfg.hidden_size, device=DEV, generator=g)
    for slot in (5, 0, 3):
        eng.write_slot(slot, layer.leaves(slot))
    got, normed = layer.run(x, norm_w, K.SequenceBatch([1, 1, 1], [5, 0, 3], state_rows=rows, device=DEV))
    want = torch.empty_like(got)
    for i, slot in enumerate((5, 0, 3)):
        eng.step_device(torch.tensor([slot], dtype=torch.int32, device=DEV), normed[i:i + 1].float().contiguous(), want[i:i + 1])
    torch.cuda.synchronize()
    assert off(got.cpu(), want.cpu()) < OUT
    eng.close()
