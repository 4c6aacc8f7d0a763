"""The Mamba2 layer of the run-of-tokens operators against 64 bits on the values that its 8 bits
stand for: beside the comparison with the float32 layer, whose bounds have to allow for e4m3."""

import pytest
import torch

from hackathon_b200 import config as C
from hackathon_b200 import kernels as K
from hackathon_b200 import weights as Wt
from tests import seqops_ref as R
from tests.test_gpu_seqops_layer import DEV, PromptLayer, off

pytestmark = pytest.mark.gpu

# Relative 2-norms. A state is the product of the operands x and b, each rounded to the activations'
# type by the projection and by the convolution, 2^-9 in bf16: 4 x 2^-9. In float32 the projection's sum
# of 256 products, within 14 x 2^-23 of its terms' magnitudes, which are about 16 times the sum, is the
# largest of some ten such errors: 2^-12. y has c, the gate and its own roundings (S, the state's copy, y)
# besides: twice the state's. Where the second norm's values e4m3, steps of at most 2^-3, move by d, the
# rounded ones move by a step for d / step of them: sqrt(2^-3 d) in the 2-norm.
STATE = {torch.bfloat16: 2.0 ** -7, torch.float32: 2.0 ** -12}
OUT = {t: (2 * d / 8) ** 0.5 for t, d in STATE.items()}


def values(q, scale):
    return q.double() * scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def weight_values(w):
    q, scale = w
    return values(q, scale.repeat_interleave(128, 0)[:q.shape[0]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
@pytest.mark.parametrize("lengths", [[150, 37, 0, 260], [1, 1, 1, 1]], ids=["prompts", "steps"])
def test_layer_on_its_own_8_bit_values(dtype, lengths):
    cfg = C.D2
    sd = Wt.generate(Wt.mamba2_specs("", cfg.hidden_size), seed=4)
    slots, rows = [5, 0, 2, 3], 6
    g = torch.Generator(device=DEV).manual_seed(2)
    u = torch.randn(sum(lengths), cfg.hidden_size, device=DEV, generator=g)
    norm_w = torch.rand(cfg.hidden_size, device=DEV, generator=g) + 0.5
    layer = PromptLayer(cfg, sd, rows, dtype)
    layer.window.copy_(torch.randn(layer.window.shape, device=DEV, generator=g))
    layer.ssm.copy_(torch.randn(layer.ssm.shape, device=DEV, generator=g))
    window, ssm = layer.window.clone(), layer.ssm.clone()
    got, normed = layer.run(u, norm_w, K.SequenceBatch(lengths, slots, state_rows=rows, device=DEV))
    assert K.device_error() == 0

    h = K.rms_norm_fp8(u.to(dtype), norm_w, eps=1e-6)  # the same 8 bits
    p = values(h.q, h.scale) @ weight_values(layer.w_in).T
    inner, bc = layer.inner, layer.bc
    ch, heads = inner + 2 * bc, (cfg.mamba_heads, cfg.mamba_head_size)
    xbc, window, _ = R.conv(window, p[:, :ch], layer.conv_w, layer.conv_b, lengths, slots, True)
    dt = normed.double() @ layer.dt_w.double().T + layer.dt_b.double()
    y, ssm, _, _ = R.scan(ssm, xbc[:, :inner].unflatten(1, heads), xbc[:, inner:inner + bc], xbc[:, inner + bc:], dt, layer.a, lengths, slots,
                          layer.d, p[:, ch:].unflatten(1, heads))
    y = y.flatten(1)
    n = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * layer.norm.double()
    scale = n.abs().unflatten(1, (-1, 128)).amax(-1) / 448
    q = (n / scale.repeat_interleave(128, 1)).float().to(torch.float8_e4m3fn)
    want = values(q, scale) @ weight_values(layer.w_out).T
    for what, mine, ref, tol in (("window", layer.window, window, STATE[dtype]), ("ssm", layer.ssm, ssm, STATE[dtype]), ("out", got, want, OUT[dtype])):
        assert off(mine.cpu(), ref.cpu()) < tol, (what, off(mine.cpu(), ref.cpu()), tol)
