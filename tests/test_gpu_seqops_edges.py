"""The run-of-tokens operators where their contract is easily broken: sequence ends inside a
chunk, plans and extents at their limits, values at the ends of their types."""

import pytest
import torch

from hackathon_b200 import kernels as K
from tests import seqops_ref as R
from tests.test_gpu_seqops import DEV, PAIRS, TYPES, gen, ids, rnd, scan_inputs

pytestmark = pytest.mark.gpu


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
