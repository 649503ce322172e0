"""Calls of the encoder of linear cost's operators that stand beside those of
test_gpu_delta.py: long rows of segments, arrays that autograd's hooks have put
elsewhere, states that a graph has saved, more rows than one launch's axis holds.

Tolerances are those of test_gpu_delta.py with p = 2^-24 for every type: inputs are
exact in their pieces and what is computed from them has three."""

import pytest
import test_gpu_delta as base
import torch

pytestmark = pytest.mark.gpu

TYPES = base.TYPES


@pytest.fixture(autouse=True)
def _digits(monkeypatch):
    for dtype in TYPES:
        monkeypatch.setitem(base.P, dtype, 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv,reverse", [(24, 40, False), (64, 64, True), (128, 128, False)])
def test_many_segments(monkeypatch, dk, dv, reverse, dtype):
    """Twenty-six segments in a row, whose maps go through two buffers or, of 128
    channels, through one; a short chain beside them."""
    from mlcg_amd import ops

    print(f"delta joins {dk} {dv} {dtype}", flush=True)
    c = base._case([64 * 25 + 5, 130], 2, 1, dk, dv, dtype, keep=True, state=True)
    c["reverse"] = reverse
    c["decay"] *= 0.02  # the first segments still count in the last
    monkeypatch.setattr(ops, "_delta_segment_tiles", lambda *a: 1)
    first = base._check(c)
    for name, t in base._run(c).items():
        assert torch.equal(t, first[name]), name
