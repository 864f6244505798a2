"""fp32 values near the top of their range in the scan.  A value from 0x1.ffp127 on (3.396e38) is
finite, but rounds to an infinity in bf16, whose planes the matrix products are formed from.

Tolerances as in tests/test_gpu_blocks.py: k fp32 roundings of the sum over absolute values."""
from __future__ import annotations

import pytest
import torch

import moc
from oracle import block_oracle as O
from tests.test_gpu_blocks import F32, F64, dev, near, rnd, scan_inputs

pytestmark = pytest.mark.gpu
TOP = torch.finfo(F32).max


@pytest.mark.parametrize("value", [TOP, -TOP, 3.397e38, 3.3895e38, 2.0 ** 127])
@pytest.mark.parametrize("which", ["x", "B", "C"])
def test_values_near_the_top_are_finite(which, value):
    """One such value among ordinary ones, with what multiplies it small enough that results are finite."""
    ins = scan_inputs((2, 140), 2, 16, 1, 16, F32)
    clean = moc.selective_scan(**{k: dev(v) for k, v in ins.items()})[0]
    ins["B"] *= 2.0 ** -30
    ins["C"] *= 2.0 ** -30
    if which != "x":
        ins["x"] *= 2.0 ** -30
    ins["D"] *= 2.0 ** -30
    small = moc.selective_scan(**{k: dev(v) for k, v in ins.items()})[0]
    t = ins[which].clone()
    t[(0, 70, 1, 3) if which == "x" else (0, 70, 0, 3)] = value
    ins[which] = t
    y, fin = moc.selective_scan(**{k: dev(v) for k, v in ins.items()}, output_final_state=True)
    assert clean.isfinite().all()
    assert torch.equal(y[1], small[1]) and torch.equal(y[0, :70], small[0, :70])
    flat = {k: (v.flatten(0, 1) if v.ndim > 1 else v) for k, v in ins.items()}
    u = O.step_lengths(flat["dt"], flat["dt_bias"], True)
    seqs = O.spans(280, 140, None)
    want, want_fin = O.scan(flat["x"], u, flat["A"], flat["B"], flat["C"], flat["D"], seqs)
    ab = lambda t: t.to(F64).abs()  # noqa: E731
    ya, fa = O.scan(ab(flat["x"]), u, flat["A"], ab(flat["B"]), ab(flat["C"]), ab(flat["D"]), seqs)
    near("y", y.flatten(0, 1), want, ya, 16 + 140 + 384)
    near("state", fin, want_fin, fa, 16 + 140 + 384)


def test_gradients_near_the_top():
    """dy with such a value: dx, dC of finite size against the oracle."""
    ins = scan_inputs((1, 70), 2, 16, 1, 16, F32)
    for k in ("x", "B", "C", "D"):
        ins[k] *= 2.0 ** -30
    dy = rnd(1, 70, 2, 16, seed=9)
    dy[0, 40, 1, 3] = TOP
    flat = {k: (v.flatten(0, 1) if v.ndim > 1 else v) for k, v in ins.items()}
    u = O.step_lengths(flat["dt"], flat["dt_bias"], True)
    _, g = O.scan(flat["x"], u, flat["A"], flat["B"], flat["C"], flat["D"], [(0, 70)], dy=dy[0])
    ab = lambda t: t.to(F64).abs()  # noqa: E731
    _, ga = O.scan(ab(flat["x"]), u, flat["A"], ab(flat["B"]), ab(flat["C"]), ab(flat["D"]), [(0, 70)], dy=ab(dy[0]))
    leaves = {k: dev(v).requires_grad_() for k, v in ins.items()}
    y, _ = moc.selective_scan(**leaves)
    dx, dB, dC = torch.autograd.grad(y, [leaves[k] for k in ("x", "B", "C")], dev(dy))
    k = 2 * (16 + 70 + 384)
    for name, got, want, size in (("dx", dx, g[0], ga[0]), ("dB", dB, g[3], ga[3]), ("dC", dC, g[4], ga[4])):
        near(name, got.flatten(0, 1), want, size, k + 2)
