"""The scan's results of bf16 inputs are as exact as their own rounding lets them be.

Tolerances (fixed from the arithmetic before the first run).  Every factor that the kernels
form themselves enters a product with at most 2^-16 of it lost, and sums are fp32.  A bf16
result is off by its own rounding, whose norm is that of round(want) - want (about 2^-9.3 of
the result's), and by what its factors lost: two of them, 2^-15 of the result, so that the
norm of the whole is at most 1 + 2^-15 / 2^-9.3 = 1.02 times that of the rounding; 1.05 is
asked for.  One rounding of one factor to bf16 (2^-9.3 of it) would make it 1.4.

Gradients of fp32 parameters are sums of such products over tokens, of random sign, rounded
in fp32 only: each product is off by at most 2^-15 of itself (two factors), and the sum of
their errors grows as the sum itself does.  2^-11 of the norm over the heads, sixteen times as
much, leaves room for heads whose sum happens to be small."""
from __future__ import annotations

import pytest
import torch

import moc
from oracle import block_oracle as O
from tests.test_gpu_blocks import BF16, F32, F64, dev, rnd, scan_inputs

pytestmark = pytest.mark.gpu


def slow_inputs(lead, H, P, G, N, par, seed=0):
    """Decays slow enough that what a chunk gets from the ones before it counts as much as its own."""
    ins = scan_inputs(lead, H, P, G, N, BF16, seed=seed, par=par)
    ins["A"] = (-torch.linspace(0.05, 1.0, H)).to(par)
    ins["dt_bias"] = torch.full((H,), -3.0).to(par)
    return ins


def off(got, want):
    return (got.detach().cpu().to(F64) - want).norm()


def own_rounding(want, dtype):
    return (want.to(dtype).to(F64) - want).norm()


SHAPES = [((2, 200), 4, 64, 1, 128), ((1, 300), 6, 33, 3, 100), ((2, 260), 4, 64, 2, 64), ((1, 150), 3, 36, 1, 20),
          ((1, 200), 2, 128, 1, 256), ((1, 130), 2, 80, 1, 130), ((2, 700), 2, 20, 1, 16)]


@pytest.mark.parametrize("lead, H, P, G, N", SHAPES)
def test_outputs(lead, H, P, G, N):
    ins = slow_inputs(lead, H, P, G, N, F32)
    init = rnd(lead[0], H, P, N, seed=20, scale=0.3)
    flat = {k: (v.flatten(0, 1) if v.ndim > 1 else v) for k, v in ins.items()}
    u = O.step_lengths(flat["dt"], flat["dt_bias"], True)
    seqs = O.spans(lead[0] * lead[1], lead[1], None)
    want, fin = O.scan(flat["x"], u, flat["A"], flat["B"], flat["C"], flat["D"], seqs, init=init)
    y, got_fin = moc.selective_scan(**{k: dev(v) for k, v in ins.items()}, cache=dev(init), output_final_state=True)
    assert off(y.flatten(0, 1), want) <= 1.05 * own_rounding(want, BF16)
    assert off(got_fin, fin) <= 2.0 ** -16 * fin.norm()


@pytest.mark.parametrize("lead, H, P, G, N", SHAPES)
def test_gradients(lead, H, P, G, N):
    ins = slow_inputs(lead, H, P, G, N, F32)
    init, dfin = rnd(lead[0], H, P, N, seed=20, scale=0.3), rnd(lead[0], H, P, N, seed=21)
    dy = rnd(*lead, H, P, seed=50, dtype=BF16)
    flat = {k: (v.flatten(0, 1) if v.ndim > 1 else v) for k, v in ins.items()}
    u = O.step_lengths(flat["dt"], flat["dt_bias"], True)
    seqs = O.spans(lead[0] * lead[1], lead[1], None)
    _, (dx, du, dA, dB, dC, dD, dinit, _) = O.scan(flat["x"], u, flat["A"], flat["B"], flat["C"], flat["D"], seqs,
                                                   init=init, dy=dy.flatten(0, 1), dfin=dfin)
    ddt = du * O.sigmoid_of(u, True)
    leaves = {k: dev(v).requires_grad_() for k, v in ins.items()}
    cache = dev(init).requires_grad_()
    y, fin = moc.selective_scan(**leaves, cache=cache, output_final_state=True)
    names = ["x", "dt", "B", "C", "A", "D", "dt_bias"]
    got = torch.autograd.grad([y, fin], [*(leaves[k] for k in names), cache], [dev(dy), dev(dfin)])
    for name, g, want in zip(names, got[:4], (dx, ddt, dB, dC)):
        assert off(g.flatten(0, 1), want) <= 1.05 * own_rounding(want, BF16), name
    for name, g, want in zip(names[4:], got[4:], (dA, dD, ddt.sum(0))):
        assert g.dtype == F32 and off(g, want) <= 2.0 ** -11 * want.norm(), name
    assert off(got[7], dinit) <= 2.0 ** -16 * dinit.norm()
