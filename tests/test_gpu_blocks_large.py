"""Sizes of the operators next to the MoC layers that pass what a grid counts.

Tolerances (fixed from the arithmetic before the first run) stand with the checks."""
from __future__ import annotations

import pytest
import torch

import moc
from tests.test_gpu_blocks import BF16, DEV, F32, F64

pytestmark = pytest.mark.gpu


def _random(*shape, seed):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed), dtype=BF16)


def test_norm_of_rows_past_2_to_26():
    """dw and db are 2^27 columns of partial sums, 32 a workgroup of 1024 threads."""
    D = (1 << 26) + 5
    x, dy = _random(2, D, seed=1).requires_grad_(), _random(2, D, seed=2)
    w, b = torch.ones(D, device=DEV, requires_grad=True), torch.zeros(D, device=DEV, requires_grad=True)
    y = moc.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    # db is a sum of two bf16 numbers in fp32, rounded once or exact
    assert torch.equal(db, dy[0].float() + dy[1].float())
    want_w, want_y = torch.zeros(D, device=DEV, dtype=F64), None
    size = torch.zeros(D, device=DEV, dtype=F64)
    for r in range(2):
        v = x[r].detach().double()
        xh = (v - v.mean()) / torch.sqrt(v.var(unbiased=False) + 1e-5)
        # y is off by its rounding, half a step, and the statistics': sums of 2^18 numbers a lane, whose
        # rounding errors grow as the root of their number: 2^9 of them, and the lanes' 8 additions
        room = xh.abs() * (2.0 ** -8 * 1.01 + 2.0 ** 10 * 2.0 ** -24) + 2.0 ** 10 * 2.0 ** -24
        assert ((y[r].detach().double() - xh).abs() <= room).all()
        want_w += dy[r].double() * xh
        size += dy[r].double().abs() * (xh.abs() + 1)
    assert ((dw.double() - want_w).abs() <= 2.0 ** 10 * 2.0 ** -24 * size).all()
    assert dx.isfinite().all()


def test_conv_of_channels_past_2_to_23():
    """16 taps and the bias of 2^23 channels: 17 x 2^23 columns of partial sums."""
    D, S, T = (1 << 23) + 3, 16, 2
    x, dy = _random(1, T, D, seed=1).requires_grad_(), _random(1, T, D, seed=2)
    w, b = torch.ones(S, D, device=DEV, requires_grad=True), torch.zeros(D, device=DEV, requires_grad=True)
    y, _ = moc.causal_conv(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    xf, g = x.detach().float()[0], dy.float()[0]
    # sums of at most two products of bf16 numbers, exact in fp32 but for the one addition
    assert torch.equal(y[0, 0], x[0, 0]) and torch.equal(y[0, 1], (xf[0] + xf[1]).to(BF16))
    assert torch.equal(db, g[0] + g[1]) and torch.equal(dw[S - 2], g[1] * xf[0]) and not dw[:S - 2].any()
    assert torch.allclose(dw[S - 1], g[0] * xf[0] + g[1] * xf[1], rtol=2.0 ** -22, atol=1e-6)
    assert torch.equal(dx[0, 1], dy[0, 1]) and torch.equal(dx[0, 0], (g[0] + g[1]).to(BF16))
