"""The scan's gradients by their norm, on inputs whose gradients do not cancel: x, B, C and dy
scatter around 1 and decays are slow, so that what crosses chunks is a large part of dA and ddt.

The element-wise bounds of tests/test_gpu_blocks.py are worst cases over sums of absolute
values, wider than the sums themselves where millions of terms of random sign cancel: there a
gradient of zero, or one without a part of it, would pass for dA and ddt_bias.  Here a part
that is missing shows; test_missing_parts_show holds that, without a GPU.

Tolerances (relative to the norm, fixed from the arithmetic before the first run).  Rounded to
bf16, every element is off by at most half a step, 2^-8 of it, and so is the norm; what the
kernels' own factors in two planes lose (2^-15 of a product) is 2^-11 with all sums behind it.
fp32 sums of up to 2^8 products in a row, of one sign here, lose at most 2^-16 of it; sums
within a chunk that da takes the difference of are at most four times as large: 2^-14."""
from __future__ import annotations

import pytest
import torch

import moc
from oracle import block_oracle as O
from tests.test_gpu_blocks import BF16, DEV, F32, F64, dev, rnd, scan_inputs

NAMES = ("x", "dt", "A", "B", "C", "D", "dt_bias")

# the shapes of tests/test_gpu_blocks.py: (lead, H, P, G, N, cu)
SHAPES = [((B, T), H, P, G, N, None) for B, T, H, P, G, N in (
    (1, 1, 1, 1, 1, 1), (2, 1, 2, 8, 1, 4), (1, 2, 3, 5, 3, 7), (2, 63, 2, 16, 1, 16), (1, 64, 4, 64, 2, 64),
    (2, 65, 2, 40, 1, 24), (1, 130, 6, 33, 3, 100), (1, 200, 2, 64, 1, 128), (1, 77, 2, 80, 1, 130),
    (1, 70, 1, 128, 1, 256), (1, 90, 5, 72, 1, 31), (2, 700, 2, 20, 1, 16), (2, 700, 1, 64, 1, 72), (2, 100, 2, 24, 2, 20),
    (2, 130, 4, 36, 2, 100), (1, 200, 2, 20, 1, 12), (1, 77, 2, 68, 1, 132), (3, 65, 2, 64, 1, 4), (1, 70, 1, 4, 1, 252))]
SHAPES += [((n,), 2, 24, 1, 40, cu) for cu, n in (
    ([0, 1, 1, 2, 66, 66, 130], 130), ([3, 70], 150), ([0, 64, 128], 128), ([5, 5], 9), ([0, 600, 610], 610))]


def firm(lead, H, P, G, N, dtype, par=F32):
    ins = scan_inputs(lead, H, P, G, N, dtype, par=par)
    for k in ("x", "B", "C"):
        ins[k] = (1 + 0.5 * ins[k].float()).to(dtype)
    ins["dt"] = (0.5 * ins["dt"].float()).to(dtype)
    ins["A"] = (-torch.linspace(0.02, 0.3, H)).to(par)
    ins["dt_bias"] = torch.full((H,), -3.0).to(par)
    return ins


def case(lead, H, P, G, N, cu, dtype, par=F32):
    """(inputs, flat inputs, u, sequences, init, dfin, dy)."""
    ins = firm(lead, H, P, G, N, dtype, par)
    flat = {k: (v.flatten(0, 1) if v.ndim > 1 and cu is None else v) for k, v in ins.items()}
    seqs = O.spans(flat["x"].shape[0], None if cu is not None else lead[1], cu)
    u = O.step_lengths(flat["dt"], flat["dt_bias"], True)
    init, dfin = (None, None) if cu is not None else (rnd(lead[0], H, P, N, seed=20, mean=1.0) * 0.5,
                                                      rnd(lead[0], H, P, N, seed=21, mean=1.0))
    dy = rnd(*ins["x"].shape, seed=50, dtype=dtype, mean=1.0)
    return ins, flat, u, seqs, init, dfin, dy


def oracle(flat, u, seqs, init, dfin, dy):
    """Gradients by name, in 64 bits."""
    dyf = dy.reshape(flat["x"].shape)
    _, (dx, du, dA, dB, dC, dD, dinit, _) = O.scan(flat["x"], u, flat["A"], flat["B"], flat["C"], flat["D"], seqs,
                                                   init=init, dy=dyf, dfin=dfin)
    ddt = du * O.sigmoid_of(u, True)
    return dict(zip(NAMES, (dx, ddt, dA, dB, dC, dD, ddt.sum(0)))) | {"init": dinit}


def room(name, dtype, par):
    """Accepted distance, relative to the gradient's norm."""
    stored = F32 if name == "init" else (par if name in ("A", "D", "dt_bias") else dtype)
    return (2.0 ** -8 if stored == BF16 else 0.0) + (2.0 ** -11 if dtype == BF16 else 2.0 ** -14)


def distance(got, want):
    got, want = got.detach().cpu().to(F64).reshape(want.shape), want.to(F64)
    return float((got - want).norm() / want.norm()) if want.norm() > 0 else float(got.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, par", [(BF16, F32), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("lead, H, P, G, N, cu", SHAPES)
def test_gradients(lead, H, P, G, N, cu, dtype, par):
    ins, flat, u, seqs, init, dfin, dy = case(lead, H, P, G, N, cu, dtype, par)
    want = oracle(flat, u, seqs, init, dfin, dy)
    leaves = {k: dev(v).requires_grad_() for k, v in ins.items()}
    more, outs = {}, [dev(dy)]
    if cu is None:
        leaves["init"] = dev(init).requires_grad_()
        more = dict(cache=leaves["init"], output_final_state=True)
        outs.append(dev(dfin))
        if lead[1] == 1:
            # (a cache and one token are a step: without the cache)
            leaves.pop("init"), more.pop("cache"), want.pop("init")
            want = oracle(flat, u, seqs, None, dfin, dy)
    else:
        more = dict(cu_seqlens=torch.tensor(cu, device=DEV), max_seqlen=max(b - a for a, b in seqs))
    y, fin = moc.selective_scan(**{k: leaves[k] for k in NAMES}, **more)
    got = torch.autograd.grad([y] if cu is not None else [y, fin], list(leaves.values()), outs)
    for name, g in zip(leaves, got):
        far = distance(g, want[name])
        assert far <= room(name, dtype, par), f"{name}: {far:.3g} of {room(name, dtype, par):.3g}"


def _without_crossing(flat, u, seqs, init, dfin, dy):
    """(ddt, dA) without z, the part of da that crosses a chunk of 64 tokens from end to end, and
    (ddt, dA) of chunks that know nothing of each other."""
    want = oracle(flat, u, seqs, init, dfin, dy)
    dyf = dy.reshape(flat["x"].shape).to(F64)
    H, P = dyf.shape[1:]
    G, N = flat["B"].shape[1:]
    x, A = flat["x"].to(F64), flat["A"].to(F64)
    Bh, Ch = (flat[k].to(F64).repeat_interleave(H // G, 1) for k in ("B", "C"))
    a = torch.exp(u * A)
    z, chunks = torch.zeros_like(u), []
    for q, (lo, hi) in enumerate(seqs):
        h = torch.zeros(H, P, N, dtype=F64) if init is None else init[q].to(F64)
        before = {}
        for t in range(lo, hi):
            if (t - lo) % 64 == 0:
                before[t] = h
                chunks.append((t, min(t + 64, hi)))
            h = a[t, :, None, None] * h + (u[t, :, None] * x[t])[:, :, None] * Bh[t][:, None]
        dh = torch.zeros(H, P, N, dtype=F64) if dfin is None else dfin[q].to(F64)
        for t in reversed(list(before)):
            end = min(t + 64, hi)
            z[t:end] = (before[t] * dh).sum((1, 2)) * a[t:end].prod(0)
            for i in range(end - 1, t - 1, -1):
                dh = a[i, :, None, None] * (dh + dyf[i][:, :, None] * Ch[i][:, None])
    sig = O.sigmoid_of(u, True)
    no_z = (want["dt"] - sig * A * z, want["A"] - (u * z).sum(0))
    alone = oracle(flat, u, chunks, None, None, dy)
    return want, no_z, (alone["dt"], alone["A"])


@pytest.mark.parametrize("lead, H, P, G, N, cu", SHAPES)
def test_missing_parts_show(lead, H, P, G, N, cu):
    """At every listed shape zeros are at least twice as far as accepted, and so are, in dA of fp32 parameters (and ddt of
    fp32 inputs), gradients without what crosses a chunk from end to end (where there is a state before it and a
    gradient behind it) and those of chunks by themselves (where there are two, or states)."""
    _, flat, u, seqs, init, dfin, dy = case(lead, H, P, G, N, cu, F32)
    want, no_z, alone = _without_crossing(flat, u, seqs, init, dfin, dy)
    longest = max(b - a for a, b in seqs)
    for dtype, par in ((BF16, F32), (BF16, BF16), (F32, F32)):
        for name in NAMES:
            if want[name].norm() > 0:
                assert distance(torch.zeros_like(want[name]), want[name]) > 2 * room(name, dtype, par)
    for k, name, dtype in ((1, "A", BF16), (1, "A", F32), (0, "dt", F32)):
        limit = 2 * room(name, dtype, F32)
        if init is not None or longest > 128:
            assert distance(no_z[k], want[name]) > limit, name
        if init is not None or longest > 64:
            assert distance(alone[k], want[name]) > limit, name
