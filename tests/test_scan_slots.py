"""Where the scan keeps states: the library's byte queries over packed sequences, and a model of
the slots (without a GPU); on the GPU, packed sequences that use them."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

import moc
from moc import _lib
from tests.test_blocks_cpu import FAKE, _table
from tests.test_gpu_blocks import BF16, F32, check_scan, dev, scan_inputs


def _packed(n_seqs, n_tokens=16384, **kw):
    d = dict(heads=32, head_dim=64, groups=32, state_dim=128, x_stride=2048, dt_stride=32, b_stride=4096,
             c_stride=4096, cu_seqlens=FAKE, n_seqs=n_seqs, n_tokens=n_tokens, seq_len=0)
    d.update(kw)
    return _table(**d)


@pytest.mark.parametrize("x_dtype", [0, 1])
def test_states_do_not_grow_with_the_number_of_sequences(x_dtype):
    """512 or 4096 sequences in 16384 tokens keep what two keep, but for 12 bytes a head and token
    place and 12 a head and chunk of the partial sums."""
    L = _lib.lib()
    def sizes(n_seqs):
        ref = ctypes.byref(_packed(n_seqs, x_dtype=x_dtype))
        return (L.moc_scan_saved_bytes(ref), L.moc_scan_forward_workspace_bytes(ref, 1),
                L.moc_scan_backward_workspace_bytes(ref))

    few = sizes(2)
    assert all(few)
    state = 32 * 64 * 128 * 4
    assert few[0] <= (16384 // 64) * state + (16384 // 64 + 4) * 32 * 64 * 12 + 4096
    for n_seqs in (512, 4096):
        many = sizes(n_seqs)
        more = n_seqs - 2
        assert many[0] - few[0] <= more * 32 * 64 * 12 + 1024
        assert many[1] == few[1]
        assert many[2] - few[2] <= more * 32 * 12 + 1024


def _model(edges, q):
    """Slots of a piece's entering state, forwards and in reverse, as the kernels form them."""
    fwd, rev = [], []
    for lo, hi in zip(edges[:-1], edges[1:]):
        pieces = -(-(hi - lo) // q)
        fwd += [lo // q + k - 1 for k in range(1, pieces)]
        rev += [lo // q + k for k in range(pieces - 1)]
    return fwd, rev


def test_slots_are_distinct_and_few():
    rng = random.Random(0)
    for _ in range(300):
        n, q = rng.randint(1, 2000), rng.choice([64, 128, 192])
        cuts = sorted(rng.randint(0, n) for _ in range(rng.randint(0, 40)))
        for slots in _model([0, *cuts, n], q):
            assert len(set(slots)) == len(slots) and all(0 <= s < n // q for s in slots)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cu, n", [([0, 700, 701, 765, 829, 830, 1530, 1658, 2600], 2600), ([63, 127, 900, 1023, 1025], 1700),
                                   ([0, 129, 258, 258, 387, 515], 643)])
def test_long_and_short_sequences(dtype, cu, n):
    """Sequences of several segments next to ones of a token, at edges off every multiple of 64."""
    check_scan(scan_inputs((n,), 2, 20, 1, 16, dtype), cu=cu)


@pytest.mark.gpu
def test_memory_of_many_sequences():
    """1024 sequences of 16 tokens, forward and backward: what the call allocates stays near its inputs' size."""
    H, P, N, n = 8, 64, 64, 16384
    ins = {k: dev(v).requires_grad_() for k, v in scan_inputs((n,), H, P, 1, N, BF16).items()}
    cu = torch.arange(0, n + 1, 16, device="cuda:0")
    states = n // 64 * H * P * N * 4
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y, _ = moc.selective_scan(**ins, cu_seqlens=cu, max_seqlen=16)
    torch.autograd.grad(y, list(ins.values()), torch.ones_like(y))
    peak = torch.cuda.max_memory_allocated() - before
    # kept states twice, segments' at most as much, u and s of 1280 chunks, inputs' gradients and dy
    assert peak <= 3 * states + 1300 * H * 64 * 12 + 8 * ins["x"].numel() * 2 + (8 << 20)
