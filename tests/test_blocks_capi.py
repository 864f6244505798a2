"""Argument checks of the C entries of the operators next to the MoC layers that go past single
arguments (no call gets past them; no GPU)."""
from __future__ import annotations

import ctypes

from moc import _lib
from tests.test_blocks_cpu import ERR_ARG, FAKE, _table


def test_a_packed_scan_has_no_initial_state():
    """Its first chunks keep no state, so that the backward would read what nobody wrote."""
    L = _lib.lib()
    ref = ctypes.byref(_table(cu_seqlens=FAKE, n_seqs=2, seq_len=0))
    grads = _lib.MocScanGrads(*[FAKE] * 7, None)
    assert L.moc_scan_backward(ref, FAKE, 1, None, FAKE, 1 << 40, ctypes.byref(grads), FAKE, 0, None) == ERR_ARG
    assert b"fixed-length" in L.moc_last_error()
