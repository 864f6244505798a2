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


def test_chunks_of_a_differentiated_scan_fit_a_grid():
    """The backward's workgroups have 512 threads, and a grid counts threads in 32 bits: 2^23 chunks are
    refused before anything is launched, by the forward that would keep states for it too."""
    L = _lib.lib()
    small = dict(heads=1, head_dim=1, groups=1, state_dim=1, x_stride=1, dt_stride=1, b_stride=1, c_stride=1)
    fits = ctypes.byref(_table(**small, n_tokens=64, seq_len=64))
    grads = _lib.MocScanGrads(*[FAKE] * 7, None)
    ERR_WORKSPACE = -3
    for kw in (dict(n_tokens=(1 << 22) + (1 << 23), seq_len=1),              # a chunk a token
               dict(n_tokens=1 << 29, seq_len=1 << 29),                      # 2^23 chunks of 64
               dict(n_tokens=1 << 20, cu_seqlens=FAKE, n_seqs=1 << 23, seq_len=0)):
        ref = ctypes.byref(_table(**small, **kw))
        assert L.moc_scan_saved_bytes(ref) == 0 and L.moc_scan_backward_workspace_bytes(ref) == 0
        assert L.moc_scan_forward_workspace_bytes(ref, 1) == 0 and L.moc_scan_forward_workspace_bytes(ref, 0) > 0
        assert L.moc_scan_forward(ref, FAKE, None, None, FAKE, 1 << 50, FAKE, 0, None) == ERR_ARG
        assert L.moc_scan_backward(ref, FAKE, 0, None, FAKE, 1 << 50, ctypes.byref(grads), FAKE, 0, None) == ERR_ARG
        assert b"too many chunks" in L.moc_last_error()
        assert L.moc_scan_forward(ref, FAKE, None, None, None, 0, FAKE, 0, None) == ERR_WORKSPACE  # (past the checks)
    assert L.moc_scan_backward(fits, FAKE, 0, None, FAKE, 1 << 50, ctypes.byref(grads), FAKE, 0, None) == ERR_WORKSPACE


def test_norm_workspace_of_long_rows():
    """Rows past what a workgroup's registers hold are summed in 64 parts: no more is asked for."""
    L = _lib.lib()
    assert L.moc_norm_backward_workspace_bytes(4096, 1 << 20) == 64 * 2 * (1 << 20) * 4
    assert L.moc_norm_backward_workspace_bytes(3, 1 << 20) == 3 * 2 * (1 << 20) * 4
    assert L.moc_norm_backward_workspace_bytes(4096, 16384) == 512 * 2 * 16384 * 4
    assert L.moc_norm_backward_workspace_bytes(4096, 16385) == 64 * 2 * 16385 * 4


def test_conv_channels_fit_a_grid():
    """2^31 - 1 channels, two a lane, would be a grid of 2^32 threads, which runs none of them."""
    L = _lib.lib()
    for dim in ((1 << 31) - 1, 1 << 30, 0):
        assert L.moc_conv_forward(FAKE, FAKE, None, None, FAKE, None, None, 0, 0, 1, 1, dim, 16, 0, 0, 0, 0, None) == ERR_ARG
        assert L.moc_conv_backward(FAKE, FAKE, None, FAKE, FAKE, FAKE, None, None, 0, 0, 1, 1, dim, 16, 0, 0, 0, 0, FAKE,
                                   1 << 60, None) == ERR_ARG
        assert L.moc_conv_update(FAKE, FAKE, None, FAKE, 1, 1, 1, FAKE, 1, dim, 16, 0, 0, 0, 0, None) == ERR_ARG
        assert b"dim must be" in L.moc_last_error()
