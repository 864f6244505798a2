"""Tensor subclasses through the operators next to the MoC layers: results have the type of x."""
from __future__ import annotations

import pytest
import torch

import moc
from moc import _lib, ops
from tests.test_gpu_blocks import BF16, DEV, F32, dev, rnd, scan_inputs


class Tagged(torch.Tensor):
    """A subclass without __torch_dispatch__: nothing in its dispatch keys."""


class _Recorder:
    """In the library's place: takes every call, says that it went well."""

    def __getattr__(self, name):
        return lambda *args: 64 if name.endswith("_bytes") else 0


def test_scan_launches_keep_the_type(monkeypatch):
    monkeypatch.setattr(_lib, "lib", _Recorder)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: None)
    ins = scan_inputs((2, 5), 2, 4, 1, 3, BF16, par=F32)
    order = [ins[q] for q in ("x", "dt", "A", "B", "C", "D", "dt_bias")]
    wide = torch.zeros(2, 5, 2, 9, dtype=BF16)[..., :4].as_subclass(Tagged)  # (not contiguous)
    for x in (order[0].as_subclass(Tagged), wide):
        args = [x, *order[1:]]
        y, fin, saved = ops.launch_scan_forward(*args, None, softplus=True, final_state=True, keep=True)
        assert type(y) is Tagged and type(fin) is Tagged and y.is_contiguous() and fin.dtype == F32
        grads = ops.launch_scan_backward(*args, order[0], None, saved, softplus=True, has_init=True, need_init=True)
        assert type(grads[0]) is Tagged and type(grads[7]) is Tagged and type(grads[1]) is torch.Tensor
        assert all(g.is_contiguous() and g.shape == t.shape for g, t in zip(grads, args))
        step = [t[:, :1] if t.ndim > 1 else t for t in args]
        assert type(ops.launch_scan_update(*step, torch.zeros(2, 2, 4, 3), softplus=True)) is Tagged


@pytest.mark.gpu
def test_subclasses_keep_their_type():
    x, w, b = (dev(t) for t in (rnd(2, 20, 32, seed=1, dtype=BF16), rnd(4, 32, seed=2), rnd(32, seed=3)))
    ins = {k: dev(v) for k, v in scan_inputs((2, 20), 2, 16, 1, 8, BF16).items()}
    tag = lambda t: t.as_subclass(Tagged)  # noqa: E731
    H, s = _lib.host(), dict(ins)
    assert H.norm(x, b, b, 1e-5) is not None
    assert H.norm(tag(x), b, b, 1e-5) is None and H.norm(x, tag(b), b, 1e-5) is None
    assert H.conv(tag(x), w, b, None, 0, False, None) is None
    assert H.conv(x, w, tag(b), None, 0, False, None) is None
    assert H.scan(tag(s["x"]), s["dt"], s["A"], s["B"], s["C"], None, None, None, True, False, None) is None
    assert H.scan(s["x"], s["dt"], tag(s["A"]), s["B"], s["C"], None, None, None, True, False, None) is None
    cut = lambda d, k: {q: (v[:, :k] if v.ndim > 1 else v) for q, v in d.items()}  # noqa: E731
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            pairs = []
            for t, i in ((tag(x), dict(ins, x=tag(ins["x"]))), (x, ins)):
                cc, sc = torch.zeros(2, 32, 4, dtype=BF16, device=DEV), torch.zeros(2, 2, 16, 8, device=DEV)
                pairs.append((moc.layer_norm(t, b, b), moc.causal_conv(t, w, b, "silu")[0],
                              moc.causal_conv(t, w, cache=cc)[0], moc.causal_conv(t[:, :1], w, cache=cc)[0],
                              *moc.selective_scan(**i, output_final_state=True),
                              moc.selective_scan(**cut(i, 1), cache=sc)[0]))
            for got, want in zip(*pairs):
                assert type(got) is Tagged and type(want) is torch.Tensor
                assert torch.equal(got.as_subclass(torch.Tensor), want)
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(moc.layer_norm(tag(leaf)).sum(), leaf)
    want, = torch.autograd.grad(moc.layer_norm(leaf).sum(), leaf)
    assert torch.equal(g.as_subclass(torch.Tensor), want)
