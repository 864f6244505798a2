"""The operators next to the MoC layers under forward-mode differentiation and tracing, for
inputs that do not ask for gradients: without a GPU, each launch replaced by one that writes
its output where no tracer and no tangent can see it, as the kernels do."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import moc
from moc import blocks, ops


def _hidden(like, value):
    """A tensor that nothing watched being filled."""
    y = torch.empty(like.shape, dtype=like.dtype)
    y.detach().numpy()[...] = value.detach().numpy()
    return y


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    def norm(x, weight, bias, eps, keep):
        return _hidden(x, 2 * x), None, None

    def conv(x, weight, bias, cache, *, activation_flag, cu_seqlens=None, final_state=False):
        return _hidden(x, 3 * x), (_hidden(x, x).sum() if final_state else None)

    def conv_step(x, weight, bias, cache, *, activation_flag):
        cache.detach().numpy()[...] += 1
        return _hidden(x, 4 * x)

    def scan(x, dt, A, B, C, D, dt_bias, init, *, softplus, final_state, keep, cu_seqlens=None):
        return _hidden(x, 5 * x), (_hidden(x, x) if final_state else None), None

    def scan_step(x, dt, A, B, C, D, dt_bias, state, *, softplus):
        state.detach().numpy()[...] += 1
        return _hidden(x, 6 * x)

    monkeypatch.setattr(blocks, "_on_gpu", lambda x: False)
    monkeypatch.setattr(blocks, "_check_tensors", lambda x, **others: None)
    for name, f in (("norm_forward", norm), ("conv_forward", conv), ("conv_update", conv_step),
                    ("scan_forward", scan), ("scan_update", scan_step)):
        monkeypatch.setattr(ops, f"launch_{name}", f)


def _scan(x, cache=None, **kw):
    B, T = x.shape[:2]
    one = torch.ones(B, T, 1, 3)
    return moc.selective_scan(x.unflatten(-1, (2, 2)), torch.ones(B, T, 2), torch.ones(2), one, one, cache=cache,
                              **kw)[0].flatten(-2)


W = torch.ones(3, 4)
CALLS = {
    "norm": lambda x: moc.layer_norm(x),
    "conv": lambda x: moc.causal_conv(x, W)[0],
    "conv with a state": lambda x: moc.causal_conv(x, W, output_final_state=True)[0],
    "conv from a cache": lambda x: moc.causal_conv(x, W, cache=torch.zeros(2, 4, 3))[0],
    "conv step": lambda x: moc.causal_conv(x[:, :1], W, cache=torch.zeros(2, 4, 3))[0],
    "scan": _scan,
    "scan from a cache": lambda x: _scan(x, torch.zeros(2, 2, 2, 3), output_final_state=True),
    "scan step": lambda x: _scan(x[:, :1], torch.zeros(2, 2, 2, 3)),
    "scan step, strided state": lambda x: _scan(x[:, :1], torch.zeros(2, 2, 3, 2).transpose(2, 3)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_a_tangent_is_refused(name):
    x = torch.randn(2, 5, 4)
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            CALLS[name](forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", list(CALLS))
def test_a_trace_holds_the_call(name):
    x, x2 = torch.randn(2, 5, 4), torch.randn(2, 5, 4)
    want = CALLS[name](x2)
    traced = torch.jit.trace(CALLS[name], (x,), check_trace=False)
    assert any(n.kind() == "prim::PythonOp" for n in traced.graph.nodes()) or "Function" in str(traced.graph)
    torch.full((2, 5, 4), float("nan"))  # (memory that an unrecorded output could be found in)
    assert torch.equal(traced(x2), want)


def test_steps_are_not_differentiable_and_in_place():
    w = W.clone().requires_grad_()
    cache, state = torch.zeros(2, 4, 3), torch.zeros(2, 2, 3, 2).transpose(2, 3)
    y, got = moc.causal_conv(torch.randn(2, 1, 4), w, cache=cache, output_final_state=True)
    assert got is cache and not y.requires_grad and (cache == 1).all() and cache._version == 1
    x = torch.randn(2, 1, 4, requires_grad=True)
    assert not _scan(x, state).requires_grad and (state == 1).all()
