"""Calls of the operators next to the MoC layers that something watches: the host module hands
them back, tracers record them, tangents are refused."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

import moc
from moc import _lib
from tests.test_gpu_blocks import BF16, DEV, F32, dev, rnd, scan_inputs

pytestmark = pytest.mark.gpu

B, T, H, P, N, S = 2, 37, 2, 16, 24, 4
INS = scan_inputs((B, T), H, P, 1, N, BF16)
W, BIAS = rnd(S, H * P, seed=2), rnd(H * P, seed=3)


def _scan(x, cache=None, one=False, **kw):
    cut = (lambda t: t[:, :1]) if one else (lambda t: t)
    rest = {k: (cut(dev(v)) if v.ndim > 1 else dev(v)) for k, v in INS.items() if k != "x"}
    return moc.selective_scan(cut(x).unflatten(-1, (H, P)), **rest, cache=cache, **kw)[0].flatten(-2)


CALLS = {
    "norm": lambda x: moc.layer_norm(x, dev(BIAS), dev(BIAS)),
    "conv": lambda x: moc.causal_conv(x, dev(W), dev(BIAS), "silu")[0],
    "conv prompt": lambda x: moc.causal_conv(x, dev(W), cache=torch.ones(B, H * P, S, dtype=BF16, device=DEV),
                                             output_final_state=True)[0],
    "conv step": lambda x: moc.causal_conv(x[:, :1], dev(W), cache=torch.ones(B, H * P, S, dtype=BF16, device=DEV))[0],
    "scan": _scan,
    "scan prompt": lambda x: _scan(x, torch.ones(B, H, P, N, device=DEV), output_final_state=True),
    "scan step": lambda x: _scan(x, torch.ones(B, H, P, N, device=DEV), one=True),
}


def _x(seed):
    return dev(rnd(B, T, H * P, seed=seed, dtype=BF16))


def test_host_module_hands_watched_calls_back():
    x, host = _x(1), _lib.host()
    i = {k: dev(v) for k, v in INS.items()}
    def calls(t):
        return [host.norm(t, None, None, 1e-5), host.conv(t, dev(W), None, None, 0, False, None),
                host.scan(t.unflatten(-1, (H, P)), i["dt"], i["A"], i["B"], i["C"], None, None, None, True, False, None)]

    assert all(v is not None for v in calls(x))
    got = []
    with forward_ad.dual_level():
        got += calls(forward_ad.make_dual(x, x))
    torch.func.grad(lambda t: (got.extend(calls(t)), t.sum())[1])(x)
    torch.func.vmap(lambda t: (got.extend(calls(t[None])[:2]), t)[1])(x)
    torch.jit.trace(lambda t: (got.extend(calls(t)), t)[1], (x,), check_trace=False)

    class Seen(TorchDispatchMode):
        ops = 0

        def __torch_dispatch__(self, func, types, args, kwargs=None):
            self.ops += 1
            return func(*args, **(kwargs or {}))

    with Seen() as seen:
        got += calls(x)
        ys = [f(x) for f in CALLS.values()]
    assert len(got) == 14 and all(v is None for v in got) and seen.ops > 0
    assert all(torch.equal(y, f(x)) for y, f in zip(ys, CALLS.values()))


@pytest.mark.parametrize("name", list(CALLS))
def test_a_tangent_is_refused(name):
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            CALLS[name](forward_ad.make_dual(_x(1), _x(2)))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", list(CALLS))
def test_a_trace_holds_the_call(name, grad):
    x2 = _x(2)
    want = CALLS[name](x2)
    traced = torch.jit.trace(CALLS[name], (_x(1).requires_grad_(grad),), check_trace=False)
    assert torch.equal(traced(x2), want)
