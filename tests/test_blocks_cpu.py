"""The operators next to the MoC layers without a GPU: the 64-bit oracle's gradients
against autograd and against differences, refusals, modules, and the C ABI's argument
checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

import moc
from moc import _lib, blocks, ops
from oracle import block_oracle as O

F64 = torch.float64


def _scan_inputs(seed=0, n=9, H=4, P=3, G=2, N=5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    return r(n, H, P), r(n, H).abs() * 0.3, -r(H).abs() - 0.2, r(n, G, N), r(n, G, N), r(H)


def test_oracle_scan_gradients_are_autograds():
    ins = _scan_inputs()
    seqs = O.spans(9, None, [2, 3, 3, 8])
    assert seqs == [(0, 2), (2, 3), (3, 8), (8, 9)]
    g = torch.Generator().manual_seed(5)
    init = torch.randn(len(seqs), 4, 3, 5, generator=g, dtype=F64)
    dy, dfin = torch.randn(9, 4, 3, generator=g, dtype=F64), torch.randn(len(seqs), 4, 3, 5, generator=g, dtype=F64)
    _, grads = O.scan(*ins, seqs, init=init, dy=dy, dfin=dfin)
    leaves = [t.clone().requires_grad_() for t in (*ins, init)]
    x, u, A, B, C, D, h0 = leaves
    ys, total = [None] * 9, 0.0
    for q, (lo, hi) in enumerate(seqs):  # the recurrence again, for autograd
        h = h0[q]
        for t in range(lo, hi):
            Bh, Ch = B[t].repeat_interleave(2, 0), C[t].repeat_interleave(2, 0)
            h = torch.exp(u[t] * A)[:, None, None] * h + u[t][:, None, None] * x[t][:, :, None] * Bh[:, None]
            ys[t] = (h * Ch[:, None]).sum(-1) + D[:, None] * x[t]
        total = total + (h * dfin[q]).sum()
    total = total + (torch.stack(ys) * dy).sum()
    for got, want in zip(grads, torch.autograd.grad(total, leaves)):
        torch.testing.assert_close(got, want, rtol=1e-10, atol=1e-12)


def test_oracle_scan_gradients_are_differences():
    ins = _scan_inputs(1, n=5)
    seqs = [(0, 5)]
    dy = torch.randn(5, 4, 3, generator=torch.Generator().manual_seed(2), dtype=F64)
    _, grads = O.scan(*ins, seqs, dy=dy)
    for k, t in enumerate(ins):
        for e in (0, t.numel() // 2, t.numel() - 1):
            for_one = []
            for d in (1e-6, -1e-6):
                moved = [v.clone() for v in ins]
                moved[k].view(-1)[e] += d
                for_one.append((O.scan(*moved, seqs)[0] * dy).sum())
            want = (for_one[0] - for_one[1]) / 2e-6
            assert abs(grads[k].reshape(-1)[e] - want) < 1e-6 * max(1.0, abs(want))


@pytest.mark.parametrize("act", [False, True])
def test_oracle_conv_gradients_are_autograds(act):
    g = torch.Generator().manual_seed(3)
    x, w, b = (torch.randn(*s, generator=g, dtype=F64) for s in ((11, 4), (3, 4), (4,)))
    dy = torch.randn(11, 4, generator=g, dtype=F64)
    seqs = O.spans(11, None, [0, 1, 7])
    y, dx, dw, db = O.conv(x, w, b, act, seqs, dy=dy)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    parts = []
    for lo, hi in seqs:
        xs = torch.nn.functional.pad(leaves[0][lo:hi], (0, 0, 2, 0))
        p = sum(leaves[1][s] * xs[s:s + hi - lo] for s in range(3)) + leaves[2]
        parts.append(torch.nn.functional.silu(p) if act else p)
    want = torch.cat(parts)
    torch.testing.assert_close(y, want.detach())
    for got, w_ in zip((dx, dw, db), torch.autograd.grad(want, leaves, dy)):
        torch.testing.assert_close(got, w_)


def test_oracle_norm_is_torchs():
    g = torch.Generator().manual_seed(4)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=F64) for s in ((5, 7), (7,), (7,), (5, 7)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.nn.functional.layer_norm(leaves[0], (7,), leaves[1], leaves[2], 1e-3)
    y, *grads = O.norm(x, w, b, 1e-3, dy)
    torch.testing.assert_close(y, want.detach())
    for got, w_ in zip(grads, torch.autograd.grad(want, leaves, dy)):
        torch.testing.assert_close(got, w_)


# ---------------------------------------------------------------------------
# refusals: a tensor that says it is on the GPU, so that no check needs one

class _Cuda(torch.Tensor):
    is_cuda = True


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Cuda)


def test_cpu_tensors_are_refused():
    for call in (lambda: moc.layer_norm(torch.zeros(2, 4)),
                 lambda: moc.causal_conv(torch.zeros(1, 2, 4), torch.zeros(3, 4)),
                 lambda: moc.selective_scan(torch.zeros(1, 2, 1, 4), torch.zeros(1, 2, 1), torch.zeros(1),
                                            torch.zeros(1, 2, 1, 3), torch.zeros(1, 2, 1, 3))):
        with pytest.raises(ValueError, match="must all be CUDA tensors"):
            call()


@pytest.mark.parametrize("kw, error, match", [
    (dict(x=_t(2, 4, dtype=torch.float16)), TypeError, "unsupported x dtype"),
    (dict(x=_t(0, 4)), ValueError, "no empty one"),
    (dict(x=_t()), ValueError, "last axis"),
    (dict(x=_t(2, 4), weight=_t(5)), ValueError, "weight must have shape"),
    (dict(x=_t(2, 4), bias=_t(4, 1)), ValueError, "bias must have shape"),
    (dict(x=_t(2, 4), weight=_t(4, dtype=torch.int32)), TypeError, "weight must be floating point"),
])
def test_norm_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        moc.layer_norm(**kw)


_CU = torch.tensor([0, 2], dtype=torch.int32).as_subclass(_Cuda)


@pytest.mark.parametrize("kw, error, match", [
    (dict(activation="gelu"), ValueError, "unsupported activation"),
    (dict(x=_t(2, 4)), ValueError, r"x must be \[B,T,D\]"),
    (dict(weight=_t(3, 5)), ValueError, "dimensions disagree"),
    (dict(weight=_t(17, 4)), ValueError, "at most 16"),
    (dict(weight=_t(0, 4)), ValueError, "must not be empty"),
    (dict(x=_t(1, 0, 4)), ValueError, "must not be empty"),
    (dict(bias=_t(3)), ValueError, "bias must have shape"),
    (dict(cache=_t(1, 4, 2)), ValueError, "cache must have shape"),
    (dict(cache=_t(1, 4, 3, dtype=torch.float32)), ValueError, "cache must be a torch.bfloat16"),
    (dict(x=_t(2, 1, 4), cache=_t(1, 4, 3).expand(2, 4, 3)), ValueError, "share memory"),
    (dict(max_seqlen=3), ValueError, "must be None"),
    (dict(x=_t(2, 4), cu_seqlens=_CU), ValueError, "max_seqlen is required"),
    (dict(x=_t(2, 4), cu_seqlens=_CU, max_seqlen=0), ValueError, "positive Python int"),
    (dict(x=_t(2, 4), cu_seqlens=_CU, max_seqlen=2, output_final_state=True), ValueError, "only supported"),
    (dict(x=_t(2, 4), cu_seqlens=_CU.to(torch.float32).as_subclass(_Cuda), max_seqlen=2), TypeError, "int32 or"),
    (dict(x=_t(2, 4), cu_seqlens=torch.tensor([0, 2]), max_seqlen=2), ValueError, "CUDA tensor"),
])
def test_conv_refusals(kw, error, match):
    args = dict(x=_t(1, 2, 4), weight=_t(3, 4))
    args.update(kw)
    with pytest.raises(error, match=match):
        moc.causal_conv(**args)


@pytest.mark.parametrize("kw, error, match", [
    (dict(x=_t(2, 3, 4, 8)[0]), ValueError, "x/dt/B/C must be"),
    (dict(dt=_t(2, 3, 4, dtype=torch.float32)), TypeError, "same dtype"),
    (dict(dt=_t(2, 3, 5)), ValueError, "dimensions disagree"),
    (dict(dt=_t(2, 2, 4)), ValueError, "shapes differ"),
    (dict(C=_t(2, 3, 2, 7)), ValueError, "dimensions disagree"),
    (dict(B=_t(2, 3, 3, 6), C=_t(2, 3, 3, 6)), ValueError, "must divide the heads"),
    (dict(A=_t(3)), ValueError, "A must have shape"),
    (dict(D=_t(4, 8)), ValueError, "D must have shape"),
    (dict(dt_bias=_t(1)), ValueError, "dt_bias must have shape"),
    (dict(x=_t(2, 3, 4, 129)), ValueError, "at most 128"),
    (dict(B=_t(2, 3, 2, 257), C=_t(2, 3, 2, 257)), ValueError, "at most 256"),
    (dict(x=_t(2, 3, 4, 0)), ValueError, "must all be positive"),
    (dict(cache=_t(2, 4, 8, 6)), ValueError, "cache must be a torch.float32"),
    (dict(cache=_t(2, 4, 6, 8, dtype=torch.float32)), ValueError, "cache must have shape"),
])
def test_scan_refusals(kw, error, match):
    args = dict(x=_t(2, 3, 4, 8), dt=_t(2, 3, 4), A=_t(4), B=_t(2, 3, 2, 6), C=_t(2, 3, 2, 6))
    args.update(kw)
    with pytest.raises(error, match=match):
        moc.selective_scan(**args)


def test_modules():
    torch.manual_seed(0)
    c = moc.CausalConv(6, 4, activation="silu")
    assert {k: tuple(v.shape) for k, v in c.named_parameters()} == {"weight": (4, 6), "bias": (6,)}
    assert c.weight.abs().max() <= 0.5 and c.state_size == 24
    with pytest.raises(ValueError):
        moc.CausalConv(6, 4, activation="relu")
    with pytest.raises(ValueError, match="step expects x"):
        c.step(torch.zeros(2, 2, 6))
    s = moc.SelectiveScan(4, 8, 16, n_groups=2)
    assert {k: tuple(v.shape) for k, v in s.named_parameters()} == {"A_log": (4,), "D": (4,), "dt_bias": (4,)}
    u = torch.nn.functional.softplus(s.dt_bias)
    assert (u >= 0.9e-3).all() and (u <= 0.11).all() and (s.A_log.exp() <= 16.001).all()
    assert s.state_size == 4 * 8 * 16
    with pytest.raises(ValueError, match="must divide the heads"):
        moc.SelectiveScan(4, 8, 16, n_groups=3)
    with pytest.raises(ValueError, match="must have 32 channels"):
        s(torch.zeros(1, 2, 31), torch.zeros(1, 2, 4), torch.zeros(1, 2, 32), torch.zeros(1, 2, 32))
    n = moc.LayerNorm(5, bias=False)
    assert n.bias is None and torch.equal(n.weight, torch.ones(5))


def test_token_rows():
    wide = torch.zeros(2, 5, 30)
    for t, inner, want in ((wide[..., :12].unflatten(-1, (3, 4)), 2, 30), (wide[..., 7:8], 1, 30),
                           (torch.zeros(2, 5, 12).unflatten(-1, (3, 4)), 2, 12), (wide[:1, ..., :6], 1, 30),
                           (wide[:, :1, :6], 1, 150), (torch.zeros(7, 3, 4), 2, 12)):
        rows, step = ops.token_rows(t, inner)
        assert rows is t and step == want
    for t, inner in ((wide.transpose(0, 1)[..., :6], 1), (wide[..., ::2], 1), (wide[:, :1, :6].expand(2, 3, 6), 1),
                     (torch.zeros(2, 5, 4, 3).transpose(2, 3), 2), (wide[:, :4], 1)):
        rows, step = ops.token_rows(t, inner)
        assert rows.is_contiguous() and step == t.shape[-1] * (t.shape[-2] if inner == 2 else 1)
        assert torch.equal(rows, t)


# ---------------------------------------------------------------------------
# the C ABI's checks (no call gets past them)

FAKE = 0x1000
ERR_ARG, ERR_DTYPE, ERR_WORKSPACE = -1, -2, -3


@pytest.mark.parametrize("kw, code", [
    (dict(rows=0), ERR_ARG), (dict(dim=-1), ERR_ARG), (dict(x_dt=2), ERR_DTYPE), (dict(w_dt=9), ERR_DTYPE),
    (dict(x=None), ERR_ARG), (dict(mean=None), ERR_ARG), (dict(rows=1 << 31), ERR_ARG),
])
def test_capi_norm_arguments(kw, code):
    a = dict(x=FAKE, mean=FAKE, rows=4, dim=8, x_dt=1, w_dt=1)
    a.update(kw)
    L = _lib.lib()
    assert L.moc_norm_forward(a["x"], FAKE, FAKE, FAKE, a["mean"], FAKE, a["rows"], a["dim"], a["x_dt"], a["w_dt"], 0,
                              1e-5, None) == code
    assert L.moc_last_error()
    if "mean" not in kw:
        assert L.moc_norm_backward(a["x"], FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, a["rows"], a["dim"], a["x_dt"],
                                   a["w_dt"], 0, FAKE, 1 << 30, None) == code


def test_capi_workspaces():
    L = _lib.lib()
    assert L.moc_norm_backward(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 1, 1, 0, FAKE,
                               L.moc_norm_backward_workspace_bytes(4, 8) - 1, None) == ERR_WORKSPACE
    need = L.moc_conv_backward_workspace_bytes(100, 64, 4, 1)
    assert need >= 5 * 64 * 4
    assert L.moc_conv_backward(FAKE, FAKE, None, FAKE, FAKE, FAKE, None, None, 0, 0, 100, 50, 64, 4, 1, 1, 1, 0, FAKE,
                               need - 1, None) == ERR_WORKSPACE
    assert L.moc_norm_backward_workspace_bytes(0, 8) == 0 and L.moc_conv_backward_workspace_bytes(4, 0, 1, 1) == 0


@pytest.mark.parametrize("kw, code", [
    (dict(ks=0), ERR_ARG), (dict(ks=17), ERR_ARG), (dict(n=0), ERR_ARG), (dict(T=3), ERR_ARG), (dict(act=2), ERR_ARG),
    (dict(x_dt=2), ERR_DTYPE), (dict(cu=FAKE, n_seqs=0), ERR_ARG), (dict(cu=FAKE, n_seqs=2), ERR_ARG),
    (dict(n=1 << 31, T=1 << 31), ERR_ARG), (dict(x=None), ERR_ARG),
])
def test_capi_conv_arguments(kw, code):
    a = dict(x=FAKE, cu=None, n_seqs=0, n=8, T=4, ks=4, x_dt=1, act=0)
    a.update(kw)
    # (the packed call is refused for its cache)
    assert _lib.lib().moc_conv_forward(a["x"], FAKE, FAKE, FAKE, FAKE, FAKE, a["cu"], 0, a["n_seqs"], a["n"], a["T"],
                                       16, a["ks"], a["x_dt"], 1, 1, a["act"], None) == code


def _table(**kw):
    d = dict(x=FAKE, dt=FAKE, a=FAKE, b=FAKE, c=FAKE, d=None, dt_bias=None, x_stride=32, dt_stride=4, b_stride=12,
             c_stride=12, cu_seqlens=None, n_seqs=0, n_tokens=6, seq_len=3, heads=4, head_dim=8, groups=2, state_dim=6,
             cu_seqlens_i64=0, x_dtype=1, a_dtype=0, d_dtype=0, bias_dtype=0, dt_softplus=1)
    d.update(kw)
    return _lib.MocScan(*[d[n] for n, _ in _lib.MocScan._fields_])


@pytest.mark.parametrize("kw, code", [
    (dict(x=None), ERR_ARG), (dict(heads=0), ERR_ARG), (dict(groups=3), ERR_ARG), (dict(head_dim=129), ERR_ARG),
    (dict(state_dim=257), ERR_ARG), (dict(heads=40000, groups=1), ERR_ARG), (dict(x_dtype=2), ERR_DTYPE),
    (dict(a_dtype=7), ERR_DTYPE), (dict(dt_softplus=2), ERR_ARG), (dict(x_stride=31), ERR_ARG),
    (dict(x_stride=1 << 31), ERR_ARG), (dict(dt_stride=1 << 31), ERR_ARG), (dict(b_stride=1 << 31), ERR_ARG),
    (dict(c_stride=1 << 40), ERR_ARG),
    (dict(seq_len=4), ERR_ARG), (dict(n_tokens=0), ERR_ARG), (dict(cu_seqlens=FAKE, n_seqs=0), ERR_ARG),
    (dict(cu_seqlens=FAKE, n_seqs=2), ERR_ARG),
])
def test_capi_scan_arguments(kw, code):
    L = _lib.lib()
    t = _table(**kw)
    ref = ctypes.byref(t)
    assert L.moc_scan_forward(ref, FAKE, FAKE, FAKE, FAKE, 1 << 40, FAKE, 1 << 40, None) == code
    grads = _lib.MocScanGrads(*[FAKE] * 8)
    assert L.moc_scan_backward(ref, FAKE, 0, FAKE, FAKE, 1 << 40, ctypes.byref(grads), FAKE, 1 << 40, None) == code
    if "cu_seqlens" not in kw or kw["n_seqs"] == 0:
        assert L.moc_scan_saved_bytes(ref) == 0 and L.moc_last_error()


def test_capi_states_read_and_written_are_two_tensors():
    L = _lib.lib()
    ref = ctypes.byref(_table())
    assert L.moc_scan_forward(ref, FAKE, FAKE, FAKE, FAKE, 1 << 40, FAKE, 1 << 40, None) == ERR_ARG
    grads = _lib.MocScanGrads(*[FAKE] * 8)
    assert L.moc_scan_backward(ref, FAKE, 0, FAKE, FAKE, 1 << 40, ctypes.byref(grads), FAKE, 1 << 40, None) == ERR_ARG
    assert L.moc_conv_forward(FAKE, FAKE, None, FAKE, FAKE, FAKE, None, 0, 0, 8, 4, 16, 4, 1, 1, 1, 0, None) == ERR_ARG
    assert b"same tensor" in L.moc_last_error()


def test_capi_scan_workspaces():
    L = _lib.lib()
    t = _table()
    ref = ctypes.byref(t)
    # u, s (12 bytes a token slot and head; 2 sequences of one chunk) and the chunks' states
    assert L.moc_scan_saved_bytes(ref) >= 2 * 64 * 4 * 12 + 2 * 4 * 8 * 6 * 2
    need = L.moc_scan_forward_workspace_bytes(ref, 0)
    assert need > L.moc_scan_forward_workspace_bytes(ref, 1)
    assert L.moc_scan_forward(ref, FAKE, None, None, None, 0, FAKE, need - 1, None) == ERR_WORKSPACE
    assert L.moc_scan_forward(ref, FAKE, None, None, FAKE, 8, FAKE, 1 << 40, None) == ERR_WORKSPACE
    grads = _lib.MocScanGrads(*[FAKE] * 8)
    assert L.moc_scan_backward(ref, FAKE, 0, None, FAKE, 1 << 40, ctypes.byref(grads), FAKE,
                               L.moc_scan_backward_workspace_bytes(ref) - 1, None) == ERR_WORKSPACE
    step = _table(seq_len=3)
    assert L.moc_scan_update(ctypes.byref(step), FAKE, FAKE, None) == ERR_ARG  # three tokens a sequence


def test_written_bumps_the_version():
    t = torch.zeros(3)
    v = t._version
    blocks._written(t)
    assert t._version == v + 1
    with torch.inference_mode():
        blocks._written(torch.zeros(3))
