"""The operators next to the MoC layers on the GPU against the 64-bit oracle.

Tolerances (fixed from the arithmetic before the first run).  Every result is a sum of
products, so its error is bounded by a multiple of the same sum over absolute values
(``size``): ``k`` fp32 roundings (k * 2^-24 of it; k counts a result's additions and the
roundings of its factors), ``m`` roundings of a bf16 matrix operand (m * 2^-8 of it, bf16
scans only), and one rounding of the result to its dtype (half a step of the result)."""
from __future__ import annotations

import pytest
import torch

import moc
from moc import _lib
from oracle import block_oracle as O

pytestmark = pytest.mark.gpu

F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
DEV = "cuda:0"


def near(name, got, want, size, k, m=0.0):
    got64, want, size = got.detach().cpu().to(F64), want.to(F64), size.to(F64)
    assert got64.shape == want.shape, f"{name}: {tuple(got64.shape)} vs {tuple(want.shape)}"
    assert torch.isfinite(got64).all(), f"{name}: not finite"
    room = k * O.F32_HALF * size + m * O.half_step(BF16) * size
    if got.dtype != F32:
        room = room * 1.01 + O.half_step(got.dtype) * want.abs()
        if got.dtype == F16:
            room = room + 2.0 ** -25  # (half the subnormal step)
    err = (got64 - want).abs()
    bad = err > room + 1e-37
    if bad.any():
        i = int((err / (room + 1e-37)).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off; worst at {i}: got "
                             f"{got64.flatten()[i].item():.8g}, want {want.flatten()[i].item():.8g}, room "
                             f"{room.flatten()[i].item():.3g}")


def rnd(*shape, seed=0, dtype=F32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype)


def dev(t):
    return None if t is None else t.to(DEV)


# ---------------------------------------------------------------------------
# layer norm

NORM_K = 256  # up to 80 additions a lane and 8 across them, three sums deep


def check_norm(x, w, b, dy, eps=1e-5, leading=None):
    leaves = [None if t is None else dev(t).requires_grad_() for t in (x, w, b)]
    y = moc.layer_norm(*leaves, eps=eps)
    with torch.no_grad():
        assert torch.equal(moc.layer_norm(*leaves, eps=eps), y)
    has = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, has, dev(dy)))
    x2 = x.reshape(-1, x.shape[-1])
    want = O.norm(x2, w, b, eps, dy.reshape(x2.shape))
    x64 = x2.to(F64)
    rstd = 1 / torch.sqrt(x64.var(-1, unbiased=False, keepdim=True) + eps)
    X = rstd * (x64.abs() + x64.abs().mean(-1, keepdim=True))
    wa = torch.ones(x.shape[-1], dtype=F64) if w is None else w.to(F64).abs()
    ga = dy.reshape(x2.shape).to(F64).abs() * wa
    near("y", y.reshape(x2.shape), want[0], X * wa + (0 if b is None else b.to(F64).abs()), NORM_K)
    size_x = rstd * (ga + ga.mean(-1, keepdim=True) + X * (ga * X).mean(-1, keepdim=True))
    near("dx", next(grads).reshape(x2.shape), want[1], size_x, 2 * NORM_K)
    dya = dy.reshape(x2.shape).to(F64).abs()
    if w is not None:
        near("dw", next(grads), want[2], (dya * X).sum(0), NORM_K)
    if b is not None:
        near("db", next(grads), want[3], dya.sum(0), NORM_K)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows, dim", [(1, 1), (1, 2), (3, 7), (5, 64), (37, 100), (130, 128), (9, 129), (4, 513),
                                       (67, 1000), (3, 1131), (5, 2048), (6, 2049), (2, 4096), (3, 8191), (2, 8192),
                                       (2, 16384), (3, 20000), (1500, 72)])
def test_norm(dtype, rows, dim):
    check_norm(rnd(rows, dim, seed=1, dtype=dtype, mean=0.4), rnd(dim, seed=2, dtype=dtype, mean=1.0),
               rnd(dim, seed=3, dtype=dtype), rnd(rows, dim, seed=4, dtype=dtype))


@pytest.mark.parametrize("w_dt, b_dt", [(F32, None), (None, BF16), (None, None), (F16, F32), (BF16, F16)])
def test_norm_parameters(w_dt, b_dt):
    w = None if w_dt is None else rnd(200, seed=2, dtype=w_dt)
    b = None if b_dt is None else rnd(200, seed=3, dtype=b_dt)
    check_norm(rnd(3, 5, 200, seed=1, dtype=BF16), w, b, rnd(3, 5, 200, seed=4, dtype=BF16), eps=1e-3)


def test_norm_layouts():
    """Strided, offset (unaligned) and broadcast tensors give what their copies give."""
    x = dev(rnd(6, 5, 64, seed=1, dtype=BF16))
    w, b = dev(rnd(64, seed=2)), dev(rnd(64, seed=3))
    want = moc.layer_norm(x, w, b)
    assert torch.equal(moc.layer_norm(x.transpose(0, 1), w, b), want.transpose(0, 1))
    off = torch.empty(6 * 5 * 64 + 3, dtype=BF16, device=DEV)[3:].view(6, 5, 64)
    off.copy_(x)
    assert torch.equal(moc.layer_norm(off, w, b), want)
    one = x.clone().requires_grad_()
    moc.layer_norm(one, w, b).sum().backward()  # the gradient of a sum: every stride 0
    two = x.clone().requires_grad_()
    moc.layer_norm(two, w, b).backward(torch.ones_like(x))
    assert torch.equal(one.grad, two.grad)


def test_norm_constant_rows_and_large_means():
    x = torch.full((4, 96), 3.0)
    x[1] = 0
    y = moc.layer_norm(dev(x))
    assert torch.equal(y.cpu(), torch.zeros(4, 96))
    check_norm(rnd(4, 96, seed=1, mean=50.0), None, None, rnd(4, 96, seed=2))


def test_norm_infinities_stay_in_their_row():
    x = rnd(4, 64, seed=1)
    want = moc.layer_norm(dev(x))
    x[2, 5] = float("inf")
    x[3, 1] = float("nan")
    got = moc.layer_norm(dev(x))
    assert torch.equal(got[:2], want[:2]) and got[2:].isnan().all()


def test_norm_past_32_bit_offsets():
    rows, dim = (1 << 21) + 3, 2048  # 2^32 elements and some
    x = torch.zeros(rows, dim, dtype=BF16, device=DEV)
    tail = dev(rnd(3, dim, seed=1, dtype=BF16))
    x[-3:] = tail
    assert torch.equal(moc.layer_norm(x)[-3:], moc.layer_norm(tail))


# ---------------------------------------------------------------------------
# causal convolution

def check_conv(x, w, b, act, dy=None, cu=None, history=None, cu_dtype=torch.int32):
    """Outputs and gradients of x [B, T, D] or packed [N, D] (cu: list)."""
    D = x.shape[-1]
    flat = x.reshape(-1, D)
    seqs = O.spans(flat.shape[0], None if cu is not None else x.shape[1], cu)
    more = {} if cu is None else {"cu_seqlens": torch.tensor(cu, dtype=cu_dtype, device=DEV), "max_seqlen": len(flat)}
    leaves = [None if t is None else dev(t).requires_grad_() for t in (x, w, b)]
    y, st = moc.causal_conv(*leaves, activation="silu" if act else None, **more)
    assert st is None
    with torch.no_grad():
        assert torch.equal(moc.causal_conv(*leaves, activation="silu" if act else None, **more)[0], y)
    want = O.conv(flat, w, b, act, seqs, dy=dy.reshape(flat.shape))
    pa = O.conv(flat.to(F64).abs(), w.to(F64).abs(), None if b is None else b.to(F64).abs(), False, seqs)
    near("y", y.reshape(flat.shape), want[0], pa, 64)
    ga = dy.reshape(flat.shape).to(F64).abs() * ((1 + pa) if act else 1)
    _, dxa, dwa, dba = O.conv(flat.to(F64).abs(), w.to(F64).abs(), None, False, seqs, dy=ga)
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dev(dy))
    near("dx", got[0].reshape(flat.shape), want[1], dxa, 64)
    near("dw", got[1], want[2], dwa, 160)
    if b is not None:
        near("db", got[2], want[3], dba, 160)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, T, D, S, act", [
    (1, 1, 1, 1, False), (2, 1, 8, 4, True), (1, 2, 5, 3, False), (3, 3, 64, 4, True), (2, 17, 130, 2, True),
    (1, 130, 512, 4, False), (2, 65, 520, 7, True), (1, 40, 24, 8, False), (2, 33, 16, 9, True), (1, 70, 10, 13, False),
    (1, 9, 36, 16, True), (2, 700, 1028, 3, True)])
def test_conv(dtype, B, T, D, S, act):
    check_conv(rnd(B, T, D, seed=1, dtype=dtype), rnd(S, D, seed=2, dtype=dtype, scale=0.5), rnd(D, seed=3, dtype=dtype),
               act, rnd(B, T, D, seed=4, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cu, n, S", [([0, 1, 1, 2, 50, 50, 130], 130, 4), ([3, 10, 64], 90, 3), ([0, 5], 5, 8),
                                      ([7, 7], 20, 4), (list(range(0, 81)), 80, 5)])
def test_conv_packed(dtype, cu, n, S):
    check_conv(rnd(n, 72, seed=1, dtype=dtype), rnd(S, 72, seed=2, dtype=F32, scale=0.5), None, True,
               rnd(n, 72, seed=4, dtype=dtype), cu=cu, cu_dtype=torch.int64 if S == 3 else torch.int32)
    x = dev(rnd(n, 72, seed=1, dtype=dtype))
    w, cu_t = dev(rnd(S, 72, seed=2)), torch.tensor(cu, device=DEV)
    a = moc.causal_conv(x, w, cu_seqlens=cu_t, max_seqlen=n)[0]
    assert torch.equal(moc.causal_conv(x[None], w, cu_seqlens=cu_t, max_seqlen=n)[0], a[None])


@pytest.mark.parametrize("w_dt, b_dt", [(F32, F16), (F16, F32), (F64, BF16)])
def test_conv_parameters(w_dt, b_dt):
    check_conv(rnd(2, 30, 40, seed=1, dtype=BF16), rnd(4, 40, seed=2, dtype=BF16).to(w_dt),
               rnd(40, seed=3, dtype=BF16).to(b_dt), True, rnd(2, 30, 40, seed=4, dtype=BF16))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T, S", [(2, 4), (3, 4), (4, 4), (5, 3), (90, 8), (2, 1), (3, 16)])
def test_conv_from_a_cache(dtype, T, S):
    B, D = 3, 40
    x, w, b = rnd(B, T, D, seed=1, dtype=dtype), rnd(S, D, seed=2, dtype=dtype, scale=0.5), rnd(D, seed=3, dtype=dtype)
    cache = rnd(B, D, S, seed=5, dtype=dtype)
    seqs = O.spans(B * T, T, None)
    want = O.conv(x.reshape(-1, D), w, b, True, seqs, history=cache.transpose(1, 2))
    size = O.conv(x.reshape(-1, D).abs(), w.abs(), b.abs(), False, seqs, history=cache.abs().transpose(1, 2))
    with torch.no_grad():
        y, fin = moc.causal_conv(dev(x), dev(w), dev(b), "silu", cache=dev(cache), output_final_state=True)
    near("y", y.reshape(-1, D), want, size, 64)
    state = torch.cat((cache, x.transpose(1, 2)), 2)[:, :, -S:]
    assert torch.equal(fin.cpu(), state)
    # without a cache: zeros before the prompt
    fin0 = moc.causal_conv(dev(x), dev(w), output_final_state=True)[1]
    assert torch.equal(fin0.cpu(), torch.cat((torch.zeros_like(cache), x.transpose(1, 2)), 2)[:, :, -S:])
    # with gradients: the same values, and those of the cache
    leaves = [dev(t).requires_grad_() for t in (x, w, b, cache)]
    y2, fin2 = moc.causal_conv(*leaves[:3], "silu", cache=leaves[3], output_final_state=True)
    assert torch.equal(y2, y) and torch.equal(fin2, fin)
    dy = rnd(B, T, D, seed=6, dtype=dtype)
    every = torch.cat((cache.transpose(1, 2)[:, 1:], x), 1)
    dy_all = torch.cat((torch.zeros(B, S - 1, D, dtype=dtype), dy), 1)
    _, dxe, dwe, _ = O.conv(every.reshape(-1, D), w, b, True, O.spans(B * (T + S - 1), T + S - 1, None),
                            dy=dy_all.reshape(-1, D))
    dxe = dxe.reshape(B, T + S - 1, D)
    pa = O.conv(every.reshape(-1, D).abs(), w.abs(), b.abs(), False, O.spans(B * (T + S - 1), T + S - 1, None))
    ga = dy_all.reshape(-1, D).abs() * (1 + pa)
    _, dxa, dwa, _ = O.conv(every.reshape(-1, D).abs(), w.abs(), None, False, O.spans(B * (T + S - 1), T + S - 1, None),
                            dy=ga)
    dxa = dxa.reshape(B, T + S - 1, D)
    gx, gw, _, gc = torch.autograd.grad(y2, leaves, dev(dy))
    near("dx", gx, dxe[:, S - 1:], dxa[:, S - 1:], 64)
    near("dw", gw, dwe, dwa, 160)
    near("dcache", gc[:, :, 1:], dxe[:, :S - 1].transpose(1, 2), dxa[:, :S - 1].transpose(1, 2), 64)
    assert not gc[:, :, :1].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, D, S", [(1, 1, 1), (3, 40, 4), (2, 130, 3), (5, 64, 8), (2, 33, 16)])
def test_conv_steps_continue_a_prompt(dtype, B, D, S):
    x, w, b = (dev(t) for t in (rnd(B, 9, D, seed=1, dtype=dtype), rnd(S, D, seed=2, dtype=dtype),
                                rnd(D, seed=3, dtype=dtype)))
    whole, fin = moc.causal_conv(x, w, b, "silu", output_final_state=True)
    _, cache = moc.causal_conv(x[:, :5], w, b, "silu", output_final_state=True)
    strided = torch.empty(B, S, D, dtype=dtype, device=DEV).transpose(1, 2)  # a cache of other strides
    strided.copy_(cache)
    version = cache._version
    for t in range(5, 9):
        y, st = moc.causal_conv(x[:, t:t + 1], w, b, "silu", cache=cache, output_final_state=True)
        y2, none = moc.causal_conv(x[:, t:t + 1], w, b, "silu", cache=strided)
        assert st is cache and none is None
        assert torch.equal(y, whole[:, t:t + 1]) and torch.equal(y2, y)
    assert torch.equal(cache, fin) and torch.equal(strided, fin) and cache._version > version


def test_conv_is_moc_with_one_route():
    """The layer next to it: MoC on one route of weight 1 is this convolution."""
    x, w = dev(rnd(2, 50, 64, seed=1, dtype=BF16)), dev(rnd(4, 64, seed=2, dtype=BF16))
    want, _ = moc.moc_hip(x, torch.ones(2, 50, 1, dtype=BF16, device=DEV), w[None], activation="silu")
    got, _ = moc.causal_conv(x, w, activation="silu")
    assert (got.float() - want.float()).abs().max() <= 2 ** -7 * want.float().abs().max()


def test_conv_infinities_stay_in_their_window():
    x = rnd(2, 40, 16, seed=1)
    w = dev(rnd(4, 16, seed=2))
    want = moc.causal_conv(dev(x), w)[0]
    x[0, 20, 3] = float("nan")
    got = moc.causal_conv(dev(x), w)[0]
    bad = torch.zeros(2, 40, 16, dtype=torch.bool)
    bad[0, 20:24, 3] = True
    assert torch.equal(got.isnan().cpu(), bad) and torch.equal(got[~bad.to(DEV)], want[~bad.to(DEV)])


def test_conv_past_32_bit_offsets():
    n, D = (1 << 20) + 37, 2056
    x = torch.zeros(n, D, dtype=BF16, device=DEV)
    tail = dev(rnd(40, D, seed=1, dtype=BF16))
    x[-40:] = tail
    w = dev(rnd(4, D, seed=2, dtype=BF16))
    cu = torch.tensor([0, n - 40, n], device=DEV)
    y = moc.causal_conv(x, w, cu_seqlens=cu, max_seqlen=n)[0]
    assert torch.equal(y[-40:], moc.causal_conv(tail[None], w)[0][0])


# ---------------------------------------------------------------------------
# selective scan

def scan_inputs(lead, H, P, G, N, dtype, seed=0, par=None):
    par = par or dtype
    return dict(x=rnd(*lead, H, P, seed=seed + 1, dtype=dtype), dt=rnd(*lead, H, seed=seed + 2, dtype=dtype, scale=0.7),
                A=(-rnd(H, seed=seed + 3).abs() * 6 - 0.3).to(par), B=rnd(*lead, G, N, seed=seed + 4, dtype=dtype),
                C=rnd(*lead, G, N, seed=seed + 5, dtype=dtype), D=rnd(H, seed=seed + 6, dtype=par),
                dt_bias=rnd(H, seed=seed + 7, dtype=par, mean=-2.0))


def check_scan(ins, cu=None, init=None, dfin=None, softplus=True, grads=True, cu_dtype=torch.int32, seed=50):
    x, dt, A, B, C, D, bias = (ins[k] for k in ("x", "dt", "A", "B", "C", "D", "dt_bias"))
    H, P = x.shape[-2:]
    G, N = B.shape[-2:]
    flat = lambda t, inner: t.reshape(-1, *t.shape[t.ndim - inner:])  # noqa: E731
    xf, dtf, Bf, Cf = flat(x, 2), flat(dt, 1), flat(B, 2), flat(C, 2)
    n = xf.shape[0]
    seqs = O.spans(n, None if cu is not None else x.shape[1], cu)
    fixed = cu is None
    T = max(b - a for a, b in seqs)
    dy = rnd(*x.shape, seed=seed, dtype=x.dtype)
    u = O.step_lengths(dtf, bias, softplus)
    (want_y, want_fin), g = O.scan(xf, u, A, Bf, Cf, D, seqs, init=init, dy=flat(dy, 2), dfin=dfin)
    ab = lambda t: None if t is None else t.to(F64).abs()  # noqa: E731
    (ya, fa), ga = O.scan(ab(xf), u, A, ab(Bf), ab(Cf), ab(D), seqs, init=ab(init), dy=ab(flat(dy, 2)), dfin=ab(dfin))
    bf = x.dtype == BF16
    k, m = N + T + 384, 1.02 if bf else 0.0
    names = ["x", "dt", "A", "B", "C", "D", "dt_bias"]
    leaves = {q: None if ins[q] is None else dev(ins[q]).requires_grad_() for q in names}
    cache = None if init is None else dev(init).requires_grad_()
    more = dict(dt_softplus=softplus)
    if not fixed:
        more |= dict(cu_seqlens=torch.tensor(cu, dtype=cu_dtype, device=DEV), max_seqlen=T)
    y, fin = moc.selective_scan(**leaves, cache=cache, output_final_state=fixed, **more)
    with torch.no_grad():
        y2, fin2 = moc.selective_scan(**leaves, cache=cache, output_final_state=fixed, **more)
    assert torch.equal(y, y2)
    near("y", flat(y, 2), want_y, ya, k, m)
    if fixed:
        assert torch.equal(fin, fin2) and fin.dtype == F32
        near("state", fin, want_fin, fa, k)
    if not grads:
        return
    has = [t for t in leaves.values() if t is not None] + ([] if cache is None else [cache])
    outs, gouts = ([y], [dev(dy)]) if dfin is None else ([y, fin], [dev(dy), dev(dfin)])
    got = torch.autograd.grad(outs, has, gouts, retain_graph=True)
    again = torch.autograd.grad(outs, has, gouts)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    got = iter(got)
    k = 2 * k
    dxa, _, dAa, dBa, dCa, dDa, dia, daa = ga
    sig = O.sigmoid_of(u, softplus)
    A64 = A.to(F64).abs()
    dua = ga[1] - A.to(F64) * daa + A64 * daa
    # pairs within a chunk cancel between the row and column sums that da is formed from:
    # up to 256 fp32 roundings of all of a sequence's pairs
    pairs = torch.zeros_like(u)
    ya0 = ya - (0 if D is None else ab(D)[:, None] * ab(xf))
    for a_, b_ in seqs:
        pairs[a_:b_] = (ab(flat(dy, 2))[a_:b_] * ya0[a_:b_]).sum((0, 2))
    slack = 256 * O.F32_HALF * A64 * pairs
    near("dx", flat(next(got), 2), g[0], dxa, k, m)
    roomy = (k * O.F32_HALF + 2 * m * O.half_step(BF16))
    near("ddt", flat(next(got), 1), g[1] * sig, (dua + slack / roomy) * sig, k, 2 * m)
    near("dA", next(got), g[2], dAa + ((u * slack) / A64).sum(0) / roomy, k + n, 2 * m)
    near("dB", flat(next(got), 2), g[3], dBa, k + H, m)
    near("dC", flat(next(got), 2), g[4], dCa, k + H, m)
    if D is not None:
        near("dD", next(got), g[5], dDa, k + n)
    if bias is not None:
        near("ddt_bias", next(got), (g[1] * sig).sum(0), ((dua + slack / roomy) * sig).sum(0), k + n, 2 * m)
    if cache is not None:
        near("dcache", next(got), g[6], dia, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, T, H, P, G, N", [
    (1, 1, 1, 1, 1, 1), (2, 1, 2, 8, 1, 4), (1, 2, 3, 5, 3, 7), (2, 63, 2, 16, 1, 16), (1, 64, 4, 64, 2, 64),
    (2, 65, 2, 40, 1, 24), (1, 130, 6, 33, 3, 100), (1, 200, 2, 64, 1, 128), (1, 77, 2, 80, 1, 130),
    (1, 70, 1, 128, 1, 256), (1, 90, 5, 72, 1, 31)])
def test_scan(dtype, B, T, H, P, G, N):
    check_scan(scan_inputs((B, T), H, P, G, N, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H, P, N", [(2, 20, 16), (1, 64, 72)])
def test_scan_segments(dtype, H, P, N):
    """Long sequences of few heads: walked in several segments."""
    check_scan(scan_inputs((2, 700), H, P, 1, N, dtype), init=rnd(2, H, P, N, seed=20), dfin=rnd(2, H, P, N, seed=21))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2, 64, 100])
def test_scan_states(dtype, T):
    ins = scan_inputs((2, T), 2, 24, 2, 20, dtype, par=F32)
    check_scan(ins, init=rnd(2, 2, 24, 20, seed=20), dfin=rnd(2, 2, 24, 20, seed=21))
    check_scan(ins, init=rnd(2, 2, 24, 20, seed=20))
    check_scan(ins, dfin=rnd(2, 2, 24, 20, seed=21))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cu, n", [([0, 1, 1, 2, 66, 66, 130], 130), ([3, 70], 150), ([0, 64, 128], 128),
                                   ([5, 5], 9), (list(range(0, 41)), 40), ([0, 600, 610], 610)])
def test_scan_packed(dtype, cu, n):
    check_scan(scan_inputs((n,), 2, 24, 1, 40, dtype), cu=cu, cu_dtype=torch.int64 if n == 150 else torch.int32)


@pytest.mark.parametrize("kw", [dict(D=None), dict(dt_bias=None), dict(D=None, dt_bias=None)])
def test_scan_without_parameters(kw):
    ins = scan_inputs((2, 50), 2, 16, 1, 16, BF16, par=F32)
    ins.update(kw)
    check_scan(ins)


def test_scan_without_softplus():
    ins = scan_inputs((2, 70), 2, 16, 1, 16, F32)
    ins["dt"] = ins["dt"].abs() * 0.1
    ins["dt_bias"] = ins["dt_bias"].abs() * 0.05
    check_scan(ins, softplus=False)


def test_scan_parameter_dtypes():
    ins = scan_inputs((1, 40), 3, 16, 1, 16, BF16, par=BF16)
    ins["A"], ins["D"], ins["dt_bias"] = ins["A"].to(F16), ins["D"].float(), ins["dt_bias"].double()
    check_scan(ins)


def test_scan_far_decays():
    """Running sums of thousands, step lengths of almost 0 and decay rates of 0."""
    ins = scan_inputs((1, 150), 3, 16, 1, 16, F32)
    ins["dt_bias"] = torch.tensor([4.0, -30.0, 0.0])
    ins["A"] = torch.tensor([-40.0, -3.0, 0.0])
    check_scan(ins)


def test_scan_packed_has_a_batch_axis():
    ins = {k: dev(v) for k, v in scan_inputs((90,), 2, 16, 1, 16, BF16).items()}
    cu = torch.tensor([0, 30, 90], device=DEV)
    want, _ = moc.selective_scan(**ins, cu_seqlens=cu, max_seqlen=60)
    one = {k: (v[None] if v.ndim > 1 else v) for k, v in ins.items()}
    got, _ = moc.selective_scan(**one, cu_seqlens=cu, max_seqlen=60)
    assert torch.equal(got, want[None])
    # each sequence by itself
    for lo, hi in ((0, 30), (30, 90)):
        part = {k: (v[None, lo:hi] if v.ndim > 1 else v) for k, v in ins.items()}
        assert torch.equal(moc.selective_scan(**part)[0][0], want[lo:hi])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_reads_slices_in_place(dtype):
    """x, dt, B and C as slices of one projection give what their copies give."""
    H, P, G, N = 3, 16, 1, 24
    ins = scan_inputs((2, 80), H, P, G, N, dtype)
    for pad in (0, 1, 8):
        wide = torch.cat([ins[k].reshape(2, 80, -1) for k in ("x", "B", "C", "dt")] + [torch.zeros(2, 80, pad, dtype=dtype)],
                         -1)
        wide = dev(wide).requires_grad_()
        x, B, C, dt, _ = wide.split([H * P, G * N, G * N, H, pad], -1)
        par = {k: dev(ins[k]) for k in ("A", "D", "dt_bias")}
        y, fin = moc.selective_scan(x.unflatten(-1, (H, P)), dt, par["A"], B.unflatten(-1, (G, N)),
                                    C.unflatten(-1, (G, N)), par["D"], par["dt_bias"], output_final_state=True)
        own = {k: dev(ins[k]).requires_grad_() for k in ("x", "dt", "B", "C")}
        y2, fin2 = moc.selective_scan(**own, **par, output_final_state=True)
        assert torch.equal(y, y2) and torch.equal(fin, fin2)
        dy = dev(rnd(2, 80, H, P, seed=9, dtype=dtype))
        gw, = torch.autograd.grad(y, wide, dy)
        gx, gdt, gB, gC = torch.autograd.grad(y2, list(own.values()), dy)
        want = torch.cat([t.reshape(2, 80, -1) for t in (gx, gB, gC, gdt)], -1)
        assert torch.equal(gw[..., :want.shape[-1]], want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B, T, H, P, G, N", [
    (2, 130, 4, 36, 2, 100), (1, 200, 2, 20, 1, 12), (1, 77, 2, 68, 1, 132), (3, 65, 2, 64, 1, 4), (1, 70, 1, 4, 1, 252)])
def test_scan_of_multiples_of_four(dtype, B, T, H, P, G, N):
    check_scan(scan_inputs((B, T), H, P, G, N, dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H, P, G, N", [(6, 33, 3, 100), (2, 40, 1, 128), (2, 72, 1, 130), (2, 80, 1, 256), (3, 5, 1, 7)])
def test_scan_uses_nothing_behind_the_last_token(dtype, H, P, G, N):
    """Whatever lies behind the last token of x, dt, B and C in memory (here NaN or 0) changes no bit."""
    T = 130
    ins = scan_inputs((1, T), H, P, G, N, dtype)
    dy = rnd(1, T, H, P, seed=9, dtype=dtype)
    results = []
    for tail in (0.0, float("nan")):
        leaves = {}
        for q, t in ins.items():
            if q in ("x", "dt", "B", "C"):
                t = torch.cat([t, torch.full_like(t[:, :64], tail)], 1)
            leaves[q] = dev(t).requires_grad_()
        cut = {q: t[:, :T] if q in ("x", "dt", "B", "C") else t for q, t in leaves.items()}
        y, fin = moc.selective_scan(**cut, output_final_state=True, dt_softplus=True)
        dyt = torch.cat([dy, torch.full_like(dy[:, :64], tail)], 1)
        g = torch.autograd.grad([y], list(leaves.values()), [dev(dyt)[:, :T]])
        results.append((y, fin, *(t[:, :T] if t.ndim > 1 else t for t in g)))
    for a, b in zip(*results):
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H, P, G, N", [(2, 64, 1, 128), (3, 5, 3, 7), (4, 80, 2, 16), (1, 128, 1, 256), (2, 16, 1, 1)])
def test_scan_steps(dtype, H, P, G, N):
    ins = scan_inputs((3, 6), H, P, G, N, dtype)
    init = rnd(3, H, P, N, seed=20)
    d = {k: dev(v) for k, v in ins.items()}
    cache = dev(init)
    odd = torch.empty(3, H, N, P, device=DEV).transpose(2, 3)  # a state of other strides
    odd.copy_(cache)
    ys = []
    for t in range(6):
        one = {k: (v[:, t:t + 1] if v.ndim > 1 else v) for k, v in d.items()}
        y, st = moc.selective_scan(**one, cache=cache, output_final_state=True)
        y2, _ = moc.selective_scan(**one, cache=odd)
        assert st is cache and torch.equal(y, y2) and torch.equal(cache, odd)
        ys.append(y)
    flat = lambda t: t.reshape(-1, *t.shape[2:])  # noqa: E731
    u = O.step_lengths(flat(ins["dt"]), ins["dt_bias"], True)
    seqs = O.spans(18, 6, None)
    want_y, want_fin = O.scan(flat(ins["x"]), u, ins["A"], flat(ins["B"]), flat(ins["C"]), ins["D"], seqs, init=init)
    ab = lambda t: t.to(F64).abs()  # noqa: E731
    ya, fa = O.scan(ab(flat(ins["x"])), u, ins["A"], ab(flat(ins["B"])), ab(flat(ins["C"])), ab(ins["D"]), seqs,
                    init=ab(init))
    near("y", flat(torch.cat(ys, 1)), want_y, ya, N + 128)
    near("state", cache, want_fin, fa, 128)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_prompt_in_pieces(dtype):
    """A prompt piece by piece, each from the last one's state, is the whole prompt."""
    ins = scan_inputs((2, 150), 2, 32, 1, 32, dtype)
    d = {k: dev(v) for k, v in ins.items()}
    _, whole = moc.selective_scan(**d, output_final_state=True)
    cache = None
    for lo, hi in ((0, 70), (70, 71), (71, 150)):
        part = {k: (v[:, lo:hi] if v.ndim > 1 else v) for k, v in d.items()}
        _, cache = moc.selective_scan(**part, cache=cache, output_final_state=True)
    # (the same sums in other orders: fp32 roundings of the state's size)
    u = O.step_lengths(ins["dt"].reshape(300, 2), ins["dt_bias"], True)
    ab = lambda t: t.reshape(300, *t.shape[2:]).to(F64).abs()  # noqa: E731
    _, fa = O.scan(ab(ins["x"]), u, ins["A"], ab(ins["B"]), ab(ins["C"]), None, O.spans(300, 150, None))
    near("state", cache, whole.cpu(), fa, 2 * (32 + 150 + 384))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["x", "dt", "B", "C"])
def test_scan_infinities_reach_later_tokens_only(dtype, value, which):
    """What an infinity or NaN in token 70 of the first sequence reaches: nothing before it,
    nothing of the other sequence, and of x nothing but its own channel."""
    if which == "dt" and value > 0:
        value = float("nan")
    ins = scan_inputs((2, 140), 2, 16, 1, 16, dtype)
    clean = moc.selective_scan(**{k: dev(v) for k, v in ins.items()})[0]
    t = ins[which].clone()
    t[(0, 70, 1, 3)[:t.ndim] if which in ("x", "dt") else (0, 70, 0, 3)] = value
    ins[which] = t
    got = moc.selective_scan(**{k: dev(v) for k, v in ins.items()})[0]
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :70], clean[0, :70])
    heads = slice(None) if which in ("B", "C") else slice(1, 2)
    assert not got[0, 70, heads].isfinite().all()
    assert torch.equal(got[0, 70:, :1], clean[0, 70:, :1]) or which in ("B", "C")
    if which == "x":
        keep = [p for p in range(16) if p != 3]
        assert torch.equal(got[0, 70:, 1][:, keep], clean[0, 70:, 1][:, keep])
        assert not got[0, 70:, 1, 3].isfinite().any()
    if which == "C":
        assert torch.equal(got[0, 71:], clean[0, 71:])


def test_scan_past_32_bit_offsets():
    n, H, P, N = 139000, 256, 64, 16  # 2^31 elements of x and some
    x = torch.zeros(n, H, P, dtype=BF16, device=DEV)
    ins = {k: dev(v) for k, v in scan_inputs((100,), H, P, 1, N, BF16).items()}
    x[-100:] = ins["x"]
    dt, B, C = (torch.zeros(n, *ins[k].shape[1:], dtype=BF16, device=DEV) for k in ("dt", "B", "C"))
    for t, k in ((dt, "dt"), (B, "B"), (C, "C")):
        t[-100:] = ins[k]
    cu = torch.tensor([0, n - 100, n], device=DEV)
    y, _ = moc.selective_scan(x, dt, ins["A"], B, C, ins["D"], ins["dt_bias"], cu_seqlens=cu, max_seqlen=n)
    want, _ = moc.selective_scan(**{k: (v[None] if v.ndim > 1 else v) for k, v in ins.items()})
    assert torch.equal(y[-100:], want[0])


# ---------------------------------------------------------------------------
# together, graphs, streams

class Block(torch.nn.Module):
    """norm -> projection -> causal convolution -> scan -> projection: the operators as
    a block around them uses them, a MoC layer in the convolution's place if asked."""

    def __init__(self, dim=64, heads=2, head_dim=32, state=16, routed=False):
        super().__init__()
        self.inner, self.heads, self.state = heads * head_dim, heads, state
        self.norm = moc.LayerNorm(dim)
        self.w_in = torch.nn.Linear(dim, self.inner + 2 * state + heads, bias=False)
        self.conv = moc.MoC(self.inner, dim, 4, 4, "silu") if routed else moc.CausalConv(self.inner, 4, "silu")
        self.scan = moc.SelectiveScan(heads, head_dim, state)
        self.w_out = torch.nn.Linear(self.inner, dim, bias=False)
        self.routed = routed

    def forward(self, x, caches=None, **kw):
        z = self.norm(x)
        v, B, C, dt = self.w_in(z).split([self.inner, self.state, self.state, self.heads], -1)
        want = {"output_final_state": True} if caches is not None else {}
        c0, c1 = caches if caches else (None, None)
        v, s0 = self.conv(v, z, cache=c0, **want, **kw) if self.routed else self.conv(v, cache=c0, **want, **kw)
        y, s1 = self.scan(v, dt, B, C, cache=c1, **want, **kw)
        return x + self.w_out(y), (s0, s1)


@pytest.mark.parametrize("routed", [False, True])
def test_block_trains_and_serves(routed):
    torch.manual_seed(0)
    m = Block(routed=routed).to(DEV)
    x = dev(rnd(2, 90, 64, seed=1)).requires_grad_()
    y, _ = m(x)
    y.square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters()) and x.grad.isfinite().all()
    # a derivative along a direction, against differences (fp32: a step of 2^-7, second order)
    d = dev(rnd(2, 90, 64, seed=2))
    with torch.no_grad():
        f = lambda s: m(x + s * d)[0].double().square().mean()  # noqa: E731
        want = (f(2.0 ** -7) - f(-2.0 ** -7)) / 2 ** -6
    torch.testing.assert_close((x.grad.double() * d).sum(), want, rtol=2e-3, atol=1e-6)
    with torch.no_grad():
        whole, _ = m(x)
        part, caches = m(x[:, :80], caches=())
        outs = [part]
        for t in range(80, 90):
            o, caches = m(x[:, t:t + 1], caches=caches)
            outs.append(o)
    torch.testing.assert_close(torch.cat(outs, 1), whole, rtol=1e-4, atol=1e-4)
    # packed: each sequence is what it is alone
    cu = torch.tensor([0, 33, 90], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        packed, _ = m(x[0], cu_seqlens=cu, max_seqlen=57)
        torch.testing.assert_close(packed[33:], m(x[:1, 33:])[0][0], rtol=1e-4, atol=1e-4)


def test_steps_in_a_graph():
    torch.manual_seed(0)
    m = Block().to(DEV).to(BF16)
    x = dev(rnd(4, 12, 64, seed=1, dtype=BF16))
    with torch.no_grad():
        _, first = m(x[:, :4], caches=())
        eager = tuple(c.clone() for c in first)
        held = tuple(c.clone() for c in first)
        x_in = torch.empty(4, 1, 64, dtype=BF16, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x_in.copy_(x[:, :1])
            m(x_in, caches=tuple(c.clone() for c in first))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y_out, _ = m(x_in, caches=held)
        for c, e in zip(held, first):
            c.copy_(e)
        for t in range(4, 12):
            want, eager = m(x[:, t:t + 1], caches=eager)
            x_in.copy_(x[:, t:t + 1])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y_out, want) and all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_training_in_a_graph(dtype):
    """Forward and gradients of all three operators, captured and replayed on new inputs
    with eager work between, give the eager results."""
    H, P, N, T = 2, 32, 16, 300
    par = {k: dev(v).requires_grad_() for k, v in scan_inputs((1, 1), H, P, 1, N, dtype).items() if v.ndim == 1}
    w, b = dev(rnd(4, H * P, seed=30, dtype=dtype)).requires_grad_(), dev(rnd(H * P, seed=31, dtype=dtype)).requires_grad_()
    nw = dev(rnd(H * P, seed=32, dtype=dtype)).requires_grad_()

    def step(x, dt, B, C, dy):
        v = moc.layer_norm(x, nw)
        v, _ = moc.causal_conv(v, w, b, "silu")
        y, _ = moc.selective_scan(v.unflatten(-1, (H, P)), dt, par["A"], B, C, par["D"], par["dt_bias"])
        return (y, *torch.autograd.grad(y, (x, dt, B, C, w, b, nw, *par.values()), dy))

    def inputs(seed):
        i = scan_inputs((2, T), H, P, 1, N, dtype, seed=seed)
        return [dev(t) for t in (i["x"].flatten(2), i["dt"], i["B"], i["C"], rnd(2, T, H, P, seed=seed + 9, dtype=dtype))]

    static = [t.requires_grad_(k < 4) for k, t in enumerate(inputs(0))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for seed in (100, 200, 300):
        new = inputs(seed)
        with torch.no_grad():
            for s, t in zip(static, new):
                s.copy_(t)
        want = step(*[t.requires_grad_(k < 4) for k, t in enumerate(new)])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_two_streams_at_once():
    """Calls on two streams at a time do not share anything."""
    ins = [{k: dev(v) for k, v in scan_inputs((1, 400), 4, 64, 1, 64, BF16, seed=s).items()} for s in (0, 40)]
    want = [moc.selective_scan(**i)[0] for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(moc.selective_scan(**ins[k])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[k]) for k in (0, 1) for g in got[k])


def test_double_backward_is_refused():
    x = dev(rnd(2, 8)).requires_grad_()
    g, = torch.autograd.grad(moc.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|differentiate"):
        torch.autograd.grad(g.sum(), x)


def test_library_refuses_what_python_would():
    x = dev(rnd(1, 4, 8))
    with pytest.raises(RuntimeError, match="kernel_size must be in"):
        moc.ops.launch_conv_forward(x, dev(rnd(17, 8)), None, None, activation_flag=0)
    assert _lib.lib().moc_last_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scan_strides_of_a_single_token_are_not_read(dtype):
    H, P, G, N = 2, 64, 1, 64
    ins = {q: dev(t) for q, t in scan_inputs((1, 1), H, P, G, N, dtype).items()}
    order = [ins[q] for q in ("x", "dt", "A", "B", "C", "D", "dt_bias")]
    dy = dev(rnd(1, 1, H, P, seed=9, dtype=dtype))
    plain = moc.ops._scan_table

    def run():
        y, fin, saved = moc.ops.launch_scan_forward(*order, None, softplus=True, final_state=True, keep=True)
        return y, fin, *moc.ops.launch_scan_backward(*order, dy, None, saved, softplus=True, has_init=False,
                                                     need_init=False)

    def zero_strides(*args):
        table, held = plain(*args)
        table.x_stride = table.dt_stride = table.b_stride = table.c_stride = 0
        return table, held

    want = run()
    with pytest.MonkeyPatch.context() as m:
        m.setattr(moc.ops, "_scan_table", zero_strides)
        got = run()
    assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)
    assert want[0].abs().sum() > 0


def test_python_functions_are_the_host_modules(monkeypatch):
    """Without the host module the Python functions make the same calls."""
    def everything():
        out = []
        w, b = dev(rnd(96, seed=2)).requires_grad_(), dev(rnd(96, seed=3, dtype=BF16)).requires_grad_()
        cw = dev(rnd(4, 96, seed=4)).requires_grad_()
        x = dev(rnd(2, 70, 96, seed=1, dtype=BF16)).requires_grad_()
        cu = torch.tensor([0, 5, 70], dtype=torch.int32, device=DEV)
        ins = {k: dev(v).requires_grad_() for k, v in scan_inputs((2, 70), 4, 24, 2, 16, BF16, par=F32).items()}
        one = lambda k: {q: (v[0] if v.ndim > 1 else v) for q, v in k.items()}  # noqa: E731
        init = dev(rnd(2, 4, 24, 16, seed=9)).requires_grad_()
        for y in (moc.layer_norm(x, w, b), moc.layer_norm(x), moc.causal_conv(x, cw, b, "silu")[0],
                  moc.causal_conv(x[0], cw, cu_seqlens=cu, max_seqlen=65)[0],
                  moc.selective_scan(**ins)[0], moc.selective_scan(**one(ins), cu_seqlens=cu, max_seqlen=65)[0],
                  *moc.selective_scan(**ins, cache=init, output_final_state=True)):
            leaves = [t for t in (x, w, b, cw, init, *ins.values())]
            out += [y, *[g for g in torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True,
                                                              allow_unused=True)
                         if g is not None]]
        with torch.no_grad():
            out += moc.causal_conv(x, cw, b, "silu", output_final_state=True)
            c = out[-1].clone()
            out += moc.causal_conv(x, cw, b, cache=c, output_final_state=True)
            out += moc.causal_conv(x[:, :1], cw, b, cache=c, output_final_state=True)
            out += moc.selective_scan(**ins, output_final_state=True)
            c = out[-1].clone()
            out += moc.selective_scan(**{k: (v[:, 1:2] if v.ndim > 1 else v) for k, v in ins.items()}, cache=c,
                                      output_final_state=True)
        return out

    here = everything()
    monkeypatch.setattr(_lib, "_host", _lib._NoHost)
    there = everything()
    assert len(here) == len(there) and all(torch.equal(a, b) for a, b in zip(here, there))
