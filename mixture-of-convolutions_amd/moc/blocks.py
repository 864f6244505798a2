"""The operators that stand next to the MoC layers in a block, with the layers'
contract: fixed-length ``[B, T, ..]`` or packed inputs behind ``cu_seqlens``,
``cache`` / ``output_final_state`` for serving, and with a cache and one token per
sequence the decode step, in place on the cache and not differentiable.

* ``causal_conv`` / ``CausalConv``: the short causal convolution with one kernel per
  channel for every token (what a MoC layer with a single route of weight 1 computes);
* ``selective_scan`` / ``SelectiveScan``: the selective state space scan that such
  convolutions feed;
* ``layer_norm`` / ``LayerNorm``: the norm whose output the MoC layers route by.

All run as hand-written HIP kernels of libmoc_hip.so, forward, backward and step;
there is no fallback.  Calls go through the host module (csrc/moc_host.cpp) where they
are ones that it takes; the Python functions below are the same calls for all others.
Every launch below stands in an autograd function, also where no gradient is asked for, so
that a tracer records it and an input with a tangent is refused (a launch by itself is seen
by neither).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .api import SUPPORTED_DTYPES, _final_state, _is_length, activation_flag


# ---------------------------------------------------------------------------
# validation

def _check_tensors(x: torch.Tensor, **others: torch.Tensor | None) -> None:
    if not x.is_cuda or any(t is not None and not t.is_cuda for t in others.values()):
        raise ValueError(f"x, {', '.join(others)} must all be CUDA tensors")
    if any(t is not None and t.device != x.device for t in others.values()):
        raise ValueError(f"x, {', '.join(others)} must be on the same CUDA device")
    if x.dtype not in SUPPORTED_DTYPES:
        raise TypeError(f"unsupported x dtype: {x.dtype}")
    for name, t in others.items():
        if t is not None and not t.is_floating_point():
            raise TypeError(f"{name} must be floating point, got {t.dtype}")


def _check_packing(x: torch.Tensor, cu_seqlens, max_seqlen, cache, output_final_state) -> None:
    """The packed arguments, by the rules of the MoC layers."""
    if cu_seqlens is None:
        if max_seqlen is not None:
            raise ValueError("max_seqlen must be None when cu_seqlens is None")
        return
    if cache is not None or output_final_state:
        raise ValueError("cache and output_final_state are only supported for fixed-length inputs")
    if max_seqlen is None:
        raise ValueError("max_seqlen is required for varlen inputs")
    if not cu_seqlens.is_cuda or cu_seqlens.device != x.device:
        raise ValueError("cu_seqlens must be a CUDA tensor on the same device as x")
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be rank-1 with at least two entries")
    if cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise TypeError("cu_seqlens must have dtype torch.int32 or torch.int64")
    if not isinstance(max_seqlen, int) or max_seqlen <= 0:
        raise ValueError("max_seqlen must be a positive Python int")


def _check_state(cache: torch.Tensor, shape: tuple, dtype: torch.dtype, x: torch.Tensor, step: bool) -> None:
    if tuple(cache.shape) != shape:
        raise ValueError(f"cache must have shape {shape}, got {tuple(cache.shape)}")
    if cache.device != x.device or cache.dtype != dtype:
        raise ValueError(f"cache must be a {dtype} tensor on the device of x")
    if step and any(size > 1 and stride == 0 for size, stride in zip(cache.shape, cache.stride())):
        raise ValueError("a step writes its cache in place: no two of its elements may share memory")


def _on_gpu(x) -> bool:
    """Whether the host module is asked first (it hands back what is not its own)."""
    return isinstance(x, torch.Tensor) and x.is_cuda


def _operand(t: torch.Tensor | None) -> torch.Tensor | None:
    """A parameter as the kernels read it: contiguous, fp32, bf16 or fp16."""
    return None if t is None else ops._operand(t)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _written(cache: torch.Tensor) -> None:
    """Tells autograd that a kernel wrote ``cache``."""
    if not cache.is_inference():
        torch.autograd.graph.increment_version(cache)


# ---------------------------------------------------------------------------
# layer norm

class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        y, mean, rstd = ops.launch_norm_forward(x, weight, bias, eps, keep)
        if keep:
            ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*ops.launch_norm_backward(x, weight, bias, dy, mean, rstd, need[0], need[1], need[2]),
                None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis of ``x`` (bf16 or fp32, any rank from 1):
    ``(x - mean) / sqrt(var + eps) * weight + bias`` with fp32 statistics.
    ``weight`` and ``bias`` are ``[dim]`` in any floating dtype, or None."""
    if _on_gpu(x):
        y = _lib.host().norm(x, weight, bias, eps)
        if y is not None:
            return y
    _check_tensors(x, weight=weight, bias=bias)
    if x.ndim < 1 or x.numel() == 0:
        raise ValueError(f"x must have a last axis and no empty one, got shape {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must have shape {(x.shape[-1],)}, got {tuple(t.shape)}")
    x, weight, bias = x.contiguous(), _operand(weight), _operand(bias)
    return _LayerNormFunction.apply(x, weight, bias, float(eps), _wants_grad(x, weight, bias))


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters: weight ones, bias zeros (or none)."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True) -> None:
        super().__init__()
        self.dim = dim
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)


# ---------------------------------------------------------------------------
# causal convolution

class _CausalConvFunction(torch.autograd.Function):
    """Differentiable in x, weight and bias, without a cache."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, cu_seqlens):
        y, _ = ops.launch_conv_forward(x, weight, bias, None, activation_flag=act, cu_seqlens=cu_seqlens)
        ctx.save_for_backward(x, weight, bias, cu_seqlens)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, cu_seqlens = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*ops.launch_conv_backward(x, weight, bias, dy, activation_flag=ctx.act, need_x=need[0],
                                          need_w=need[1], need_b=need[2], cu_seqlens=cu_seqlens), None, None)


class _CausalConvPromptFunction(torch.autograd.Function):
    """Returns (y, final state or None); applied where no gradient is asked for."""

    @staticmethod
    def forward(ctx, x, weight, bias, cache, act, want_state):
        return ops.launch_conv_forward(x, weight, bias, cache, activation_flag=act, final_state=want_state)


class _CausalConvStepFunction(torch.autograd.Function):
    """In place on the cache; applied without gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, cache, act):
        return ops.launch_conv_update(x, weight, bias, cache, activation_flag=act)


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                activation: str | None = None, cache: torch.Tensor | None = None,
                output_final_state: bool = False, cu_seqlens: Optional[torch.Tensor] = None,
                max_seqlen: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``y[t] = act(bias + sum_s weight[s] x[t-(S-1-s)])`` per channel; returns
    ``(y, final state or None)``.

    x ``[B, T, D]``, or packed ``[N, D]`` / ``[1, N, D]`` behind ``cu_seqlens`` (tokens
    outside every sequence start their own history); bf16 or fp32.  weight ``[S, D]``,
    S from 1 to 16 (the last row multiplies the current token, as in a MoC basis); bias
    ``[D]`` or None; any floating dtype.  activation: None, "silu" or "swish".
    cache ``[B, D, S]`` in the x dtype, the newest input last: with T == 1 the step,
    in place on it (returned as the state); with more tokens the history before
    them.  The final state is the last S inputs, as a new tensor."""
    act = activation_flag(activation)
    if _on_gpu(x) and (cu_seqlens is None) == (max_seqlen is None):
        if cu_seqlens is None or (x.ndim == 2 and _is_length(max_seqlen)):
            out = _lib.host().conv(x, weight, bias, cache, act, bool(output_final_state), cu_seqlens)
            if out is not None:
                return out
    _check_tensors(x, weight=weight, bias=bias)
    _check_packing(x, cu_seqlens, max_seqlen, cache, output_final_state)
    restore = False
    if cu_seqlens is not None and x.ndim == 3 and x.shape[0] == 1:
        x, restore = x[0], True
    if x.ndim != (3 if cu_seqlens is None else 2) or weight.ndim != 2:
        raise ValueError("x must be [B,T,D], or [N,D] / [1,N,D] with cu_seqlens, and weight [S,D]")
    S, D = weight.shape
    if x.shape[-1] != D:
        raise ValueError(f"x/weight dimensions disagree: D={x.shape[-1]} vs {D}")
    if bias is not None and tuple(bias.shape) != (D,):
        raise ValueError(f"bias must have shape {(D,)}, got {tuple(bias.shape)}")
    if x.numel() == 0 or weight.numel() == 0:
        raise ValueError("x and weight must not be empty")
    if S > _lib.CONV_MAX_KERNEL:
        raise ValueError(f"kernel_size must be at most {_lib.CONV_MAX_KERNEL}, got {S}")
    x, weight, bias = x.contiguous(), _operand(weight), _operand(bias)
    if cu_seqlens is not None:
        y = _CausalConvFunction.apply(x, weight, bias, act, cu_seqlens.contiguous())
        return (y[None] if restore else y), None
    B, T, _ = x.shape
    if cache is not None:
        _check_state(cache, (B, D, S), x.dtype, x, T == 1)
        if T == 1:
            with torch.no_grad():
                y = _CausalConvStepFunction.apply(x[:, 0], weight, bias, cache, act)
            _written(cache)
            return y[:, None], (cache if output_final_state else None)
    if _wants_grad(x, weight, bias, cache):
        if cache is None:
            y = _CausalConvFunction.apply(x, weight, bias, act, None)
        else:
            # the S - 1 newest cached inputs, then the tokens themselves: one more copy of x and
            # of dy (4 x 4096 x 2048, 4 taps, bf16: 198 us where 91 without a cache), for a
            # backward that knows no cache
            every = torch.cat((cache.transpose(1, 2)[:, 1:], x), 1)
            y = _CausalConvFunction.apply(every, weight, bias, act, None)[:, S - 1:]
        return y, (_final_state(x, cache, S) if output_final_state else None)
    if cache is not None:
        cache = cache.contiguous()
    return _CausalConvPromptFunction.apply(x, weight, bias, cache, act, bool(output_final_state))


class CausalConv(nn.Module):
    """``causal_conv`` with its parameters ``weight`` [kernel_size, dim] and ``bias``
    [dim] (or none), both uniform in +-1/sqrt(kernel_size)."""

    def __init__(self, dim: int, kernel_size: int, activation: str | None = None,
                 bias: bool = True) -> None:
        super().__init__()
        activation_flag(activation)
        self.dim = dim
        self.kernel_size = kernel_size
        self.activation = activation
        self.weight = nn.Parameter(torch.empty(kernel_size, dim))
        self.bias = nn.Parameter(torch.empty(dim)) if bias else None
        bound = 1.0 / math.sqrt(kernel_size)
        for p in self.parameters():
            nn.init.uniform_(p, a=-bound, b=bound)

    def forward(self, x: torch.Tensor, cache: torch.Tensor | None = None,
                output_final_state: bool = False, cu_seqlens: Optional[torch.Tensor] = None,
                max_seqlen: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor | None]:
        return causal_conv(x, self.weight, self.bias, self.activation, cache=cache,
                           output_final_state=output_final_state, cu_seqlens=cu_seqlens,
                           max_seqlen=max_seqlen)

    def step(self, x: torch.Tensor, cache: torch.Tensor | None = None,
             output_final_state: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
        if x.ndim != 3 or x.shape[1] != 1:
            raise ValueError(f"step expects x with shape [B, 1, D], got {tuple(x.shape)}")
        if cache is None:
            cache = x.new_zeros(x.shape[0], self.dim, self.kernel_size)
        return self.forward(x, cache=cache, output_final_state=output_final_state)

    @property
    def state_size(self) -> int:
        return self.dim * self.kernel_size


# ---------------------------------------------------------------------------
# selective scan

class _SelectiveScanFunction(torch.autograd.Function):
    """Returns (y, final state or None)."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, dt_bias, cache, softplus, want_state, cu_seqlens, keep):
        y, fin, saved = ops.launch_scan_forward(x, dt, A, B, C, D, dt_bias, cache, softplus=softplus,
                                                final_state=want_state, keep=keep, cu_seqlens=cu_seqlens)
        if not keep:
            return y, fin
        ctx.save_for_backward(x, dt, A, B, C, D, dt_bias, saved, cu_seqlens)
        ctx.softplus = softplus
        ctx.has_init = cache is not None
        ctx.set_materialize_grads(False)
        return y, fin

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfin):
        *ins, saved, cu_seqlens = ctx.saved_tensors
        if dy is None:
            if dfin is None:
                return (None,) * 12
            dy = torch.zeros_like(ins[0])
        if dfin is not None:
            dfin = dfin.float().contiguous()
        grads = ops.launch_scan_backward(*ins, dy, dfin, saved, softplus=ctx.softplus,
                                         has_init=ctx.has_init, need_init=ctx.needs_input_grad[7],
                                         cu_seqlens=cu_seqlens)
        return (*[g if need else None for g, need in zip(grads, ctx.needs_input_grad)], None, None, None, None)


class _SelectiveScanStepFunction(torch.autograd.Function):
    """In place on the cache; applied without gradients."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, dt_bias, cache, softplus):
        state = cache.contiguous()
        y = ops.launch_scan_update(x, dt, A, B, C, D, dt_bias, state, softplus=softplus)
        if state is not cache:
            cache.copy_(state)
        return y


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                   C: torch.Tensor, D: torch.Tensor | None = None,
                   dt_bias: torch.Tensor | None = None, cache: torch.Tensor | None = None,
                   output_final_state: bool = False, dt_softplus: bool = True,
                   cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None
                   ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Selective state space scan; returns ``(y, final state or None)``.  Per head, with
    a ``[P, N]`` state h::

        u_t = softplus(dt_t + dt_bias)          (dt_softplus=False: dt_t + dt_bias)
        h_t = exp(u_t A) h_{t-1} + u_t x_t (x) B_t
        y_t = h_t C_t + D x_t

    x ``[B, T, H, P]``, dt ``[B, T, H]``, B and C ``[B, T, G, N]`` in one dtype (bf16 or
    fp32; G divides H, heads h of group ``h // (H // G)`` share B and C), or packed, without
    the batch axis or with one of size 1, behind ``cu_seqlens`` (tokens outside every
    sequence are sequences of their own).  A, D and dt_bias ``[H]`` in any floating dtype,
    D and dt_bias or None.  P up to 128, N up to 256.  Slices of a wider projection are
    read in place where a token's values are contiguous.

    cache ``[B, H, P, N]`` fp32: with T == 1 the step, in place on it (returned as the
    state); with more tokens the state before them.  The final state is a new fp32
    tensor.  States and sums are fp32; with bf16 inputs the state and the token-to-token
    weights enter matrix products with 16 bits of significand, so that results are off by
    their own rounding.  An infinity or NaN in one token reaches the outputs of that token
    and later ones of its sequence only.  The exponential of u A summed over up to 64
    neighbouring tokens must be finite in fp32 (it is where u A is not positive)."""
    softplus = bool(dt_softplus)
    if _on_gpu(x) and (cu_seqlens is None) == (max_seqlen is None):
        if cu_seqlens is None or (x.ndim == 3 and _is_length(max_seqlen)):
            out = _lib.host().scan(x, dt, A, B, C, D, dt_bias, cache, softplus, bool(output_final_state),
                                   cu_seqlens)
            if out is not None:
                return out
    _check_tensors(x, dt=dt, A=A, B=B, C=C, D=D, dt_bias=dt_bias)
    _check_packing(x, cu_seqlens, max_seqlen, cache, output_final_state)
    restore = False
    if cu_seqlens is not None and x.ndim == 4 and all(t.ndim > 0 and t.shape[0] == 1 for t in (x, dt, B, C)):
        x, dt, B, C, restore = x[0], dt[0], B[0], C[0], True
    lead = 2 if cu_seqlens is None else 1
    if (x.ndim, dt.ndim, B.ndim, C.ndim) != (lead + 2, lead + 1, lead + 2, lead + 2):
        raise ValueError("x/dt/B/C must be [B,T,H,P]/[B,T,H]/[B,T,G,N]/[B,T,G,N], or the same without the "
                         "batch axis (or with one of size 1) with cu_seqlens")
    if any(t.dtype != x.dtype for t in (dt, B, C)):
        raise TypeError("x, dt, B and C must have the same dtype")
    tokens, (H, P), (G, N) = tuple(x.shape[:lead]), x.shape[-2:], B.shape[-2:]
    if any(tuple(t.shape[:lead]) != tokens for t in (dt, B, C)):
        raise ValueError("x, dt, B and C batch/time shapes differ")
    if dt.shape[-1] != H or tuple(C.shape[-2:]) != (G, N):
        raise ValueError(f"x/dt or B/C dimensions disagree: H={H} vs {dt.shape[-1]}, "
                         f"G,N={(G, N)} vs {tuple(C.shape[-2:])}")
    for name, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None and tuple(t.shape) != (H,):
            raise ValueError(f"{name} must have shape {(H,)}, got {tuple(t.shape)}")
    if min(*tokens, H, P, G, N) <= 0:
        raise ValueError("token, head, channel, group and state counts must all be positive")
    if H % G:
        raise ValueError(f"the groups of B and C must divide the heads: {G} vs {H}")
    if P > _lib.SCAN_MAX_HEAD_DIM or N > _lib.SCAN_MAX_STATE_DIM:
        raise ValueError(f"P must be at most {_lib.SCAN_MAX_HEAD_DIM} and N at most {_lib.SCAN_MAX_STATE_DIM}, "
                         f"got {P} and {N}")
    A, D, dt_bias = _operand(A), _operand(D), _operand(dt_bias)
    if cu_seqlens is not None:
        cu_seqlens = cu_seqlens.contiguous()
    elif cache is not None:
        step = tokens[1] == 1
        _check_state(cache, (tokens[0], H, P, N), torch.float32, x, step)
        if step:
            with torch.no_grad():
                y = _SelectiveScanStepFunction.apply(x, dt, A, B, C, D, dt_bias, cache, softplus)
            _written(cache)
            return y, (cache if output_final_state else None)
        cache = cache.contiguous()
    want = bool(output_final_state)
    y, fin = _SelectiveScanFunction.apply(x, dt, A, B, C, D, dt_bias, cache, softplus, want, cu_seqlens,
                                          _wants_grad(x, dt, A, B, C, D, dt_bias, cache))
    return (y[None] if restore else y), fin


class SelectiveScan(nn.Module):
    """``selective_scan`` with its parameters ``A_log``, ``D`` and ``dt_bias`` [n_heads]
    (``A = -exp(A_log)``, so that states decay).  Inputs are a block's projections:
    x ``[.., n_heads * head_dim]``, dt ``[.., n_heads]``, B and C ``[.., n_groups *
    state_dim]``; y has x's shape.  A starts uniform in [-16, -1], softplus(dt_bias)
    log-uniform in [0.001, 0.1], D at 1."""

    def __init__(self, n_heads: int, head_dim: int, state_dim: int, n_groups: int = 1) -> None:
        super().__init__()
        if n_groups <= 0 or n_heads % n_groups:
            raise ValueError(f"the groups of B and C must divide the heads: {n_groups} vs {n_heads}")
        self.n_heads = n_heads
        self.head_dim = head_dim
        self.state_dim = state_dim
        self.n_groups = n_groups
        u = torch.exp(torch.empty(n_heads).uniform_(math.log(1e-3), math.log(0.1)))
        self.A_log = nn.Parameter(torch.log(torch.empty(n_heads).uniform_(1.0, 16.0)))
        self.D = nn.Parameter(torch.ones(n_heads))
        self.dt_bias = nn.Parameter(u + torch.log(-torch.expm1(-u)))

    def forward(self, x: torch.Tensor, dt: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                cache: torch.Tensor | None = None, output_final_state: bool = False,
                cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None
                ) -> tuple[torch.Tensor, torch.Tensor | None]:
        heads, states = (self.n_heads, self.head_dim), (self.n_groups, self.state_dim)
        for name, t, (m, n) in (("x", x, heads), ("B", B, states), ("C", C, states)):
            if t.ndim < 1 or t.shape[-1] != m * n:
                raise ValueError(f"{name} must have {m * n} channels, got shape {tuple(t.shape)}")
        y, state = selective_scan(x.unflatten(-1, heads), dt, -torch.exp(self.A_log.float()),
                                  B.unflatten(-1, states), C.unflatten(-1, states), self.D, self.dt_bias,
                                  cache=cache, output_final_state=output_final_state,
                                  cu_seqlens=cu_seqlens, max_seqlen=max_seqlen)
        return y.flatten(-2), state

    def step(self, x: torch.Tensor, dt: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
             cache: torch.Tensor | None = None, output_final_state: bool = False
             ) -> tuple[torch.Tensor, torch.Tensor | None]:
        if x.ndim != 3 or x.shape[1] != 1:
            raise ValueError(f"step expects x with shape [B, 1, H*P], got {tuple(x.shape)}")
        if cache is None:
            cache = torch.zeros(x.shape[0], self.n_heads, self.head_dim, self.state_dim,
                                dtype=torch.float32, device=x.device)
        return self.forward(x, dt, B, C, cache=cache, output_final_state=output_final_state)

    @property
    def state_size(self) -> int:
        return self.n_heads * self.head_dim * self.state_dim


__all__ = ["LayerNorm", "CausalConv", "SelectiveScan", "layer_norm", "causal_conv", "selective_scan"]
