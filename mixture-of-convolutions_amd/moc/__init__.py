"""Mixture-of-Convolutions on MI355X: drop-in for the reference ``moc`` package.

The forward, backward and decode paths run as hand-written gfx950 HIP kernels
in libmoc_hip.so, reached through a C ABI (include/moc_hip.h).  Next to the layers
stand the other operators of a block around them: a causal convolution with one
kernel for every token, the selective state space scan that such convolutions
feed, and layer norm (which makes the routing input).
"""
from .api import MoC, MoCGroup, moc_hip, moc_triton, router_linear
from .blocks import (CausalConv, LayerNorm, SelectiveScan, causal_conv, layer_norm,
                     selective_scan)
from .optim import match_lr_to_init_std, match_weight_decay_to_lr, moc_fan_in_std

__all__ = [
    "MoC",
    "MoCGroup",
    "moc_triton",
    "moc_hip",
    "router_linear",
    "CausalConv",
    "SelectiveScan",
    "LayerNorm",
    "causal_conv",
    "selective_scan",
    "layer_norm",
    "moc_fan_in_std",
    "match_lr_to_init_std",
    "match_weight_decay_to_lr",
]
