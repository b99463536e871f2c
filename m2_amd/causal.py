"""The parts of a causal mixer: short causal convolution, selective state space scan and group norm with an activation, for whole prompts, for training and, the
first two, for one token more.

The reference mixes sequences with both sides in view (`MonarchMixerSequenceMixing`: short convolution of three, gates and long convolutions,
bert/src/mm/monarch_mixer_sequence_mixer.py:100-154); these are their counterparts where a position may use only what lies before it.  Hidden states are
(batch, positions, channels), fp32 or bf16 on the GPU; parameters and the scan's states are fp32.  Arithmetic is fp32, results are rounded once.
Rows may lie any distance apart (one half of a projection's result, say; the scan copies what lies 2^24 values apart); other layouts are copied.  All of them are differentiable once in every tensor but
`lengths`; the steps are not.

Inside a stream capture a forward that asks for gradients is refused while a graph made on another stream still holds one of its leaves.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops

Tensor = torch.Tensor


def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None, state: Optional[Tensor] = None,
                lengths: Optional[Tensor] = None, return_state: bool = False):
    """y[:, t] = act(bias + sum_k weight[:, k] x[:, t - K + 1 + k]) of x (B, L, C), B at most 65535, each channel on its own; weight (C, K), K 1 to 8, bias (C); `activation` None or
    "silu".

    `state` (B, K - 1, C) of x's type: the inputs ahead of the first position, oldest first (None: zeros).  `lengths` (B) int64: sequence b ends there
    (values outside 0 .. L count as the nearest); what lies behind is not read, y and gradients are 0 there.  With `return_state`: (y, state), the last K - 1 inputs of each
    sequence, which the next part or `causal_conv_step` goes on from."""
    y, last = ops.causal_conv(x, weight, bias, activation, state, lengths, return_state)
    return (y, last) if return_state else y


def causal_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
                     out_state: Optional[Tensor] = None) -> Tensor:
    """`causal_conv` of one position more: x (B, C) -> (B, C), any number of sequences (of 2^31 values of x).  `state` (contiguous) moves on in place, or stays and the next one goes to `out_state`."""
    return ops.causal_conv_step(x, state, weight, bias, activation, out_state)


def selective_scan(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor] = None, z: Optional[Tensor] = None,
                   dt_bias: Optional[Tensor] = None, dt_softplus: bool = False, state: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                   return_state: bool = False):
    """For every channel c and each of its N states (1 to 256), along the positions t:

        d = dt + dt_bias, softplus of it with `dt_softplus`      h[t] = exp(d[t] A[c]) h[t - 1] + d[t] x[t] B[t]      y[t] = (C[t] . h[t] + D[c] x[t]) silu(z[t])

    x, dt, z (B, L, channels); B and C (B, L, N), or (B, L, groups, N) with a group for channels / groups neighbouring channels; A (channels, N); D, dt_bias
    (channels).  `state` (B, channels, N): the states ahead of the first position (None: zeros).  `lengths` as in `causal_conv`.  With `return_state`:
    (y, state), the states behind each sequence's last position.

    Positions are worked on side by side, so results differ in rounding from one step after another, and so do states beyond fp32's range.  At most 2^20 channels, 2^26 of all
    sequences, and below 2^32 values of B."""
    y, last = ops.selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state, lengths, return_state)
    return (y, last) if return_state else y


def selective_scan_step(x: Tensor, dt: Tensor, state: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor] = None, z: Optional[Tensor] = None,
                        dt_bias: Optional[Tensor] = None, dt_softplus: bool = False, out_state: Optional[Tensor] = None) -> Tensor:
    """`selective_scan` of one position more: x, dt, z (B, channels), B and C (B, N) or (B, groups, N) -> (B, channels).  `state` (contiguous) moves on in place,
    or stays and the next one goes to `out_state`."""
    return ops.selective_scan_step(x, dt, state, A, B, C, D, z, dt_bias, dt_softplus, out_state)


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5, activation: Optional[str] = None) -> Tensor:
    """act((x - mean) / sqrt(var + eps) * weight + bias) of x (N, ..., C), mean and (biased) variance of each sample over all positions between the first and the last
    dimension and over each of `groups` groups of neighbouring channels; weight, bias (C); `activation` None, "silu" or "gelu" (erf).

    (tokens, C) normalises each token by itself, heads of channels say; (B, L, C) whole sequences, padding included.  At most 2^20 channels and 2^36 values, and below 2^24
    groups of all sequences, or of all tokens where a group passes 1024 fp32 or 2048 bf16 channels (256 where sizes or addresses are odd)."""
    return ops.group_norm(x, groups, weight, bias, eps, activation)
