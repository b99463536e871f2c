"""Linear layers with weights in 4 bits and a scale for each group of a row, for the few rows a masked-LM head answers with.

The reference has none; they stand in for `nn.Linear` in its masked-LM head (bert/src/bert_layers.py:862-877,1027-1052), whose decoder reads
all word embeddings for each handful of masked places.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import ops
from .blockdiag import _fp32_path

GROUPS = (32, 64, 128)
MAX_SIZE = 2 ** 30


def quantize_int4(weight: torch.Tensor, group_size: int = 64) -> Tuple[torch.Tensor, torch.Tensor]:
    """weight (N, K) -> (codes (N, ceil(K / 2)) uint8, even k in the low half of a byte; scales (N, ceil(K / group_size)) bf16), the weight being
    about (code - 8) * scale: scale = largest magnitude of the group / 7, rounded to bf16, codes to the nearest."""
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight: expected (N, K), got {tuple(weight.shape)}")
    if group_size not in GROUPS:
        raise ValueError(f"group_size must be one of {GROUPS}, got {group_size}")
    N, K = weight.shape
    w = weight.detach().float()
    w = torch.nn.functional.pad(w, (0, -K % group_size)).view(N, -1, group_size)
    scales = (w.abs().amax(-1) / 7).to(torch.bfloat16)
    s = scales.float().unsqueeze(-1)
    codes = (w / torch.where(s == 0, torch.ones_like(s), s)).round_().clamp_(-8, 7).add_(8).nan_to_num_(nan=8.0).to(torch.uint8).view(N, -1)
    return codes[:, 0:K + K % 2:2] | (codes[:, 1:K + K % 2:2] << 4), scales


class Int4Linear(nn.Module):
    """y = act(x W^T + bias), W (out_features, in_features) as (code - 8) * scale.

    x fp32 or bf16 (..., in_features) on the GPU, rows any distance apart; y of the same type (bf16 for fp32 input under CUDA autocast); products are exact,
    sums fp32, rounded once.  Large products of many rows take x as half-precision parts of its row's size: fp32
    values are rounded to 23 bits, and what is far below its row's largest loses more (fp32 values from 2^-27 of it on, by 2^-50 of it; bf16 from 2^-31 on, by 2^-39; scales from 2^-27 of theirs
    on, by 2^-36).  Rows of magnitudes above 2^115 may overflow inside a sum, fp32 values may be off by 2^-131 and results by 2^-144; a row
    that holds an infinity or NaN has no finite result.  Weights are constants: an input or bias that asks for gradients is refused.  `weight` holds codes and scales in the kernel's order
    (include/m2_amd.h); make it with `from_linear`, `from_weight` or `from_packed`.

    Meant for few rows: from some 250 to 1000 rows of bf16 on, by size, torch's product with weights kept in bf16 is faster (at 768 -> 30528 1024 rows take 64 us here and 63 there, 2048 120 and 105)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group_size: int = 64, device=None):
        super().__init__()
        if group_size not in GROUPS:
            raise ValueError(f"group_size must be one of {GROUPS}, got {group_size}")
        if not (0 < in_features <= MAX_SIZE and 0 < out_features <= MAX_SIZE):
            raise ValueError(f"in_features and out_features must be positive and at most 2^30, got {in_features}, {out_features}")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        nbytes = ops.int4_weight_bytes(out_features, in_features, group_size)
        weight = torch.zeros(nbytes, dtype=torch.uint8, device=device)      # scales 0: W = 0
        weight[nbytes - -(-out_features // 16) * 64:].view(torch.float32).fill_(1)
        self.register_buffer("weight", weight)
        self.register_buffer("bias", torch.zeros(out_features, dtype=torch.float32, device=device) if bias else None)

    @classmethod
    def from_packed(cls, codes: torch.Tensor, scales: torch.Tensor, in_features: int, group_size: int = 64,
                    bias: Optional[torch.Tensor] = None) -> "Int4Linear":
        """From what `quantize_int4` gives (or another quantizer of the same form)."""
        N, K = codes.shape[0], in_features
        if group_size not in GROUPS:
            raise ValueError(f"group_size must be one of {GROUPS}, got {group_size}")
        if codes.dtype != torch.uint8 or tuple(codes.shape) != (N, (K + 1) // 2):
            raise ValueError(f"codes: expected uint8 ({N}, {(K + 1) // 2}), got {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (N, -(-K // group_size)):
            raise ValueError(f"scales: expected bfloat16 ({N}, {-(-K // group_size)}), got {scales.dtype} {tuple(scales.shape)}")
        if bias is not None and tuple(bias.shape) != (N,):
            raise ValueError(f"bias: expected ({N},), got {tuple(bias.shape)}")
        self = cls(K, N, bias is not None, group_size, device="meta")
        self.weight = _in_tiles(codes.detach(), scales.detach(), K, group_size)
        assert self.weight.numel() == ops.int4_weight_bytes(N, K, group_size)
        if bias is not None:
            self.bias = bias.detach().to(torch.float32).clone()
        return self

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, group_size: int = 64) -> "Int4Linear":
        codes, scales = quantize_int4(weight, group_size)
        return cls.from_packed(codes, scales, weight.shape[1], group_size, bias)

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 64) -> "Int4Linear":
        return cls.from_weight(linear.weight, linear.bias, group_size)

    def packed(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """(codes, scales) as `from_packed` takes them."""
        return _out_of_tiles(self.weight, self.out_features, self.in_features, self.group_size)

    def dequantized(self) -> torch.Tensor:
        """The weight that the codes stand for, (out_features, in_features) fp32."""
        codes, scales = self.packed()
        values = torch.stack((codes & 15, codes >> 4), -1).view(self.out_features, -1)[:, :self.in_features].float() - 8
        return values * scales.float().repeat_interleave(self.group_size, 1)[:, :self.in_features]

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, group_size={self.group_size}"

    def forward(self, x: torch.Tensor, activation: Optional[str] = None) -> torch.Tensor:
        """`activation`: None, or "gelu" (erf)."""
        if x.shape[-1:] != (self.in_features,):
            raise ValueError(f"x: expected (..., {self.in_features}), got {tuple(x.shape)}")
        if x.dtype == torch.float32 and not _fp32_path(x):
            x = x.to(torch.bfloat16)
        buffers = self._buffers      # (nn.Module's own look-up takes 0.35 us for each)
        bias = buffers["bias"] if "bias" in buffers else self.bias
        if bias is not None and bias.dtype != torch.float32:
            bias = bias.float()
        return ops.int4_linear(x, buffers["weight"], self.out_features, self.group_size, bias, activation)


def _in_tiles(codes: torch.Tensor, scales: torch.Tensor, K: int, group: int) -> torch.Tensor:
    """The order that include/m2_amd.h states, tile by tile."""
    N = codes.shape[0]
    nt, kt = -(-N // 16), -(-K // 128)
    full = torch.full((nt * 16, kt * 128), 8, dtype=torch.uint8, device=codes.device)
    full[:N, 0:K:2] = codes[:, :(K + 1) // 2] & 15
    if K > 1:
        full[:N, 1:K:2] = codes[:, :K // 2] >> 4
    s = torch.zeros(nt * 16, kt * 128 // group, dtype=torch.bfloat16, device=codes.device)
    s[:N, :scales.shape[1]] = scales
    # (tile n, row, tile k, step, eighth, half byte's pair, value pair) -> a lane's words; value j of eight is 2 r + half, its place 4 half words of r
    v = full.view(nt, 16, kt, 4, 4, 2, 2, 2)                  # ..., r // 2, r % 2, half
    v = v.permute(0, 2, 4, 1, 3, 7, 5, 6)                     # nt, kt, eighth, row, step, half, r // 2, r % 2
    tiles = (v[..., 0] | (v[..., 1] << 4)).reshape(nt, kt, 1024)
    s = s.view(nt, 16, kt, 128 // group).permute(0, 2, 1, 3).contiguous().view(torch.uint8).view(nt, kt, -1)
    # the power of two that takes a row's largest scale to [1 / 2, 1)
    most = scales.float().abs().amax(1)
    exponent = torch.where(torch.isfinite(most) & (most > 0), torch.frexp(most).exponent, torch.zeros_like(most, dtype=torch.int32))
    factor = torch.full((nt * 16,), 127, dtype=torch.int32, device=codes.device)
    factor[:N] -= exponent.clamp(-120, 120)
    factor <<= 23      # as fp32; torch.ldexp multiplies by pow(2, e), which is not always a power of two on the GPU
    return torch.cat((torch.cat((tiles, s), -1).reshape(-1), factor.view(torch.uint8)))


def _out_of_tiles(weight: torch.Tensor, N: int, K: int, group: int) -> Tuple[torch.Tensor, torch.Tensor]:
    nt, kt = -(-N // 16), -(-K // 128)
    w = weight[:weight.numel() - nt * 16 * 4].view(nt, kt, -1)
    v = w[..., :1024].reshape(nt, kt, 4, 16, 4, 2, 2)         # nt, kt, eighth, row, step, half, r // 2
    v = torch.stack((v & 15, v >> 4), -1).permute(0, 3, 1, 4, 2, 6, 7, 5).reshape(nt * 16, kt * 128)[:N]
    s = w[..., 1024:].contiguous().view(torch.bfloat16).view(nt, kt, 16, 128 // group).permute(0, 2, 1, 3).reshape(nt * 16, -1)
    even = K + K % 2
    return v[:, 0:even:2] | (v[:, 1:even:2] << 4), s[:N, :-(-K // group)].contiguous()
