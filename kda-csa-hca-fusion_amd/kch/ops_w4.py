"""Projections of a decode step with 4-bit weights and group scales.

``linear_w4``    ``x W^T (+ residual)`` of a few rows on ``kch_linear_w4``
``quantize_w4``  a weight to its codes, scales and zero points (once, at load time)
``W4Linear``     a module that holds them in place of ``nn.Linear`` (no bias)

Codes are ``[N, K / 2]`` uint8, two a byte (low nibble: even k), scales ``[K /
group, N]`` in the activations' dtype, zero points ``[K / group, N]`` uint8 or none (8):
``W[n, k] = scales[k // group, n] * (code[n, k] - zeros[k // group, n])``.
Forward only.
"""

from __future__ import annotations

import torch
from torch import nn

from . import _lib

_GROUPS = (32, 64, 128)


def linear_w4(x, packed, scales, zeros=None, *, residual=None):
    """``x W^T`` ``[..., N]`` in ``x.dtype`` (bf16 or fp16), plus ``residual``; fp32 sums,
    rounded once. The group is ``K / scales.shape[0]``. Made for the few rows of a decode
    step; any number is taken, each 16 reading the weights again (from 64 rows of a large
    weight, or 512 of a small one, the 16-bit product is faster)."""
    fn = "linear_w4"
    if not (x.is_cuda and packed.is_cuda):
        _lib.require_gpu(fn, x, packed)
    dt, dev = x.dtype, x.get_device()
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise TypeError(f"{fn}: x must be bfloat16 or float16, got {dt}")
    if packed.dtype is not torch.uint8 or packed.dim() != 2 or not packed.is_contiguous() \
            or packed.get_device() != dev:
        raise ValueError(f"{fn}: packed must be a contiguous uint8 [N, K / 2] tensor on {x.device}, got "
                         f"{packed.dtype} {tuple(packed.shape)}")
    N, K = packed.shape
    K *= 2
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"{fn}: x {tuple(x.shape)} does not have the weights' K={K} columns")
    if scales.dim() != 2 or scales.shape[1] != N or scales.dtype is not dt or not scales.is_contiguous() \
            or scales.get_device() != dev:
        raise ValueError(f"{fn}: scales must be a contiguous {dt} [K / group, {N}] tensor on {x.device}, got "
                         f"{scales.dtype} {tuple(scales.shape)}")
    ng = scales.shape[0]
    group = K // ng if ng and K % ng == 0 else 0
    if group not in _GROUPS:
        raise ValueError(f"{fn}: {ng} rows of scales for K={K}: a group has {_GROUPS} columns")
    if zeros is not None and (zeros.dtype is not torch.uint8 or zeros.shape != scales.shape
                              or not zeros.is_contiguous() or zeros.get_device() != dev):
        raise ValueError(f"{fn}: zeros must be a contiguous uint8 {tuple(scales.shape)} tensor on {x.device}")
    if torch.is_grad_enabled() and (x.requires_grad or scales.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        raise NotImplementedError(f"{fn}: no gradients (call it under torch.no_grad())")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    M = x2.shape[0]
    ldx, one = x2.stride()
    if M == 1:
        ldx = K
    if one != 1 or ldx % 8 or ldx < K or x2.data_ptr() % 16:
        x2 = x2.detach().clone(memory_format=torch.contiguous_format)
        ldx = K
    if packed.data_ptr() % 16:
        packed = packed.clone()
    y = torch.empty(*x.shape[:-1], N, device=x.device, dtype=dt)
    r2, ldr = None, 0
    if residual is not None:
        if residual.shape != y.shape or residual.dtype is not dt or residual.get_device() != dev:
            raise ValueError(f"{fn}: residual must be {tuple(y.shape)} {dt} on {x.device}, got "
                             f"{tuple(residual.shape)} {residual.dtype}")
        r2 = residual if residual.dim() == 2 else residual.reshape(M, N)
        ldr, one = r2.stride()
        if one != 1 or ldr < N:
            r2 = r2.detach().clone(memory_format=torch.contiguous_format)
            ldr = N
    _lib.call_on(dev, "kch_linear_w4", x2.data_ptr(), ldx, packed.data_ptr(), scales.data_ptr(),
                 None if zeros is None else zeros.data_ptr(), None if r2 is None else r2.data_ptr(), ldr,
                 y.data_ptr(), N, M, N, K, group, 1 if dt is torch.bfloat16 else 2)
    return y


def quantize_w4(weight, group_size=128, *, zero_points=True, dtype=None):
    """``(packed, scales, zeros)`` of a weight ``[N, K]``, rounded to nearest group by group.

    With zero points a group's codes 0 .. 15 span its range (0 included); without, they are
    -8 .. 7 times a scale of its largest magnitude over 7. ``dtype``: of the scales (the
    weight's, where that is bf16 or fp16, else bf16)."""
    fn = "quantize_w4"
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"{fn}: weight must be a floating-point [N, K] tensor, got {weight.dtype} "
                         f"{tuple(weight.shape)}")
    N, K = weight.shape
    if group_size not in _GROUPS or K < group_size or K % group_size:
        raise ValueError(f"{fn}: group_size={group_size} must be one of {_GROUPS} and divide K={K}")
    if dtype is None:
        dtype = weight.dtype if weight.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{fn}: scales are bfloat16 or float16, got {dtype}")
    w = weight.detach().float().reshape(N, K // group_size, group_size)
    if zero_points:
        lo, hi = w.amin(-1).clamp_max(0.0), w.amax(-1).clamp_min(0.0)
        s = ((hi - lo) / 15).to(dtype)
    else:
        s = (w.abs().amax(-1) / 7).to(dtype)
    sf = s.float()
    inv = torch.where(sf > 0, 1 / sf, torch.zeros_like(sf))
    z = (-lo * inv).round().clamp(0, 15) if zero_points else torch.full_like(sf, 8.0)
    codes = (w * inv[..., None] + z[..., None]).round().clamp(0, 15).to(torch.uint8).view(N, K)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return (packed.contiguous(), s.t().contiguous(),
            z.to(torch.uint8).t().contiguous() if zero_points else None)


class W4Linear(nn.Module):
    """``nn.Linear`` without bias on 4-bit weights; ``forward(x, residual)`` adds the residual
    in the same launch. Its buffers load and save with the model."""

    def __init__(self, packed, scales, zeros=None):
        super().__init__()
        self.register_buffer("packed", packed)
        self.register_buffer("scales", scales)
        self.register_buffer("zeros", zeros)

    @classmethod
    def from_linear(cls, linear, group_size=128, *, zero_points=True, dtype=None):
        """From an ``nn.Linear`` without bias."""
        if linear.bias is not None:
            raise ValueError("W4Linear: a bias is not supported")
        return cls(*quantize_w4(linear.weight, group_size, zero_points=zero_points, dtype=dtype))

    @property
    def in_features(self) -> int:
        return 2 * self.packed.shape[1]

    @property
    def out_features(self) -> int:
        return self.packed.shape[0]

    def forward(self, x, residual=None):
        return linear_w4(x, self.packed, self.scales, self.zeros, residual=residual)


__all__ = ["W4Linear", "linear_w4", "quantize_w4"]
