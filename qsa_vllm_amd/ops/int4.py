"""Linear layers with 4-bit weights (``csrc/int4_linear.hip``).

A weight ``[out_features, in_features]`` is kept as 4-bit codes with one scale
(and, if wanted, one zero point) per output and group of 32, 64 or 128 inputs:
``w = (code - zero) * scale``, zero 8 where none is given. ``int4_pack`` lays a
checkpoint's codes out for the kernel once, ``int4_quantize`` makes codes from
a bf16 or fp16 weight by rounding to the nearest, ``int4_linear`` multiplies.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _torch_ops  # noqa: F401  (registers torch.ops.yulan_qsa_kernels)
from ._torch_ops import _require

__all__ = ["Int4Weight", "int4_linear", "int4_pack", "int4_quantize"]

_TILE_N, _TILE_K = 16, 128
_PACK_CODES = 1 << 26  # codes laid out at a time


@dataclass(frozen=True)
class Int4Weight:
    """A packed weight: tiles of 16 outputs x 128 inputs, the last ones padded
    (the layout is the C ABI's, ``qsa_int4_linear``)."""

    codes: torch.Tensor            # int32 [n tiles, k tiles, 64, 4]
    scales: torch.Tensor           # bf16 / fp16 [n tiles, k tiles, 16, 128 / group size]
    zeros: torch.Tensor | None     # uint8, shaped like scales
    out_features: int
    in_features: int
    group_size: int

    @property
    def dtype(self) -> torch.dtype:
        return self.scales.dtype

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self) -> torch.Tensor:
        """The weight ``[out_features, in_features]`` in fp32 (for checks)."""
        nt, kt = self.codes.shape[:2]
        shift = torch.tensor([4 * (i // 2) + 16 * (i % 2) for i in range(8)], device=self.device,
                             dtype=torch.int32)
        c = (self.codes.view(nt, kt, 4, 16, 4, 1) >> shift) & 15     # [nt, kt, g, n, j, i]
        c = c.permute(0, 3, 1, 4, 2, 5).reshape(nt * _TILE_N, kt * _TILE_K).float()

        def spread(t):
            t = t.permute(0, 2, 1, 3).reshape(nt * _TILE_N, -1).float()
            return t.repeat_interleave(self.group_size, dim=1)

        zero = 8.0 if self.zeros is None else spread(self.zeros)
        return ((c - zero) * spread(self.scales))[:self.out_features, :self.in_features]


def _check_group(group_size):
    _require(group_size in (32, 64, 128), f"group size must be 32, 64 or 128, got {group_size}")


def int4_pack(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
              group_size: int = 128) -> Int4Weight:
    """Lay out ``codes`` (uint8 ``[out, in]``, 0..15; higher bits are ignored),
    ``scales`` (bf16 or fp16 ``[out, ceil(in / group_size)]``) and ``zeros``
    (uint8, shaped like ``scales``, 0..15; 8 everywhere without) for the kernel.
    The last group of a row may be short. Any strides, CPU or GPU."""
    _check_group(group_size)
    _require(codes.dim() == 2 and codes.dtype == torch.uint8, "codes must be uint8 [out, in]")
    n, k = codes.shape
    _require(k > 0, "codes must have input features")
    groups = -(-k // group_size)
    _require(scales.dtype in (torch.bfloat16, torch.float16) and tuple(scales.shape) == (n, groups),
             f"scales must be bf16 or fp16 [{n}, {groups}]")
    _require(scales.device == codes.device, "scales must be on the device of codes")
    if zeros is not None:
        _require(zeros.dtype == torch.uint8 and tuple(zeros.shape) == (n, groups),
                 f"zeros must be uint8 [{n}, {groups}]")
        _require(zeros.device == codes.device, "zeros must be on the device of codes")
    nt, kt = -(-n // _TILE_N), -(-k // _TILE_K)
    all_groups = kt * (_TILE_K // group_size)
    packed = torch.empty(nt, kt, 64, 4, dtype=torch.int32, device=codes.device)
    step = max(1, _PACK_CODES // (kt * _TILE_K * _TILE_N))
    for t in range(0, nt, step):
        part = codes[t * _TILE_N:(t + step) * _TILE_N]
        tiles = min(step, nt - t)
        full = codes.new_full((tiles * _TILE_N, kt * _TILE_K), 8 if zeros is None else 0)
        full[:part.shape[0], :k] = part
        if zeros is not None and k < groups * group_size:
            # a short last group is filled up with its zero point
            last = zeros[t * _TILE_N:(t + step) * _TILE_N, -1:]
            full[:part.shape[0], k:groups * group_size] = last
        # [tile, n, k tile, j, g, i] -> words [tile, k tile, g, n, j]
        c = full.view(tiles, _TILE_N, kt, 4, 4, 8).permute(0, 2, 4, 1, 3, 5).to(torch.int32) & 15
        word = c[..., 0].clone()
        for i in range(1, 8):
            word |= c[..., i] << (4 * (i // 2) + 16 * (i % 2))
        packed[t:t + tiles] = word.reshape(tiles, kt, 64, 4)

    def by_tile(t):
        full = t.new_zeros(nt * _TILE_N, all_groups)
        full[:n, :groups] = t
        return full.view(nt, _TILE_N, kt, -1).permute(0, 2, 1, 3).contiguous()

    return Int4Weight(packed, by_tile(scales), None if zeros is None else by_tile(zeros & 15), n, k,
                      group_size)


def int4_quantize(weight: torch.Tensor, *, group_size: int = 128,
                  zero_points: bool = False) -> Int4Weight:
    """Round a bf16 or fp16 weight ``[out, in]`` to 4 bits: per group the scale
    ``max |w| / 7`` about code 8, or with ``zero_points`` ``(max - min) / 15``
    over a range that holds 0. Scales are rounded to the weight's type first, so
    each code is the nearest to ``w / scale``. Infinities, NaN and
    values from 2^127 on are refused."""
    _check_group(group_size)
    _require(weight.dim() == 2 and weight.dtype in (torch.bfloat16, torch.float16),
             "weight must be bf16 or fp16 [out, in]")
    n, k = weight.shape
    _require(k > 0, "weight must have input features")
    groups = -(-k // group_size)
    codes = torch.empty(n, k, dtype=torch.uint8, device=weight.device)
    scales = torch.empty(n, groups, dtype=weight.dtype, device=weight.device)
    zeros = torch.empty(n, groups, dtype=torch.uint8, device=weight.device) if zero_points else None
    step = max(1, _PACK_CODES // max(k, 1))
    for r in range(0, n, step):
        w = weight[r:r + step].float()
        # (past 2^127 a group's range, or its dequantized ends, pass fp32's)
        _require(bool((w.abs() < 2.0 ** 127).all()), "weight must be finite and below 2^127")
        w = torch.nn.functional.pad(w, (0, groups * group_size - k)).view(-1, groups, group_size)
        if zero_points:
            low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
            scale = (high - low) / 15
        else:
            scale = w.abs().amax(-1) / 7
        scale = scale.to(weight.dtype)
        unit = torch.where(scale == 0, torch.ones_like(scale), scale).float()
        zero = torch.full_like(unit, 8.0)
        if zero_points:
            zero = (-low / unit).round().clamp(0, 15)
            zeros[r:r + step] = zero.to(torch.uint8)
        c = (w / unit[..., None] + zero[..., None]).round().clamp(0, 15)
        codes[r:r + step] = c.view(-1, groups * group_size)[:, :k].to(torch.uint8)
        scales[r:r + step] = scale
    return int4_pack(codes, scales, zeros, group_size=group_size)


def int4_linear(x: torch.Tensor, weight: Int4Weight, bias: torch.Tensor | None = None, *,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` for ``x`` ``[..., in_features]`` of the weight's
    type (bf16 or fp16), summed in fp32 and rounded once. ``out`` (only for a
    two-dimensional ``x``) receives the result. Made for few rows, where it
    streams the 4-bit weight once (per 64 rows); it is right for any number, and
    for any values: results that are not finite at first (infinities in a row, or
    bf16 values past 2^112) are taken again term by term, which is slow."""
    rows = x
    if x.dim() != 2:
        _require(x.dim() >= 1 and out is None, "x must be [..., in_features]; out needs a 2-D x")
        rows = x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.reshape(0, 0)
    if out is None:
        out = torch.empty(rows.shape[0], weight.out_features, dtype=x.dtype, device=x.device)
    torch.ops.yulan_qsa_kernels.int4_linear(rows, weight.codes, weight.scales, weight.zeros, bias,
                                            out, weight.in_features, weight.out_features,
                                            weight.group_size)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], weight.out_features)
