"""Weights of expert products in 4 bits: laid out once, then read in place by :func:`brainstorm_amd.jit.grouped_linear_int4`."""
from typing import NamedTuple, Optional

import torch

__all__ = ["Int4Weight", "pack_int4", "quantize_int4"]

_ROWS, _COLUMNS = 16, 128  # a tile of the layout


class Int4Weight(NamedTuple):
    """Weights ``[experts, out_features, in_features]``: ``W_e[n, k] = (q - zero) * scale`` with ``q`` of 4 bits, a ``scale`` and a whole
    ``zero`` for every ``group`` (32, 64 or 128) elements of a row.  ``values`` is uint8 ``[experts, tiles of 16 rows, blocks of 128
    columns, 1024]``: byte ``16 * (16 * g + r) + 4 * j + m`` of a block belongs to row ``r`` of the tile and holds column ``32 * j + 8 * g + m``
    in its low and column ``+ 4`` in its high four bits.  ``scales`` (fp32 / fp16 / bf16) and ``zeros`` (uint8, or None: all 8)
    are ``[experts, tiles of 16 rows, groups, 16]``.  What lies behind the last row or column may hold anything finite."""

    values: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    in_features: int
    out_features: int
    group: int


def _check_group(group: int) -> None:
    if group not in (32, 64, 128):
        raise NotImplementedError(f"groups of {group} elements (32, 64 or 128 are built)")


def _ceil(n: int, by: int) -> int:
    return -(-n // by)


def _packed_values(q: torch.Tensor, into: torch.Tensor) -> None:
    """One expert's ``q`` (uint8 ``[out_features, in_features]``) into its blocks ``[tiles, blocks, 1024]``."""
    tiles, blocks, _ = into.shape
    padded = q.new_zeros(tiles * _ROWS, blocks * _COLUMNS)
    padded[:q.shape[0], :q.shape[1]] = q
    parts = padded.view(tiles, _ROWS, blocks, 4, 4, 2, 4).permute(0, 2, 4, 1, 3, 6, 5)  # [tile, block, g, r, j, m, half]
    into.copy_((parts[..., 0] | (parts[..., 1] << 4)).reshape(into.shape))


def _packed_groups(t: torch.Tensor, tiles: int) -> torch.Tensor:
    """``[experts, out_features, groups]`` as ``[experts, tiles, groups, 16]``."""
    experts, rows, groups = t.shape
    padded = t.new_zeros(experts, tiles * _ROWS, groups)
    padded[:, :rows] = t
    return padded.view(experts, tiles, _ROWS, groups).transpose(2, 3).contiguous()


def _empty_values(experts: int, rows: int, columns: int, device) -> torch.Tensor:
    return torch.empty(experts, _ceil(rows, _ROWS), _ceil(columns, _COLUMNS), 1024, dtype=torch.uint8, device=device)


def pack_int4(values: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, *, group: int = 128) -> Int4Weight:
    """Weights that are in 4 bits already: ``values`` uint8 ``[experts, out_features, in_features]`` of 0 .. 15, ``scales``
    ``[experts, out_features, groups]`` (finite) and ``zeros`` (uint8, of the same shape; 8 without them), ``groups = ceil(in_features /
    group)``.  On the host or the device; a step of loading a model, not of running it."""
    _check_group(group)
    if values.dim() != 3 or values.dtype != torch.uint8:
        raise RuntimeError("values must be a uint8 tensor [experts, out_features, in_features]")
    experts, rows, columns = values.shape
    if scales.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise NotImplementedError("scales must be fp32, fp16 or bf16")
    if scales.shape != (experts, rows, _ceil(columns, group)):
        raise RuntimeError("scales must be [experts, out_features, groups]")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise RuntimeError("zeros must be a uint8 tensor of the scales' shape")
    if values.numel() and int(values.max()) > 15:
        raise RuntimeError("values must be 0 .. 15")
    if not bool(torch.isfinite(scales).all()):
        raise RuntimeError("scales must be finite")
    packed = _empty_values(experts, rows, columns, values.device)
    for e in range(experts):
        _packed_values(values[e], packed[e])
    tiles = packed.shape[1]
    return Int4Weight(packed, _packed_groups(scales, tiles), None if zeros is None else _packed_groups(zeros, tiles), columns, rows, group)


def quantize_int4(weight: torch.Tensor, group: int = 128, *, zeros: bool = False, scale_dtype: Optional[torch.dtype] = None) -> Int4Weight:
    """``weight`` (``[experts, out_features, in_features]``, fp32 / fp16 / bf16) rounded to 4 bits.  Over every ``group`` elements of a row
    ``scale = max(|w|) / 7`` and ``q = round(w / scale) + 8``, or with ``zeros`` ``scale = (max(w, 0) - min(w, 0)) / 15``, ``zero =
    round(-min(w, 0) / scale)`` and ``q = round(w / scale) + zero``, both held to 0 .. 15.  The scale is rounded to ``scale_dtype`` (the
    weight's type) first; where it is zero, so is the group.  Weights that are not finite, and groups whose scale ``scale_dtype`` cannot hold,
    are refused.  On the host or the device; a step of loading a model, not of running it."""
    _check_group(group)
    if weight.dim() != 3 or weight.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError("weight must be an fp32, fp16 or bf16 tensor [experts, out_features, in_features]")
    scale_dtype = weight.dtype if scale_dtype is None else scale_dtype
    if scale_dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise NotImplementedError("scales must be fp32, fp16 or bf16")
    experts, rows, columns = weight.shape
    groups = _ceil(columns, group)
    packed = _empty_values(experts, rows, columns, weight.device)
    scales = torch.empty(experts, rows, groups, dtype=scale_dtype, device=weight.device)
    points = torch.empty(experts, rows, groups, dtype=torch.uint8, device=weight.device) if zeros else None
    for e in range(experts):
        padded = torch.zeros(rows, groups * group, dtype=torch.float32, device=weight.device)
        padded[:, :columns] = weight[e].detach()
        if not bool(torch.isfinite(padded).all()):
            raise RuntimeError(f"weight of expert {e} holds values that are not finite")
        parts = padded.view(rows, groups, group)
        low = parts.amin(2).clamp(max=0.0) if columns else parts.new_zeros(rows, groups)
        high = parts.amax(2).clamp(min=0.0) if columns else low
        scales[e] = ((high - low) / 15.0 if zeros else torch.maximum(high, -low) / 7.0).to(scale_dtype)
        scale = scales[e].float()
        if not bool(torch.isfinite(scale).all()):
            raise RuntimeError(f"a group of expert {e} needs a scale beyond {scale_dtype}")
        by = torch.where(scale == 0.0, 1.0, scale)
        zero = torch.where(scale == 0.0, 0.0, (-low / by).round().clamp(0, 15)) if zeros else torch.full_like(scale, 8.0)
        if zeros:
            points[e] = zero.to(torch.uint8)
        q = ((parts / by[:, :, None]).round() + zero[:, :, None]).clamp(0, 15).to(torch.uint8)
        _packed_values(q.view(rows, -1)[:, :columns], packed[e])
    tiles = packed.shape[1]
    return Int4Weight(packed, _packed_groups(scales, tiles), None if points is None else _packed_groups(points, tiles), columns, rows, group)
