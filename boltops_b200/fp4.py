"""Microscaled 4-bit floating point: rows to e2m1 codes with a scale per block, and back.

Two formats.  ``"nvfp4"``: blocks of 16 values, an E4M3 scale each, optionally one fp32 scale for the
whole tensor.  ``"mxfp4"``: blocks of 32, an E8M0 scale (a power of two) each.  Codes are packed two to
a byte along the last dimension, the first value in the low bits; a tensor's format is the dtype of
its scales, ``torch.float8_e4m3fn`` or ``torch.uint8``, wherever the framework takes one.  (mxfp4 scales are chosen so
that no value saturates.  The OCP MX specification's conversion takes ``2 ** (floor(log2(amax)) - 2)`` instead,
half of it where amax is more than 6 and less than 8 times a power of two, and saturates there.  Both are valid
encodings, and whatever reads codes and scales takes either.)  The products
that read them: ``gemm.gemm_a4w4``, ``fused_moe.fused_experts_fp4`` and ``fused_moe.fused_experts_decode``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _cabi
from ._cabi import ptr, stream_of

FORMATS = {"nvfp4": (_cabi.FP4_NV, 16, torch.float8_e4m3fn), "mxfp4": (_cabi.FP4_MX, 32, torch.uint8)}
_FORMAT_OF = {dtype: name for name, (_, _, dtype) in FORMATS.items()}
_FLOATS = {torch.bfloat16: _cabi.BF16, torch.float16: _cabi.F16, torch.float32: _cabi.F32}


def format_of(scales: torch.Tensor) -> str:
    """The format that scales of this dtype belong to."""
    name = _FORMAT_OF.get(scales.dtype)
    if name is not None:
        return name
    raise TypeError(f"4-bit scales are float8_e4m3fn (nvfp4) or uint8 (mxfp4), not {scales.dtype}")


def check_global_scale(name: str, scale: Optional[torch.Tensor], fmt: str, numel: int,
                       device: torch.device) -> Optional[torch.Tensor]:
    """A whole-tensor scale as the kernels read it: ``numel`` fp32 values on ``device``, or None."""
    if scale is None:
        return None
    if fmt != "nvfp4":
        raise ValueError(f"{name}: mxfp4 has no scale of the whole tensor")
    if scale.numel() != numel or scale.dtype != torch.float32:
        raise ValueError(f"{name} must hold {numel} float32 value(s)")
    if scale.device != device:
        raise ValueError(f"{name} is on {scale.device}, the rows on {device}")
    return scale.contiguous()


def fp4_quant(x: torch.Tensor, format: str = "nvfp4", global_scale: Optional[torch.Tensor] = None
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes [..., K/2] uint8, scales [..., K/block])`` of ``x`` [..., K] (bf16, fp16 or fp32).

    nvfp4: ``y = x * (1 / global_scale)``, ``scale = e4m3(min(amax(y) * (1/6), 448))``; mxfp4: the smallest
    power of two that is at least ``amax / 6`` (byte 0 for a block of zeros).  A code is the nearest of
    ``value / scale``, ties to even.  A block that holds a NaN or an infinity gets the NaN scale and
    reads back as NaNs."""
    spec = FORMATS.get(format)
    if spec is None:
        raise ValueError(f"unknown 4-bit format {format!r}: nvfp4 or mxfp4")
    code, block, scale_dtype = spec
    if not x.is_cuda:
        raise ValueError("boltops_b200 kernels need CUDA tensors (there is no CPU path)")
    if x.dtype not in _FLOATS:
        raise TypeError(f"fp4_quant takes bf16, fp16 or fp32, not {x.dtype}")
    shape, dev = x.shape, x.device
    if len(shape) < 1 or shape[-1] % block:
        raise ValueError(f"the last dimension must be whole blocks of {block} values ({format})")
    g = check_global_scale("global_scale", global_scale, format, 1, dev)
    cols = shape[-1]
    lead = shape[:-1]
    codes = torch.empty((*lead, cols // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((*lead, cols // block), dtype=scale_dtype, device=dev)
    n = x.numel()
    if n:
        x = ops.aligned(x)
        _cabi.call(dev, _cabi.load().bolt_fp4_quant, x.data_ptr(), _FLOATS[x.dtype], n // cols, cols, code,
                   ptr(g), codes.data_ptr(), scales.data_ptr(), stream_of(x))
        ops._count()
    return codes, scales


def fp4_dequant(codes: torch.Tensor, scales: torch.Tensor, global_scale: Optional[torch.Tensor] = None,
                dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values ``code * scale * global_scale`` [..., K] of packed codes [..., K/2]."""
    format = format_of(scales)
    code, block, _ = FORMATS[format]
    if not codes.is_cuda:
        raise ValueError("boltops_b200 kernels need CUDA tensors (there is no CPU path)")
    if codes.dtype != torch.uint8 or dtype not in _FLOATS:
        raise TypeError("fp4_dequant takes uint8 codes and gives bf16, fp16 or fp32")
    if codes.dim() < 1 or (2 * codes.shape[-1]) % block or \
            tuple(scales.shape) != (*codes.shape[:-1], 2 * codes.shape[-1] // block):
        raise ValueError(f"scales {tuple(scales.shape)} do not belong to codes {tuple(codes.shape)} "
                         f"in blocks of {block}")
    if scales.device != codes.device:
        raise ValueError(f"scales are on {scales.device}, codes on {codes.device}")
    g = check_global_scale("global_scale", global_scale, format, 1, codes.device)
    cols = 2 * codes.shape[-1]
    out = torch.empty((*codes.shape[:-1], cols), dtype=dtype, device=codes.device)
    n = out.numel()
    if n:
        codes, scales = ops.aligned(codes, 4), ops.aligned(scales, 1)
        _cabi.call(out.device, _cabi.load().bolt_fp4_dequant, codes.data_ptr(), scales.data_ptr(), n // cols, cols,
                   code, ptr(g), out.data_ptr(), _FLOATS[dtype], stream_of(out))
        ops._count()
    return out


__all__ = ["fp4_quant", "fp4_dequant"]

# (last: the package imports this module's definitions)
from .fused_moe import ops  # noqa: E402
