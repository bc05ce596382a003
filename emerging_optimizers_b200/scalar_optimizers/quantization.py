"""8-bit block-scaled numbers: the format of ``AdamW(state_bits=8)``'s moments.

Every 256 consecutive elements (in memory order) share one exponent byte, the fp32 exponent field of their largest
finite magnitude.  A code is a small float below that power of two: signed numbers have a sign, 4 exponent and 3
mantissa bits, unsigned ones 5 exponent and 3 mantissa bits.  What is not finite (unsigned: or is negative) reads back as NaN; an
unsigned number above zero never becomes zero.
"""

from __future__ import annotations

import torch

from emerging_optimizers_b200 import _native


__all__ = ["dequantize_blockwise", "quantize_blockwise"]

_VALUES = (torch.float32, torch.bfloat16)


def exponent_count(numel: int) -> int:
    """Exponent bytes of ``numel`` elements."""
    return -(-numel // _native.QUANT_BLOCK)


def quantize_blockwise(
    x: torch.Tensor, *, signed: bool, seed: int | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (uint8, the shape of ``x``) and exponent bytes (uint8, one per 256 elements) of a contiguous fp32 or bf16
    CUDA tensor.

    ``seed`` None rounds to nearest (halves away from zero); a number in [0, 2^32) rounds up with the probability of the
    part cut off, with random bits that depend on the seed and the element's place only.
    """
    _native.require_cuda(x, "x")
    if x.dtype not in _VALUES:
        raise TypeError(f"x must be torch.float32 or torch.bfloat16, got {x.dtype}")
    if not x.is_contiguous():
        raise ValueError(f"x is not contiguous (shape {tuple(x.shape)}, strides {x.stride()})")
    if x.is_neg():
        raise ValueError("x is a negated view")
    if seed is not None and not 0 <= seed < 1 << 32:
        raise ValueError(f"seed must be in [0, 2^32), got {seed}")
    codes = torch.empty_like(x, dtype=torch.uint8)
    exponents = x.new_empty(exponent_count(x.numel()), dtype=torch.uint8)
    _native.quantize_blockwise(x, signed, seed, codes, exponents)
    return codes, exponents


def dequantize_blockwise(
    codes: torch.Tensor, exponents: torch.Tensor, *, signed: bool, dtype: torch.dtype = torch.float32
) -> torch.Tensor:
    """The values that ``codes`` stand for, in ``dtype`` (fp32 or bf16: both hold them exactly as long as they are
    normal numbers there)."""
    _native.require_cuda(codes, "codes")
    if dtype not in _VALUES:
        raise TypeError(f"dtype must be torch.float32 or torch.bfloat16, got {dtype}")
    if codes.dtype != torch.uint8 or exponents.dtype != torch.uint8:
        raise TypeError(f"codes and exponents must be torch.uint8, got {codes.dtype} and {exponents.dtype}")
    if exponents.device != codes.device or exponents.numel() != exponent_count(codes.numel()):
        raise ValueError(f"exponents must be {exponent_count(codes.numel())} bytes on {codes.device}")
    if not (codes.is_contiguous() and exponents.is_contiguous()):
        raise ValueError("codes and exponents must be contiguous")
    out = torch.empty_like(codes, dtype=dtype)
    _native.dequantize_blockwise(codes, exponents, signed, out)
    return out
