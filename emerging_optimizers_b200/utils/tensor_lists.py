"""Checks of lists of tensors that a kernel takes by address: one column of addresses per role."""

from __future__ import annotations

from typing import Sequence

import torch

from emerging_optimizers_b200 import _native


__all__ = ["addresses", "common_device", "mark_written", "require_distinct"]

_T = torch.Tensor


def common_device(tensors: Sequence[torch.Tensor], name: str) -> int:
    """Index of the one CUDA device that all ``tensors`` are on."""
    devices = set(map(_T.get_device, tensors))
    if len(devices) == 1 and -1 not in devices:
        return devices.pop()
    for t in tensors:
        _native.require_cuda(t, name)
    raise ValueError(f"{name} must be on one device, got {sorted(devices)}")


def addresses(
    tensors: Sequence[torch.Tensor], name: str, device: int, dtypes: Sequence[torch.dtype], numels: Sequence[int] | None = None
) -> list[int]:
    """Addresses of ``tensors`` after checking that they are dense, on ``device``, of one of ``dtypes`` and of
    ``numels`` elements."""
    if numels is not None:
        found = list(map(_T.numel, tensors))
        if found != numels:
            if len(found) != len(numels):
                raise ValueError(f"{name}: {len(found)} tensors where {len(numels)} are needed")
            i = next(i for i, (a, b) in enumerate(zip(found, numels)) if a != b)
            raise ValueError(f"{name}[{i}] has {found[i]} elements where {numels[i]} are needed")
    if set(map(_T.get_device, tensors)) - {device}:
        for t in tensors:
            _native.require_cuda(t, name)
        raise ValueError(f"{name} must be on cuda:{device}")
    if not {t.dtype for t in tensors}.issubset(dtypes):
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {sorted({str(t.dtype) for t in tensors})}")
    if not all(map(_T.is_contiguous, tensors)):
        i = next(i for i, t in enumerate(tensors) if not t.is_contiguous())
        raise ValueError(f"{name}[{i}] is not contiguous (strides {tensors[i].stride()})")
    return list(map(_T.data_ptr, tensors))


def require_distinct(numels: Sequence[int], **columns: Sequence[int]) -> None:
    """Raise ``ValueError`` when two of the tensors that a call writes start at the same address."""
    empty = numels.count(0)
    total = sum(len(c) for c in columns.values())
    if len(set().union(*columns.values()) - {0}) != total - empty * len(columns):
        raise ValueError(f"a tensor appears twice among {', '.join(columns)}")


def mark_written(tensors: Sequence[torch.Tensor]) -> None:
    """Tell autograd that ``tensors`` changed: a backward pass that saved one of them raises instead of using it."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])
