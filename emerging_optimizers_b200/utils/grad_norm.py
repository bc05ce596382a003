"""Global gradient norm and clipping over many tensors in a few launches, without a synchronisation.

The clipping coefficient stays on the device: :func:`clip_coefficient` hands it to
``AdamW.step(grad_scale=...)``, which then scales the gradients as it reads them, so that they are read once for the
norm and never written back.  :func:`clip_grads_` / :func:`clip_grad_norm_` scale them in place for every other
consumer.
"""

from __future__ import annotations

import math
from typing import Iterable, Sequence

import torch

from emerging_optimizers_b200 import _native


__all__ = ["clip_coefficient", "clip_grad_norm_", "clip_grads_", "global_grad_norm"]


def _norm(grads: Sequence[torch.Tensor], max_norm: float, in_place: bool) -> torch.Tensor:
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if not torch.is_tensor(grads):  # a tensor would be taken apart into its rows: the table refuses it
        grads = list(grads)
    device, table, types, elements = _native.host().grads_table(grads, in_place)
    return _native.grad_norm(grads, device, table, types, elements, max_norm, in_place)


def global_grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """2-norm of all elements of ``grads`` (fp32 or bf16 CUDA tensors of one device, dense in any memory order) as an fp32
    scalar tensor.  Summed in float64 in a fixed order: the same call gives the same bits.  Squares and their sums in pairs are
    rounded to fp32 where they stay well inside its range, so that the norm is within two fp32 roundings of the exact
    one."""
    return _norm(grads, math.inf, False)[0]


def clip_coefficient(grads: Sequence[torch.Tensor], max_norm: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, min(1, max_norm / (norm + 1e-6)))`` as fp32 scalar tensors on the device; the gradients stay as they
    are.

    Pass the coefficient to ``AdamW.step(grad_scale=...)``.  A norm that is NaN gives a coefficient that is NaN.
    """
    out = _norm(grads, max_norm, False)
    return out[0], out[1]


def clip_grads_(grads: Sequence[torch.Tensor], max_norm: float) -> torch.Tensor:
    """Multiply all of ``grads`` in place by ``min(1, max_norm / (norm + 1e-6))``; returns the norm from before."""
    return _norm(grads, max_norm, True)[0]


def clip_grad_norm_(
    parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, *, error_if_nonfinite: bool = False
) -> torch.Tensor:
    """Clip the global 2-norm of the gradients of ``parameters`` in place, as ``torch.nn.utils.clip_grad_norm_`` does.

    Gradients are dense (channels-last and transposed ones too; no gaps, nothing expanded) and each appears once.
    Parameters without a gradient are passed over; with none left the result is 0.  ``error_if_nonfinite`` raises
    ``RuntimeError`` before anything is scaled if the norm is infinite or NaN (and waits for the device to know).
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite and not math.isfinite(float(global_grad_norm(grads))):
        raise RuntimeError("the total norm of the gradients is not finite, so they cannot be clipped")
    return clip_grads_(grads, max_norm)
