"""AdamW over many tensors at once, with moments in fp32 or in 8 bits.

The scalar optimizer that a model's embeddings, output layer and 1-D parameters need beside the orthogonalized ones
(the reference keeps its scalar optimizers in ``emerging_optimizers/scalar_optimizers``).  A step of a parameter group
is one launch for each mix of types (up to 384 tensors), whatever their sizes.
"""

from __future__ import annotations

from itertools import compress
from typing import Any, Callable, Sequence

import torch
import torch.optim as optim
from torch.optim.optimizer import ParamsT

from emerging_optimizers_b200 import _native, registry
from emerging_optimizers_b200.mixin import WeightDecayT
from emerging_optimizers_b200.scalar_optimizers.quantization import (
    dequantize_blockwise,
    exponent_count,
    quantize_blockwise,
)


__all__ = ["AdamW", "adamw_step", "adamw_step_8bit"]

_FLOATS = (torch.float32, torch.bfloat16)
_MASK32 = (1 << 32) - 1


def _check_hyperparameters(lr: Any, betas: Any, eps: float, weight_decay: float, method: str) -> None:
    if not torch.is_tensor(lr) and not lr >= 0.0:
        raise ValueError(f"Invalid learning rate: {lr}")
    if not (len(betas) == 2 and all(0.0 <= b < 1.0 for b in betas)):
        raise ValueError(f"Invalid betas: {betas}")
    if eps != 0.0 and not 2.0**-126 <= eps < 2.0**126:  # zero, or a number whose reciprocal is normal in fp32
        raise ValueError(f"Invalid epsilon: {eps}")
    if not weight_decay >= 0.0:
        raise ValueError(f"Invalid weight decay: {weight_decay}")
    if method not in _native._DECAY_METHODS:
        raise ValueError(f"Invalid weight decay method: {method}")


def _device_scalar(value: Any, name: str, device: int, dtype: torch.dtype) -> torch.Tensor:
    if not torch.is_tensor(value) or value.dtype != dtype or value.numel() != 1 or value.get_device() != device:
        raise TypeError(f"{name} must be a {dtype} tensor of one element on cuda:{device}")
    if value.is_neg():
        raise ValueError(f"{name} is a negated view")
    return value


def _listed(tensors: Any) -> Any:
    """``tensors`` as a list or tuple, which keeps what an iterator or a view makes on the way alive until the launch: the
    table holds addresses only.  A tensor would be taken apart into its rows: it stays one, and the table refuses it."""
    return tensors if tensors is None or isinstance(tensors, (list, tuple, torch.Tensor)) else list(tensors)


def _step(
    params, grads, m, v, m_exponents, v_exponents, remainders, *, lr, betas, eps, weight_decay, step,
    weight_decay_method, grad_scale, seed=0, first_index=0,
) -> None:  # fmt: skip
    _check_hyperparameters(lr, betas, eps, weight_decay, weight_decay_method)
    if not (0 <= seed <= _MASK32):
        raise ValueError(f"seed must be in [0, 2^32), got {seed}")
    params, grads, m, v, m_exponents, v_exponents, remainders = map(
        _listed, (params, grads, m, v, m_exponents, v_exponents, remainders)
    )
    if not torch.is_tensor(params) and not params:
        return
    on_host = isinstance(step, int)
    if not on_host:
        step = _listed(step)
    if on_host and step < 1:
        raise ValueError(f"step counts from 1, got {step}")
    host = _native.host()
    device, table, kinds = host.adamw_table(
        params, grads, m, v, m_exponents, v_exponents, remainders, None if on_host else step
    )
    if on_host and host.stream(device)[2]:
        raise RuntimeError(
            "a step number given as an int would be frozen into the captured graph: pass an int64 device tensor"
        )
    lr_tensor = None
    if torch.is_tensor(lr):
        if lr.is_cuda:
            lr_tensor, lr = _device_scalar(lr, "lr", device, torch.float32), 0.0
        else:
            lr = float(lr)
    if grad_scale is not None:
        _device_scalar(grad_scale, "grad_scale", device, torch.float32)
    _native.adamw_step(
        device, len(params), table, kinds, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
        method=weight_decay_method, step=step if on_host else 0, on_device=not on_host or lr_tensor is not None,
        state_bits=32 if m_exponents is None else 8, seed=seed, first_index=first_index, lr_tensor=lr_tensor,
        grad_scale=grad_scale,
    )  # fmt: skip


def adamw_step(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    *,
    lr: float | torch.Tensor,
    betas: tuple[float, float] = (0.9, 0.95),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    step: int | torch.Tensor | Sequence[torch.Tensor],
    weight_decay_method: WeightDecayT = "decoupled",
    grad_scale: torch.Tensor | None = None,
    remainders: Sequence[torch.Tensor] | None = None,
) -> None:
    """One AdamW step of a list of tensors, in place.

    All arithmetic is fp32 with one rounding per operation, the moments are fp32.  Tensors are contiguous CUDA tensors
    of one device; parameters and gradients fp32 or bf16 in any mix.  No two tensors that are written may overlap.

    Args:
        params, grads, exp_avgs, exp_avg_sqs: parameters, gradients, first and second moments, one of each per tensor.
        lr, betas, eps, weight_decay: as usual; ``lr`` may be an fp32 device scalar; ``eps`` is zero or from 2^-126 to 2^126.
        step: number of this step, from 1; or int64 device scalars (one for all or one per tensor) holding it, which a
            captured graph reads anew at every replay.
        weight_decay_method: one of :data:`emerging_optimizers_b200.mixin.WeightDecayT`.
        grad_scale: fp32 device scalar that multiplies every gradient as it is read (a clipping coefficient).
        remainders: int16, one per tensor, for bf16 parameters: the low halves of their fp32 masters, master bits =
            (bf16 bits << 16) + remainder.  Start with zeros.  Without them a bf16 parameter is rounded to nearest every
            step and loses updates below half its last place.
    """
    _step(
        params, grads, exp_avgs, exp_avg_sqs, None, None, remainders, lr=lr, betas=betas, eps=eps,
        weight_decay=weight_decay, step=step, weight_decay_method=weight_decay_method, grad_scale=grad_scale,
    )  # fmt: skip


def adamw_step_8bit(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    exp_avgs: Sequence[torch.Tensor],
    exp_avg_exponents: Sequence[torch.Tensor],
    exp_avg_sqs: Sequence[torch.Tensor],
    exp_avg_sq_exponents: Sequence[torch.Tensor],
    *,
    lr: float | torch.Tensor,
    betas: tuple[float, float] = (0.9, 0.95),
    eps: float = 1e-8,
    weight_decay: float = 0.01,
    step: int | torch.Tensor | Sequence[torch.Tensor],
    seed: int,
    weight_decay_method: WeightDecayT = "decoupled",
    grad_scale: torch.Tensor | None = None,
    remainders: Sequence[torch.Tensor] | None = None,
) -> None:
    """:func:`adamw_step` with moments in 8 bits (see :func:`quantize_blockwise`: first moments signed, second ones
    unsigned; codes of the tensor's size and one exponent byte per 256 elements, zeros at the start).

    The update uses the new moments before they are rounded.  They are then rounded at random, up with the probability
    of the part cut off, by bits from ``seed``, the tensor's place in the list, the step number and the element: to
    nearest, a moving average in 8 bits stands still as soon as a step moves it by less than half a unit.
    """
    _step(
        params, grads, exp_avgs, exp_avg_sqs, exp_avg_exponents, exp_avg_sq_exponents, remainders, lr=lr,
        betas=betas, eps=eps, weight_decay=weight_decay, step=step, weight_decay_method=weight_decay_method,
        grad_scale=grad_scale, seed=seed,
    )  # fmt: skip


def _memory_order(t: torch.Tensor) -> tuple[int, ...] | None:
    """Order of the dimensions of a dense tensor from the slowest to the fastest; None for a contiguous one."""
    if t.is_contiguous():
        return None
    order = tuple(sorted(range(t.dim()), key=lambda d: (-t.stride(d), -t.size(d))))
    if not t.permute(order).is_contiguous():
        raise ValueError(f"AdamW needs dense parameters, got shape {tuple(t.shape)} with strides {t.stride()}")
    return order


def _flat(t: torch.Tensor, order: tuple[int, ...] | None) -> torch.Tensor:
    """``t`` seen in memory order, a copy only if it is laid out otherwise."""
    t = t.detach()
    return (t if order is None else t.permute(order)).contiguous()


def _require_layout(states: Sequence[dict], orders: Sequence[tuple[int, ...] | None]) -> None:
    """What a step writes must lie as its parameter does: a copy in the parameter's order would take the update with it."""
    for state, order in zip(states, orders):
        for name in ("exp_avg", "exp_avg_sq", "remainder"):
            t = state.get(name)
            if t is not None and not (t if order is None else t.permute(order)).is_contiguous():
                raise ValueError(
                    f"a parameter changed its memory order since its state was made ({name} of shape {tuple(t.shape)} has strides "
                    f"{t.stride()}): optimizer.load_state_dict(optimizer.state_dict()) lays the state out anew"
                )


@registry.register_optimizer("fused_adamw")
class AdamW(optim.Optimizer):
    """AdamW whose step takes all tensors of a group in one launch.

    Parameters are fp32 or bf16 and dense, on CUDA; gradients fp32 or bf16.  See :func:`adamw_step` for the arithmetic.

    Args:
        params: parameters or parameter groups (groups may set ``lr``, ``betas``, ``eps`` and ``weight_decay``).
        lr: learning rate; an fp32 device scalar is read anew at every replay of a captured step.
        betas, eps, weight_decay: as usual.
        weight_decay_method: one of :data:`emerging_optimizers_b200.mixin.WeightDecayT`.
        state_bits: 32, or 8 for moments of one byte each (2 bytes a parameter in place of 8; see
            :func:`adamw_step_8bit`).
        master_remainder: keep for bf16 parameters the low 16 bits of an fp32 master in ``state["remainder"]``.
        capturable: count steps in device memory, so that :meth:`step` can be captured into a CUDA graph.  Run a step
            before the capture: it creates the state.
        seed: seed of the random rounding of 8-bit moments.
    """

    def __init__(
        self,
        params: ParamsT,
        lr: float | torch.Tensor = 3e-4,
        betas: tuple[float, float] = (0.9, 0.95),
        eps: float = 1e-8,
        weight_decay: float = 0.01,
        *,
        weight_decay_method: WeightDecayT = "decoupled",
        state_bits: int = 32,
        master_remainder: bool = False,
        capturable: bool = False,
        seed: int = 0,
    ) -> None:
        _check_hyperparameters(lr, betas, eps, weight_decay, weight_decay_method)
        if not 0 <= seed <= _MASK32:
            raise ValueError(f"seed must be in [0, 2^32), got {seed}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.weight_decay_method = weight_decay_method
        self.state_bits = state_bits
        self.master_remainder = master_remainder
        self.capturable = capturable
        self.seed = seed
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self) -> dict[str, Any]:
        """The base class keeps the groups and the state only; without these nobody could read the state."""
        own = ("weight_decay_method", "state_bits", "master_remainder", "capturable", "seed")
        return {**super().__getstate__(), **{name: getattr(self, name) for name in own}}

    # -- state -------------------------------------------------------------------------------------------------------

    def _has_remainder(self, p: torch.Tensor) -> bool:
        return self.master_remainder and p.dtype == torch.bfloat16

    def _new_state(self, p: torch.Tensor) -> dict:
        if p.dtype not in _FLOATS:
            raise TypeError(f"AdamW takes torch.float32 or torch.bfloat16 parameters, got {p.dtype}")
        _native.require_cuda(p, "a parameter of AdamW")
        _memory_order(p)
        state: dict = {"step": torch.zeros((), dtype=torch.int64, device=p.device) if self.capturable else 0}
        dtype = torch.uint8 if self.state_bits == 8 else torch.float32
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros_like(p, dtype=dtype, memory_format=torch.preserve_format)
            if self.state_bits == 8:
                state[f"{name}_exponents"] = torch.zeros(exponent_count(p.numel()), dtype=torch.uint8, device=p.device)
        if self._has_remainder(p):
            state["remainder"] = torch.zeros_like(p, dtype=torch.int16, memory_format=torch.preserve_format)
        return state

    def moments(self, p: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """First and second moment of ``p`` as new fp32 tensors, whatever they are stored in."""
        state = self.state.get(p)
        if not state:
            raise ValueError("the parameter has no state yet")
        return self._values(state, "exp_avg", True), self._values(state, "exp_avg_sq", False)

    @staticmethod
    def _values(state: dict, name: str, signed: bool) -> torch.Tensor:
        x = state[name]
        if x.dtype != torch.uint8:
            return x.clone()
        order = _memory_order(x)
        values = dequantize_blockwise(_flat(x, order), state[f"{name}_exponents"], signed=signed)
        return values if order is None else values.permute([order.index(d) for d in range(x.dim())])

    # -- step --------------------------------------------------------------------------------------------------------

    @torch.no_grad()
    def step(  # type: ignore[override]
        self, closure: Callable[[], float] | None = None, *, grad_scale: torch.Tensor | None = None
    ) -> None:
        """One step.  ``grad_scale`` (an fp32 device scalar, for instance the coefficient of
        :func:`emerging_optimizers_b200.utils.clip_coefficient`) multiplies the gradients as they are read."""
        if closure is not None:
            raise ValueError("closure is not supported")
        first_index = 0
        for group in self.param_groups:
            params, grads, uniform = _native.host().with_grads(group["params"])
            states = [self.state[p] for p in params]
            if not all(states):
                for p, state in zip(params, states):
                    if not state:
                        if p.is_cuda and torch.cuda.is_current_stream_capturing():
                            raise RuntimeError(
                                "run a step before capturing one: the state must exist when the capture begins"
                            )
                        state.update(self._new_state(p))
            # one call per device, type of parameter and step number (with device counters: whatever the number)
            steps = [0] * len(params) if self.capturable else [state["step"] + 1 for state in states]
            if uniform and len(set(steps)) == 1:
                first_index += self._call(group, params, grads, states, True, steps[0], grad_scale, first_index)
                continue
            calls = list(zip(map(torch.Tensor.get_device, params), [p.dtype for p in params], steps))
            for call in dict.fromkeys(calls):
                chosen = [c == call for c in calls]
                lists = ([*compress(t, chosen)] for t in (params, grads, states))
                first_index += self._call(group, *lists, uniform, call[2], grad_scale, first_index)
        return None

    def _call(  # type: ignore[no-untyped-def]
        self, group, params, grads, states, plain, step, grad_scale, first_index
    ) -> int:
        """The step of parameters of one device, type and step number; ``plain``: all of them and their gradients are
        contiguous.  Returns their number."""
        if not plain:
            orders = [_memory_order(p) for p in params]
            _require_layout(states, orders)
            grads = [_flat(g, o) for g, o in zip(grads, orders)]

        def column(name):  # type: ignore[no-untyped-def]
            ts = [s[name] for s in states]
            return ts if plain else [_flat(t, o) for t, o in zip(ts, orders)]

        if self.capturable:
            step = [s["step"] for s in states]
            torch._foreach_add_(step, 1)
        exponents = [None, None]
        if self.state_bits == 8:
            exponents = [[s[name] for s in states] for name in ("exp_avg_exponents", "exp_avg_sq_exponents")]
        try:
            _step(
                params if plain else [_flat(p, o) for p, o in zip(params, orders)], grads, column("exp_avg"),
                column("exp_avg_sq"), *exponents, column("remainder") if self._has_remainder(params[0]) else None,
                lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], step=step,
                weight_decay_method=self.weight_decay_method, grad_scale=grad_scale, seed=self.seed,
                first_index=first_index,
            )  # fmt: skip
        except Exception:
            if self.capturable:  # a step that was refused does not count
                torch._foreach_sub_(step, 1)
            if plain:
                _require_layout(states, [None] * len(states))  # says more than that a tensor is not contiguous
            raise
        if not self.capturable:
            for s in states:
                s["step"] = step
        return len(params)

    # -- checkpoints -------------------------------------------------------------------------------------------------

    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """Load a state that this class or ``torch.optim.AdamW`` wrote.

        Moments of the other width are converted (32 to 8 bits: rounded to nearest); types are kept as this optimizer
        has them, whatever the parameter's.
        """
        saved: dict[str, Any] = {}

        def take(_: optim.Optimizer, state_dict: dict[str, Any]) -> dict[str, Any]:
            for group in state_dict["param_groups"]:
                for key in ("amsgrad", "maximize"):
                    if group.get(key):
                        raise ValueError(f"the saved optimizer ran with {key}, which AdamW does not have")
            saved.update(state_dict)
            return {**state_dict, "state": {}}  # the base class would cast the state to the parameters' types

        def fill(_: optim.Optimizer) -> None:
            ids = [i for group in saved["param_groups"] for i in group["params"]]
            params = [p for group in self.param_groups for p in group["params"]]
            for i, p in zip(ids, params):
                if saved["state"].get(i):
                    self.state[p] = self._loaded_state(p, saved["state"][i])

        # after the last of the optimizer's own hooks on what is loaded, and before the first of those on what has been
        handles = [
            self.register_load_state_dict_pre_hook(take),
            self.register_load_state_dict_post_hook(fill, prepend=True),
        ]
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()

    @torch.no_grad()
    def _loaded_state(self, p: torch.Tensor, saved: dict) -> dict:
        state = self._new_state(p)
        if self.capturable:
            state["step"].fill_(int(saved["step"]))
        else:
            state["step"] = int(saved["step"])
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            x = saved[name].to(p.device)
            if x.shape != p.shape:
                raise ValueError(f"{name} of shape {tuple(x.shape)} does not fit a parameter of shape {tuple(p.shape)}")
            exponents = f"{name}_exponents"
            if x.dtype == torch.uint8 and self.state_bits == 8 and x.stride() == p.stride():
                state[name].copy_(x)
                state[exponents].copy_(saved[exponents])
                continue
            if x.dtype == torch.uint8:
                x = self._values({name: x, exponents: saved[exponents].to(p.device)}, name, signed)
            if self.state_bits == 8:
                order = _memory_order(p)
                values = torch.empty_like(p, dtype=torch.float32).copy_(x)
                codes, state[exponents] = quantize_blockwise(_flat(values, order), signed=signed)
                _flat(state[name], order).copy_(codes)
            else:
                state[name].copy_(x)
        if "remainder" in state and "remainder" in saved:
            state["remainder"].copy_(saved["remainder"])
        return state
