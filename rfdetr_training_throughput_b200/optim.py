"""AdamW on the device: one launch over all tensors, moments in 32 bits or in 8 (``rfm_adamw``).

``adamw_step`` is the step on lists of tensors; ``AdamW`` is a ``torch.optim.Optimizer`` on top of it
with torch's arguments.  With ``moment_bits=8`` a parameter's two moments take one byte each, plus one
float32 scale per moment and 256 elements: a quarter of the memory, and 16 instead of 28 bytes moved
per float32 parameter and step.  The codes are rounded at random (a hash of the step, the tensor's
number and the element's index, so a run is reproducible): with nearest rounding a moment that moves by
less than half a code a step would stand still.
"""

from __future__ import annotations

from typing import Any, Iterable

import torch

from . import _lib
from ._native import host

TensorList = list[torch.Tensor] | tuple[torch.Tensor, ...]

#: Elements that share one scale of the 8-bit moments.
MOMENT_BLOCK = _lib.MOMENT_BLOCK


def moment_scales(numel: int) -> int:
    """Scales of one 8-bit moment of ``numel`` elements."""
    return -(-numel // MOMENT_BLOCK)


def adamw_step(params: TensorList, grads: TensorList, exp_avg: TensorList, exp_avg_sq: TensorList,
               step: int | torch.Tensor, *, scales: tuple[TensorList, TensorList] | None = None, lr: float | torch.Tensor = 1e-3,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               grad_scale: torch.Tensor | None = None) -> None:
    """One AdamW step in place on ``params`` and their moments.

    ``params`` and ``grads``: contiguous CUDA tensors of one type (float32, bfloat16 or float16) on one
    device, pairwise of one size; nothing that is written may share memory with anything else.  Without
    ``scales``, ``exp_avg`` and ``exp_avg_sq`` are float32 tensors of the params' sizes.  With ``scales``
    (two lists of float32 tensors, of ``moment_scales(numel)`` elements each) they hold int8 and uint8
    codes (see ``rfm_adamw``).

    ``step`` is the number of this update, from 1; an int64 tensor of one element on the device, and for
    ``lr`` a float32 one, are read by the kernels, so that a captured step follows them (unchecked: a counter
    of 0 gives NaN).  ``grad_scale``
    (float32, one element, on the device) multiplies the gradients: a clipping factor or the inverse of a
    loss scale, without a host synchronisation.
    """
    device_step = device_lr = None
    if isinstance(step, torch.Tensor):
        device_step, step = step, 0
    if isinstance(lr, torch.Tensor):
        device_lr, lr = lr, 0.0
    avg_scales, avg_sq_scales = (None, None) if scales is None else scales
    host().adamw_step(params, grads, exp_avg, exp_avg_sq, avg_scales, avg_sq_scales, step, device_step, lr, device_lr,
                      betas[0], betas[1], eps, weight_decay, grad_scale)


def dequantize_moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, exp_avg_scale: torch.Tensor,
                       exp_avg_sq_scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The float32 values that one tensor's 8-bit moments stand for."""
    return host().dequantize_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)


def quantize_moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """8-bit codes and scales ``(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)`` nearest to one
    tensor's float32 moments, for states that come from 32 bits.  Not part of a step."""
    def blocks(t):
        flat = t.detach().float().reshape(-1)
        return torch.nn.functional.pad(flat, (0, -flat.numel() % MOMENT_BLOCK)).view(-1, MOMENT_BLOCK)

    m, v = blocks(exp_avg), blocks(exp_avg_sq)
    sm, sv = m.abs().amax(1), v.amax(1)
    a = torch.nan_to_num((m.abs() / sm[:, None]).sqrt() * 127, nan=0.0).round().clamp(0, 127)
    b = torch.nan_to_num((v / sv[:, None]).sqrt().sqrt() * 255, nan=0.0).round().clamp(0, 255)
    b = torch.where(v > 0, b.clamp_min(1), b)

    def codes(t, dtype):
        return t.view(-1)[:exp_avg.numel()].to(dtype).view(exp_avg.shape)

    return codes(torch.where(m < 0, -a, a), torch.int8), codes(b, torch.uint8), sm, sv


class AdamW(torch.optim.Optimizer):
    """AdamW with torch's arguments, one launch per parameter group and type.

    ``moment_bits`` 32 keeps float32 moments, 8 the codes and scales of ``adamw_step``.  With
    ``capturable`` step counters lie on the device, one for the parameters of a launch, and advance inside
    ``step()``, so that a captured step can be replayed (without it a capture raises); ``lr`` may then be a
    float32 device tensor.  ``amsgrad`` and
    ``maximize`` are not offered and raise.  A parameter's state is ``exp_avg``, ``exp_avg_sq`` (and
    ``exp_avg_scale``, ``exp_avg_sq_scale``) with ``step``; a float32 state dict loads into either form.
    """

    def __init__(self, params: Iterable, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, amsgrad: bool = False, *, maximize: bool = False,
                 foreach: bool | None = None, capturable: bool = False, differentiable: bool = False,
                 fused: bool | None = None, moment_bits: int = 32):
        if amsgrad or maximize or differentiable:
            raise NotImplementedError("amsgrad, maximize and differentiable steps are not offered")
        if moment_bits not in (8, 32):
            raise ValueError(f"moment_bits must be 8 or 32, got {moment_bits}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("a tensor lr needs capturable=True")
        b1, b2 = betas
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError("betas must be in [0, 1), eps and weight_decay not negative")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable,
                                      moment_bits=moment_bits))

    def _new_state(self, p: torch.Tensor, group: dict) -> dict:
        state: dict[str, Any] = {}
        if group["capturable"]:
            state["step"] = torch.zeros((), dtype=torch.int64, device=p.device)
        else:
            state["step"] = 0
        if group["moment_bits"] == 32:  # with the parameter's strides
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            state["exp_avg_sq"] = torch.zeros_like(state["exp_avg"])
        else:
            if not p.is_contiguous():
                raise ValueError("8-bit moments need contiguous parameters")
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
            for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                state[k] = torch.zeros(moment_scales(p.numel()), dtype=torch.float32, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient."""
        if _capturing() and not all(group["capturable"] for group in self.param_groups):
            raise RuntimeError("a captured step needs capturable=True: a host counter would stay at this step's number "
                               "in every replay")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for members in self._buckets(group):
                self._step_bucket(group, members)
        return loss

    def _buckets(self, group: dict) -> list[list]:
        """The parameters that have a gradient, with their states (new ones are not the optimiser's yet), a
        list for each launch: of one type and device, with one step count."""
        buckets: dict[tuple, list] = {}
        fresh: dict[tuple, torch.Tensor] = {}
        capturable = group["capturable"]
        for p in group["params"]:
            if p.grad is None:
                continue
            if p.grad.is_sparse:
                raise ValueError("AdamW does not take sparse gradients")
            state = self.state.get(p)
            if not state:
                state = self._new_state(p, group)
                if capturable:  # parameters of a launch that start together share one counter
                    state["step"] = fresh.setdefault((p.device, p.dtype), state["step"])
            count = id(state["step"]) if capturable else state["step"]
            buckets.setdefault((p.dtype, p.device, count), []).append((p, state))
        return list(buckets.values())

    def _step_bucket(self, group: dict, members: list) -> None:
        """One launch.  Counters and new states are the optimiser's once it has been accepted."""
        params, grads, avg, avg_sq = [], [], [], []
        for p, s in members:
            g, m, v = p.grad, s["exp_avg"], s["exp_avg_sq"]
            if not p.is_contiguous():
                p, g, m, v = _flat_alike(p, g, m, v)
            elif not g.is_contiguous():
                g = g.contiguous()
            params.append(p)
            grads.append(g)
            avg.append(m)
            avg_sq.append(v)
        scales = None
        if group["moment_bits"] == 8:
            scales = tuple([s[k] for _, s in members] for k in ("exp_avg_scale", "exp_avg_sq_scale"))
        if group["capturable"]:
            step = self._own_counter(group, members).add_(1)
        else:
            step = members[0][1]["step"] + 1
        try:
            adamw_step(params, grads, avg, avg_sq, step, scales=scales, lr=group["lr"], betas=group["betas"],
                       eps=group["eps"], weight_decay=group["weight_decay"])
        except Exception:
            if group["capturable"]:
                step.sub_(1)
            raise
        for p, s in members:
            s["step"] = step
            self.state[p] = s

    def _own_counter(self, group: dict, members: list) -> torch.Tensor:
        """The step counter of a launch's parameters: one of their own where others, of another type or
        without a gradient this time, stay at its present count."""
        counter, capturing = members[0][1]["step"], _capturing()
        mine = {id(s) for _, s in members}
        if all(s.get("step") is not counter or id(s) in mine for s in map(self.state.get, group["params"]) if s):
            if capturing:
                counter.in_a_graph = True
            return counter
        if capturing or getattr(counter, "in_a_graph", False):
            raise RuntimeError("a captured step counts for all parameters that share its step counter, and some of them "
                               "have no gradient now: before the capture, take a step with the same gradients")
        counter = counter.clone()
        for _, s in members:
            s["step"] = counter
        return counter

    def load_state_dict(self, state_dict: dict) -> None:
        """Load a state dict of this class or of ``torch.optim.AdamW``.  ``moment_bits`` and ``capturable``
        stay as constructed; moments are converted to the form they ask for."""
        kept = [(g["moment_bits"], g["capturable"]) for g in self.param_groups]
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise NotImplementedError("amsgrad and maximize steps are not offered")
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        raw = dict(zip((p for g in self.param_groups for p in g["params"]), ids))
        for group, (bits, capturable) in zip(self.param_groups, kept):
            group["moment_bits"], group["capturable"] = bits, capturable
            shared: dict[tuple, torch.Tensor] = {}
            for p in group["params"]:
                saved = state_dict["state"].get(raw[p])
                if not saved:
                    continue
                state = self._new_state(p, group)
                _adopt(state, saved, bits)
                count = int(saved["step"])
                if capturable:
                    state["step"] = shared.setdefault((p.device, p.dtype, count), state["step"].fill_(count))
                else:
                    state["step"] = count
                self.state[p] = state


def _capturing() -> bool:
    """Whether the current stream's work goes into a graph."""
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _flat_alike(data, g, m, v):
    """The dense elements of a parameter with permuted strides as one contiguous view, and the
    gradient and the moments in the same order."""
    order = sorted(range(data.dim()), key=data.stride, reverse=True)
    flat = data.permute(order)
    if not flat.is_contiguous():
        raise ValueError("parameters must be dense (no gaps or overlaps between their elements)")
    g = g.permute(order).contiguous()
    m, v = m.permute(order), v.permute(order)
    if not (m.is_contiguous() and v.is_contiguous()):
        raise ValueError("the moments must have their parameter's strides")
    return flat, g, m, v


@torch.no_grad()
def _adopt(state: dict, saved: dict, bits: int) -> None:
    """Copy saved moments, in either form, into ``state``'s."""
    device = state["exp_avg"].device
    m, v = saved["exp_avg"].to(device), saved["exp_avg_sq"].to(device)
    names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    if m.dtype == torch.int8:
        values = [m, v, saved["exp_avg_scale"].to(device), saved["exp_avg_sq_scale"].to(device)]
        if bits == 32:
            values = dequantize_moments(*(t.contiguous() for t in values))
    else:
        values = (m, v) if bits == 32 else quantize_moments(m, v)
    for name, value in zip(names, values):
        state[name].copy_(value)
