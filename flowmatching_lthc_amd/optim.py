"""AdamW over many tensors at once (gfx950 HIP kernels), its states in 32 or in 8 bits.

``AdamW`` is a ``torch.optim.Optimizer``: a step is one launch for every 56 tensors (and two for the norm of all
gradients where it clips), in place of a dozen passes over the parameters.  In the same pass it keeps fp32 master weights
of 16-bit parameters and the moving average of the weights that the reference's training script keeps beside them (the
``ema`` entry of ``checkpoint.checkpoint_state``).  ``adamw_step``, ``grad_norm`` and ``state_values`` are the operators
below it, for programs that hold their states themselves.

Per element, fp32: ``m = m b1 + g (1 - b1)``, ``v = v b2 + g^2 (1 - b2)``,
``p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)``, ``ema = ema + (p - ema) (1 - d)``.

States in 8 bits: runs of 256 elements share two fp32 scales (A, B) = (max |m|, max v), and the codes c stand for
``m = A c |c| / 127^2`` (int8) and ``v = B (c / 255)^4`` (uint8, at least 1 for v > 0).  A value is off by at most half a
step of its code: |m| by about ``sqrt(A |m|) / 127``, v by ``2 (B v^3)^(1/4) / 255``.
"""

from __future__ import annotations

from collections.abc import Callable, Iterable, Sequence

import torch
from torch import Tensor

from . import ops  # noqa: F401  (loads the native operators)
from .ops import _fake, _refuse

STATE_RUN = 256  # elements of an 8-bit state that share a scale


def _define(name: str, schema: str, fake: Callable) -> None:
    op = f"jit_thc::{name}"
    torch.library.define(op, schema)

    def refuse(first, *args, **kwargs):
        _refuse(first[0] if len(first) else torch.empty(0))

    torch.library.impl(op, "CompositeExplicitAutograd")(refuse)
    _fake(op)(fake)


_define(
    "adamw_step",
    "(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, Tensor(d!)[] scales, "
    "Tensor(e!)[] masters, Tensor(f!)[] emas, float step, float lr, float beta1, float beta2, float eps, float weight_decay, "
    "float ema_decay, Tensor? device_step, Tensor? device_lr, Tensor? grad_norm, float max_norm) -> ()",
    lambda *args: None,
)
_define(
    "adamw_state_values",
    "(Tensor[] exp_avgs, Tensor[] exp_avg_sqs, Tensor[] scales) -> (Tensor[], Tensor[])",
    lambda avgs, sqs, scales: tuple([t.new_empty(t.shape, dtype=torch.float32) for t in ts] for ts in (avgs, avgs)),
)
_define("grad_norm", "(Tensor[] grads) -> Tensor", lambda grads: grads[0].new_empty((), dtype=torch.float32))


def _list(ts: Sequence[Tensor]) -> list[Tensor]:
    return ts if isinstance(ts, list) else list(ts)


@torch.no_grad()
def adamw_step(
    params: Sequence[Tensor],
    grads: Sequence[Tensor],
    exp_avgs: Sequence[Tensor],
    exp_avg_sqs: Sequence[Tensor],
    *,
    step: int | float | Tensor,
    lr: float | Tensor = 1e-3,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 0.0,
    scales: Sequence[Tensor] = (),
    masters: Sequence[Tensor] = (),
    emas: Sequence[Tensor] = (),
    ema_decay: float = 0.0,
    grad_norm: Tensor | None = None,
    max_norm: float = 0.0,
) -> None:
    """One AdamW step of `params` in place (the module's formulas), `step` the number of this step, from 1.

    params and grads have one dtype each, of fp32, bf16 and fp16.  exp_avgs and exp_avg_sqs are fp32 in their parameters'
    layout, or, with `scales` (fp32 [2, runs of 256]), contiguous int8 and uint8 codes.  masters: fp32 copies of 16-bit
    parameters, which take the step and are rounded into them.  emas: fp32 moving averages of the step's fp32 result (of a
    16-bit parameter without a master too, before it is rounded).  grad_norm: the norm of all
    gradients (one fp32 on the device); they are scaled by min(1, max_norm / (grad_norm + 1e-6)), and where it is not finite
    nothing is changed.  What the step writes lies in memory of its own; a gradient may be there twice.  step and lr may be
    one fp32 on the device, which a captured graph reads anew on each replay."""
    if not len(params):
        return
    on_device = isinstance(step, Tensor), isinstance(lr, Tensor)
    torch.ops.jit_thc.adamw_step(
        _list(params), _list(grads), _list(exp_avgs), _list(exp_avg_sqs), _list(scales), _list(masters), _list(emas),
        1.0 if on_device[0] else float(step), 0.0 if on_device[1] else float(lr), betas[0], betas[1], eps, weight_decay, ema_decay,
        step if on_device[0] else None, lr if on_device[1] else None, grad_norm, max_norm,
    )  # fmt: skip


@torch.no_grad()
def state_values(exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor], scales: Sequence[Tensor]) -> tuple[list[Tensor], list[Tensor]]:
    """The fp32 values of 8-bit states."""
    if not len(exp_avgs):
        return [], []
    return torch.ops.jit_thc.adamw_state_values(list(exp_avgs), list(exp_avg_sqs), list(scales))


@torch.no_grad()
def grad_norm(grads: Sequence[Tensor]) -> Tensor:
    """The 2-norm of all gradients (one dtype) together, as one fp32 on their device: squares summed in 64 bits in a fixed
    order."""
    return torch.ops.jit_thc.grad_norm(list(grads))


def _capturing(t: Tensor) -> bool:
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update on the operators above.  What it has besides:

    * ``state_bits=8``: moments as 8-bit codes for parameters of at least ``min_8bit_size`` elements (4 096); the smaller
      ones, whose state costs nothing, keep 32 bits;
    * ``master_weights``: fp32 copies of 16-bit parameters, which take the steps (``state[p]["master"]``);
    * ``ema_decay``: fp32 moving averages of the weights (``state[p]["ema"]``, ``ema_params``), begun at the weights of a
      parameter's first step.  An average takes the step's fp32 result, and moves in its parameter's steps only: a parameter
      without a gradient, or a step that is left out for its norm, leaves it as it is (an update of its own after every
      step, as in the reference's training script, would go on towards the weights there);
    * ``max_norm``: clipping by the norm of all gradients, which ``last_grad_norm`` keeps on the device; a step whose norm is
      not finite changes no tensor (it is counted);
    * ``capturable``: step counts on the device, one for all parameters that have taken the same steps, and a learning rate
      that may be a tensor there, so that a captured step can be replayed.  Its states are laid out by a step outside the
      capture, with the same parameters having gradients; other captured steps are refused.

    The state has torch.optim.AdamW's names (``step``, ``exp_avg``, ``exp_avg_sq``; the codes' ``scales``), and that
    optimizer's ``state_dict`` loads."""

    def __init__(
        self,
        params: Iterable,
        lr: float | Tensor = 1e-3,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        *,
        state_bits: int = 32,
        min_8bit_size: int = 4096,
        master_weights: bool = False,
        ema_decay: float | None = None,
        max_norm: float | None = None,
        capturable: bool = False,
    ) -> None:
        if isinstance(lr, Tensor) and not capturable:
            raise ValueError("a tensor learning rate needs capturable=True")
        if not isinstance(lr, Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"eps and weight_decay must not be negative, got {eps}, {weight_decay}")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if ema_decay is not None and not 0.0 <= ema_decay <= 1.0:
            raise ValueError(f"ema_decay must be in [0, 1], got {ema_decay}")
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self.max_norm = max_norm
        self.last_grad_norm: Tensor | None = None
        defaults = dict(
            lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, min_8bit_size=min_8bit_size,
            master_weights=master_weights, ema_decay=ema_decay, capturable=capturable,
        )  # fmt: skip
        super().__init__(params, defaults)

    def __getstate__(self) -> dict:
        """What copies and pickles hold: torch's optimizers give theirs by name."""
        return {**super().__getstate__(), "max_norm": self.max_norm, "last_grad_norm": self.last_grad_norm}

    # ------------------------------------------------------------------ state
    def _init_state(self, p: Tensor, group: dict) -> dict:
        state = self.state[p]
        missing = (
            "exp_avg" not in state
            or (group["master_weights"] and p.dtype != torch.float32 and "master" not in state)
            or (group["ema_decay"] is not None and "ema" not in state)
            or (group["capturable"] and not isinstance(state["step"], Tensor))
        )
        if missing and _capturing(p):
            raise RuntimeError("a captured AdamW step needs its states: take one step outside the capture first")
        if "exp_avg" not in state:
            if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
                state["exp_avg"] = torch.zeros(p.numel(), device=p.device, dtype=torch.int8)
                state["exp_avg_sq"] = torch.zeros(p.numel(), device=p.device, dtype=torch.uint8)
                state["scales"] = torch.zeros((2, -(-p.numel() // STATE_RUN)), device=p.device)
            else:
                state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            state["step"] = 0
        if group["master_weights"] and p.dtype != torch.float32 and "master" not in state:
            state["master"] = p.detach().to(torch.float32, copy=True)
        if group["ema_decay"] is not None and "ema" not in state:
            state["ema"] = state["master"].clone() if "master" in state else p.detach().to(torch.float32, copy=True)
        return state

    def _device_step(self, states: list[dict], device: torch.device) -> Tensor:
        """The step count that a capturable group's states share, on their device."""
        have = next((s["step"] for s in states if isinstance(s["step"], Tensor)), None)
        if have is None:
            have = torch.full((), float(states[0]["step"]), device=device, dtype=torch.float32)
        for s in states:
            s["step"] = have
        return have

    def _split_counts(self) -> None:
        """Parameters that take a step which others of their shared count do not take get a count of their own."""
        for group in self.param_groups:
            if not group["capturable"]:
                continue
            stepping: dict[int, list[dict]] = {}
            resting: set[int] = set()
            for p in group["params"]:
                state = self.state.get(p, {})
                if isinstance(state.get("step"), Tensor):
                    if p.grad is None:
                        resting.add(id(state["step"]))
                    else:
                        stepping.setdefault(id(state["step"]), []).append(state)
            for at, states in stepping.items():
                if at in resting:
                    if _capturing(states[0]["exp_avg"]):
                        raise RuntimeError("a captured AdamW step needs the same gradients as the step outside the capture")
                    own = states[0]["step"].clone()
                    for state in states:
                        state["step"] = own

    def ema_params(self, params: Iterable[Tensor] | None = None) -> list[Tensor]:
        """The moving averages of `params` (the optimizer's own, in their order), in `params`' shapes: what
        ``checkpoint.checkpoint_state`` takes as ``ema_params``.  A parameter that has taken no step yet gives its weights."""
        if params is None:
            params = [p for g in self.param_groups for p in g["params"]]
        return [self.state[p]["ema"] if "ema" in self.state.get(p, {}) else p.detach().float() for p in params]

    def load_state_dict(self, state_dict: dict) -> None:
        """This optimizer's or torch.optim.AdamW's state.  States keep their own types, which torch's loader converts to
        their parameters' (codes, and the fp32 states of 16-bit parameters)."""
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("a state with amsgrad or maximize does not load: this AdamW has neither")
        own = [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            if i not in saved:
                continue
            state = self.state[p]
            for key, value in saved[i].items():
                if key == "step":
                    state[key] = value
                elif isinstance(value, Tensor):
                    kept = value.dtype if key == "scales" or not value.is_floating_point() else torch.float32
                    state[key] = value.detach().to(p.device, kept, copy=True)
                    if value.shape == p.shape and kept == torch.float32:  # the parameter's layout
                        state[key] = torch.empty_like(p, dtype=kept).copy_(state[key])
        for group, defaults in zip(self.param_groups, own):
            for key, value in defaults.items():
                group.setdefault(key, value)
            shared: dict = {}  # counts of one value that a capturable group's states share
            for p in group["params"]:
                state = self.state.get(p, {})
                if "step" in state:
                    count = float(state["step"])
                    if group["capturable"]:
                        at = (p.device, count)
                        if at not in shared:
                            shared[at] = torch.full((), count, device=p.device, dtype=torch.float32)
                        state["step"] = shared[at]
                    else:
                        state["step"] = int(count)

    # ------------------------------------------------------------------- step
    @torch.no_grad()
    def step(self, closure: Callable | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._split_counts()
        calls: dict = {}  # one call for each set of tensors that share types, device, state width and step count
        for group in self.param_groups:
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise ValueError("AdamW takes no sparse gradients")
                if not group["capturable"] and _capturing(p):
                    raise RuntimeError("a captured AdamW step needs capturable=True")
                state = self._init_state(p, group)
                step = state["step"]
                key = (id(group), p.device, p.dtype, g.dtype, "scales" in state, id(step) if isinstance(step, Tensor) else step)
                calls.setdefault(key, (group, []))[1].append((p, g, state))
        norm = self.last_grad_norm = self._norm(calls) if self.max_norm is not None else None
        counted: set[int] = set()
        for group, members in calls.values():
            states = [s for _, _, s in members]
            if group["capturable"]:
                step = self._device_step(states, members[0][0].device)
                if id(step) not in counted:
                    counted.add(id(step))
                    step.add_(1)
            else:
                step = int(states[0]["step"]) + 1
                for s in states:
                    s["step"] = step
            ema = group["ema_decay"]
            adamw_step(
                [p for p, _, _ in members], [g for _, g, _ in members], [s["exp_avg"] for s in states],
                [s["exp_avg_sq"] for s in states], step=step, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                weight_decay=group["weight_decay"], scales=[s["scales"] for s in states if "scales" in s],
                masters=[s["master"] for s in states if "master" in s], emas=[s["ema"] for s in states] if ema is not None else (),
                ema_decay=ema or 0.0, grad_norm=norm, max_norm=self.max_norm or 0.0,
            )  # fmt: skip
        return loss

    def _norm(self, calls: dict) -> Tensor | None:
        """The norm of all gradients, one launch for each type of theirs."""
        by_type: dict = {}
        for _, members in calls.values():
            for _, g, _ in members:
                by_type.setdefault((g.device, g.dtype), []).append(g)
        if len({d for d, _ in by_type}) > 1:
            raise ValueError("clipping by the norm of all gradients needs them on one device")
        norms = [grad_norm(gs) for gs in by_type.values()]
        if len(norms) <= 1:
            return norms[0] if norms else None
        return torch.linalg.vector_norm(torch.stack(norms))
