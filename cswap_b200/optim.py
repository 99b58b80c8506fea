"""The optimizer's step over all parameters in one launch, its state in 32 bits or in 8.

* ``adamw_step``: AdamW over lists of tensors, averages in float32.
* ``adamw8_step``: the same with the averages in 8 bits, 2.02 bytes a parameter in place of 8; ``adamw8_state`` makes the state of
  a tensor, ``adamw8_pack`` and ``adamw8_unpack`` take averages in and out.
* ``gradient_norm``: the norm of all gradients, which both take for clipping without a copy to the host.
* ``AdamW``: a torch.optim.Optimizer on them.

Parameters, gradients and 16-bit copies of the parameters are float32, float16 or bfloat16, each tensor of its own type.
Tensors lie densely, in the same order in memory for a parameter and what belongs to it.  No two that are written overlap, and no
gradient overlaps one that is, unless it is the very tensor that is written for its parameter.
Averages are float32 operations, rounded one by one; the same call gives the same bits.  There is no CPU implementation.
"""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import codec

ADAMW8_GROUP = 128

State8 = Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]


def _ext():
    return codec._native or codec._load()


def gradient_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all values of all tensors, one float32 on their device; squares are summed in float64."""
    return _ext().gradient_norm(tensors)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], step: Union[int, torch.Tensor], lr: Union[float, torch.Tensor] = 1e-3,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               norm: Optional[torch.Tensor] = None, max_norm: float = 1.0,
               copies: Optional[Sequence[Optional[torch.Tensor]]] = None) -> None:
    """One step, in place: with t = `step`, counted from 1, and the gradients g times c = min(1, max_norm / (norm + 1e-6)) where
    a norm is given,

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    The averages m and v are float32, whatever the parameters' types.  `copies`: tensors that receive the new parameters in
    their own types.  `step` may be one int64 on the device, `lr` one float32, for steps that are captured into a graph."""
    _ext().adamw_step(params, grads, exp_avgs, exp_avg_sqs, copies, step, lr, betas[0], betas[1], eps, weight_decay, norm,
                      max_norm)


def adamw8_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], states: Sequence[State8],
                step: Union[int, torch.Tensor], lr: Union[float, torch.Tensor] = 1e-3,
                betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                norm: Optional[torch.Tensor] = None, max_norm: float = 1.0,
                copies: Optional[Sequence[Optional[torch.Tensor]]] = None, seed: int = 0) -> None:
    """adamw_step with each parameter's averages as `adamw8_state` has them.

    Groups of 128 consecutive values share a power of two; m is held to 4 bits of mantissa (one of them not stored) over 2^17,
    v over 2^33, rounded up or down at random so that the averages are right in the mean.  The random bits follow from `seed`
    (below 2^32), the step, the tensor's place in the lists and the value's index.  A gradient that is no number leaves its
    group's averages NaN."""
    _ext().adamw8_step(params, grads, states, copies, step, lr, betas[0], betas[1], eps, weight_decay, norm, max_norm, seed)


def adamw8_state(param: torch.Tensor) -> State8:
    """A state of zeros for a parameter: codes of exp_avg and exp_avg_sq (uint8, one a value) and the scales of their groups
    (one for 128)."""
    n = param.numel()
    groups = -(-n // ADAMW8_GROUP)
    return tuple(torch.zeros(k, dtype=torch.uint8, device=param.device) for k in (n, n, groups, groups))


def adamw8_pack(states: Sequence[State8], exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor]) -> None:
    """Writes averages in float32 into states, rounded to the nearest code."""
    _ext().adamw8_convert(states, exp_avgs, exp_avg_sqs, True)


def adamw8_unpack(states: Sequence[State8], exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor]) -> None:
    """Writes the averages that states hold into float32 tensors."""
    _ext().adamw8_convert(states, exp_avgs, exp_avg_sqs, False)


# what a group with capturable has besides, of which the first two lie on the device
_DEVICE_KEYS = ("device_step", "device_lr", "told_lr")


class AdamW(torch.optim.Optimizer):
    """AdamW on adamw_step, or with `bits` 8 on adamw8_step, a launch for each group of parameters.

    `max_norm`: the gradients of all groups together are scaled to that norm where theirs is larger.  `seed`: of the rounding
    in 8 bits.  A step takes the number of steps that a parameter has been through from its state; with `capturable` it is
    counted on the device, once for all of a group, and the learning rate lies there too, so that a captured step may be
    replayed: `set_lr` changes it for replays, a scheduler's change of the groups arrives with the next step that is not
    captured.  `state_dict` has the number of steps that the device has counted; what goes on from it may count either way.
    A group of which some call is refused has made no step, the groups before it have."""

    def __init__(self, params: Iterable, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, bits: int = 32, max_norm: Optional[float] = None, seed: int = 0,
                 capturable: bool = False):
        if bits not in (8, 32):
            raise ValueError("bits must be 8 or 32")
        if not 0 <= seed < 1 << 32:
            raise ValueError("seed must be below 2^32")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError("max_norm must not be negative")
        self.bits, self.max_norm, self.seed, self.capturable = bits, max_norm, seed, capturable
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self) -> dict:
        """What copies and pickles have: torch's keeps the groups, their state and the defaults alone."""
        return {**super().__getstate__(), **{name: getattr(self, name) for name in ("bits", "max_norm", "seed", "capturable")}}

    def _state_of(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        if not state:
            state["step"] = 0
            if self.bits == 8:
                state["exp_avg"], state["exp_avg_sq"], state["exp_avg_scale"], state["exp_avg_sq_scale"] = adamw8_state(p)
            else:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return state

    def _count_on_device(self, group: dict) -> None:
        """The group's number of steps and its rate, where its parameters are."""
        held = [(p, self.state[p]) for p in group["params"] if self.state.get(p)]
        device = held[0][0].device
        group["device_step"] = torch.full((1,), max(s["step"] for _, s in held), dtype=torch.int64, device=device)
        group["device_lr"] = torch.empty(1, dtype=torch.float32, device=device).fill_(group["lr"])
        group["told_lr"] = group["lr"]

    def set_lr(self, lr: float) -> None:
        """The learning rate of all groups, also of steps that have been captured."""
        for group in self.param_groups:
            group["lr"] = lr
            if "device_lr" in group:
                group["device_lr"].fill_(lr)
                group["told_lr"] = lr

    @torch.no_grad()
    def step(self, closure=None):
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if capturing:
            fresh = any(p.grad is not None and not (self.state.get(p) and "device_step" in group)
                        for group in self.param_groups for p in group["params"])
            if fresh or not self.capturable:
                raise RuntimeError("a step is captured with capturable=True, and after one that is not")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work: List[tuple] = []  # of one group and one number of steps so far
        every: List[torch.Tensor] = []
        for at, group in enumerate(self.param_groups):
            by_step: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("AdamW takes dense gradients")
                g = p.grad
                if not (g.is_contiguous() and p.is_contiguous()) and g.stride() != p.stride():
                    g = torch.empty_like(p, dtype=g.dtype, memory_format=torch.preserve_format).copy_(g)
                state = self._state_of(p)
                every.append(g)
                by_step.setdefault(0 if self.capturable else state["step"], []).append((p, g, state))
            if self.capturable and by_step:
                if "device_step" not in group:
                    self._count_on_device(group)
                if not capturing and group["told_lr"] != group["lr"]:
                    group["device_lr"].fill_(group["lr"])
                    group["told_lr"] = group["lr"]
            work += [(at, group, taken, members) for taken, members in by_step.items()]
        if not every:
            return loss
        clip = dict(norm=gradient_norm(every), max_norm=self.max_norm) if self.max_norm is not None else {}
        for at, group, taken, members in work:
            params, grads, states = ([m[i] for m in members] for i in range(3))
            rest = dict(betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], **clip)
            step, lr = (group["device_step"].add_(1), group["device_lr"]) if self.capturable else (taken + 1, group["lr"])
            try:
                if self.bits == 8:
                    held = [(s["exp_avg"], s["exp_avg_sq"], s["exp_avg_scale"], s["exp_avg_sq_scale"]) for s in states]
                    adamw8_step(params, grads, held, step, lr, seed=(self.seed + at * 0x632be5ab) & 0xffffffff, **rest)
                else:
                    adamw_step(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], step, lr, **rest)
            except Exception:  # a call that is refused is no step
                if self.capturable:
                    group["device_step"].sub_(1)
                raise
            for state in states if not capturing else ():
                state["step"] += 1
        return loss

    def state_dict(self) -> dict:
        """As torch's.  Steps that replays have made are counted on the device alone: they are asked for here, and what lies on
        the device besides the averages stays out."""
        for group in self.param_groups:
            if "device_step" in group:
                self._set_steps(group, int(group["device_step"]))
        state = super().state_dict()
        for group in state["param_groups"]:
            for key in _DEVICE_KEYS:
                group.pop(key, None)
        return state

    def _set_steps(self, group: dict, taken: int) -> None:
        for p in group["params"]:
            if self.state.get(p):
                self.state[p]["step"] = taken

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, which casts a state to its parameter's type: here codes stay codes, averages float32.  A step that was
        captured before belongs to the state before, and is to be captured again."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().to(p.device, copy=True)
        for group in self.param_groups:
            taken, *_ = [group.pop(key, None) for key in _DEVICE_KEYS]
            if taken is not None:  # a checkpoint whose groups hold the device's count, which is the one that is right
                self._set_steps(group, int(taken))
            if self.capturable and any(self.state.get(p) for p in group["params"]):
                self._count_on_device(group)
