"""AdamW over many tensors in few launches, with moments in 32 or in 8 bits."""
from typing import Iterable, List, Optional, Sequence, Tuple

import torch

from nanotron_amd import _ops

BLOCK = _ops.ADAMW_BLOCK   # elements of an 8-bit moment that share a scale


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], *, lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, step: int, grad_scale: Optional[torch.Tensor] = None,
               copies: Optional[Sequence[Optional[torch.Tensor]]] = None) -> None:
    """One AdamW step (decoupled weight decay) over the lists, in place; step counts from 1.

    params and grads: float32, float16 or bfloat16, in any mixture; exp_avgs and exp_avg_sqs: float32.  All contiguous and
    on one device.  Arithmetic is fp32; a 16-bit parameter is rounded to nearest once a step.  grad_scale (one float32 on the
    device: a clipping factor, the inverse of a loss scale) multiplies every gradient.  lr and step are part of the launch: a
    captured graph repeats them.  copies: for each parameter a tensor
    (or None) that receives its new value, rounded from fp32 to that tensor's type, as the 16-bit weights beside fp32 masters."""
    _ops.host.adamw(params, grads, exp_avgs, exp_avg_sqs, None, None, copies, lr, betas[0], betas[1], eps, weight_decay, step, 0, grad_scale)


def adamw_8bit_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
                    exp_avg_scales: Sequence[torch.Tensor], exp_rmss: Sequence[torch.Tensor], exp_rms_scales: Sequence[torch.Tensor], *,
                    lr: float, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, step: int,
                    seed: int, grad_scale: Optional[torch.Tensor] = None, copies: Optional[Sequence[Optional[torch.Tensor]]] = None) -> None:
    """`adamw_step` with moments in 8 bits: exp_avgs holds E4M3 codes of the first moment, exp_rmss those of the ROOT of the
    second (uint8, one a parameter element); each block of 256 elements has a power-of-two scale (float32, value = code /
    scale) in the tensors beside them (`moments_8bit` makes all four).  Codes are rounded stochastically with bits hashed
    from the element's index and `seed`, which should differ from step to step.  Parameters move by the moments before they
    are rounded."""
    _ops.host.adamw(params, grads, exp_avgs, exp_rmss, exp_avg_scales, exp_rms_scales, copies, lr, betas[0], betas[1], eps, weight_decay, step, seed, grad_scale)


def moments_8bit(param: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Zero moments for `adamw_8bit_step`: (exp_avg, its scales, exp_rms, its scales)."""
    def scales():
        return torch.ones(-(-param.numel() // BLOCK), dtype=torch.float32, device=param.device)

    def codes():
        return torch.zeros(param.shape, dtype=torch.uint8, device=param.device)

    return codes(), scales(), codes(), scales()


def dequantize_moment(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What the codes of an 8-bit moment stand for, float32 in their shape."""
    return _ops.host.adamw_unpack(codes, scales)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update in few launches; `state_bits` 32 or 8 chooses the moments (`adamw_step`,
    `adamw_8bit_step`).

    Where a parameter is an fp32 master, `copies` in its group (a list beside `params`, None for a parameter without) names
    the 16-bit tensors of the model that take its new values.  A parameter is stepped by its `.grad`, or else its `main_grad`
    (what an FP8Linear with a 16-bit master leaves in fp32), or else the `.grad` of its copy (`grad_of`); zero_grad() clears
    all three.  `grad_scale` of step() multiplies all gradients (a clipping factor left on the device).  Every parameter
    counts its own steps.  `seed` shifts the stochastic rounding of 8-bit moments.  State dicts hold the moments as they are,
    and no copies; one of torch.optim.AdamW is taken over with its 32-bit moments (ValueError for amsgrad or maximize)."""

    def __init__(self, params: Iterable, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, seed: int = 0):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed, copies=None)
        self._check(defaults)
        super().__init__(params, defaults)

    @staticmethod
    def _check(group: dict) -> None:
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")
        if group["lr"] < 0 or group["eps"] < 0 or group["weight_decay"] < 0 or not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError(f"lr, eps and weight_decay must not be negative and betas lie in [0, 1), got {group['lr']}, {group['eps']}, "
                             f"{group['weight_decay']}, {group['betas']}")
        if group.get("params") is not None and group["copies"] is not None and len(group["copies"]) != len(group["params"]):
            raise ValueError(f"copies must name one tensor (or None) for each of {len(group['params'])} parameters, got {len(group['copies'])}")

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check(self.param_groups[-1])
        except Exception:   # (a TypeError of the comparisons among them)
            self.param_groups.pop()
            raise

    @staticmethod
    def grad_of(param: torch.Tensor, copy: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """The gradient that a parameter is stepped by, None if it has none."""
        for grad in (param.grad, getattr(param, "main_grad", None), None if copy is None else copy.grad):
            if grad is not None:
                return grad
        return None

    def params_and_copies(self):
        """(parameter, copy or None) of all groups."""
        for group in self.param_groups:
            yield from zip(group["params"], group["copies"] or [None] * len(group["params"]))

    def zero_grad(self, set_to_none: bool = True) -> None:
        super().zero_grad(set_to_none)
        for p, copy in self.params_and_copies():
            if getattr(p, "main_grad", None) is not None:
                if set_to_none:
                    p.main_grad = None
                else:
                    p.main_grad.zero_()
            if copy is not None and copy.grad is not None:
                if set_to_none:
                    copy.grad = None
                else:
                    copy.grad.zero_()

    def state_dict(self) -> dict:
        # (the copies are other people's tensors)
        d = super().state_dict()
        for g in d["param_groups"]:
            g["copies"] = None
        return d

    def load_state_dict(self, state_dict: dict) -> None:
        for g in state_dict["param_groups"]:   # (of torch.optim.AdamW or Adam)
            for name in ("amsgrad", "maximize"):
                if g.get(name):
                    raise ValueError(f"AdamW has no {name}, with which this state was made")
            if not g.get("decoupled_weight_decay", True) and g["weight_decay"]:
                raise ValueError("AdamW decays weights decoupled from their gradients (decoupled_weight_decay), this state's optimizer did not")
        own = [{k: g[k] for k in ("copies", "seed")} for g in self.param_groups]
        super().load_state_dict(state_dict)
        for g, kept in zip(self.param_groups, own):
            g["copies"] = kept["copies"]
            # what torch's groups do not say: moments that are not codes are 32-bit ones
            g.setdefault("seed", kept["seed"])
            g.setdefault("state_bits", 32)
        # (the base class casts state to the parameter's type; moments keep theirs, or become the fp32 that a step takes)
        for g, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(g["params"], saved["params"]):
                if key in state_dict["state"]:
                    state = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v for k, v in state_dict["state"][key].items() if k != "step"}
                    if g["state_bits"] == 32:
                        state = {k: v.float() if isinstance(v, torch.Tensor) else v for k, v in state.items()}
                    # (torch counts in a tensor; parameters share launches by their number of steps)
                    self.state[p] = {"step": int(state_dict["state"][key]["step"]), **state}

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: Optional[torch.Tensor] = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            # parameters that have taken the same number of steps share launches; so do those of one device
            runs: dict = {}
            for p, copy in zip(group["params"], group["copies"] or [None] * len(group["params"])):
                grad = self.grad_of(p, copy)
                if grad is None:
                    continue
                if grad.is_sparse:
                    raise ValueError("AdamW does not take sparse gradients")
                state = self.state[p]
                if not state:
                    state["step"] = 0
                    if group["state_bits"] == 8:
                        state["exp_avg"], state["exp_avg_scale"], state["exp_rms"], state["exp_rms_scale"] = moments_8bit(p)
                    else:
                        state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                        state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                runs.setdefault((state["step"] + 1, p.device), []).append((_plain(p), _plain(grad).contiguous(), state, copy))
            for (step, _), run in runs.items():
                params, grads, states, copies = zip(*run)
                common = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], step=step,
                              grad_scale=grad_scale, copies=copies if group["copies"] is not None else None)

                def of(name: str) -> List[torch.Tensor]:
                    return [s[name] for s in states]

                if group["state_bits"] == 8:
                    adamw_8bit_step(params, grads, of("exp_avg"), of("exp_avg_scale"), of("exp_rms"), of("exp_rms_scale"), seed=group["seed"] + step, **common)
                else:
                    adamw_step(params, grads, of("exp_avg"), of("exp_avg_sq"), **common)
                for state in states:   # (a call that refused its arguments has stepped nothing)
                    state["step"] = step
        return loss


def _plain(t: torch.Tensor) -> torch.Tensor:
    """The storage of a parameter whose class says something else about its data (an FP8Parameter's fp8 copy)."""
    return t if type(t) in (torch.Tensor, torch.nn.Parameter) else t.as_subclass(torch.Tensor)
