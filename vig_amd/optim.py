"""AdamW over the library's update kernels, with the interface of torch.optim's optimisers."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops

LEAST_8_BIT = 4096  # elements from which on a tensor's states are held in 8 bits: below, they weigh nothing beside its launch


def _capturing():
    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay; moments without amsgrad) in a few launches for all parameters together.

    state_bits=8 holds the moments of tensors of 4096 elements and more in 8 bits with a scale for each 256 (the second one as its
    root), rounded stochastically; bf16 parameters are rounded stochastically too (vig_amd.adamw_step says how).  Two runs with the same `seed` give the same bits.
    max_norm clips the gradients of all parameters, which must lie on one device, to that norm; `grad_norm` holds it afterwards, as a
    number on the device.  A step whose norm is not finite changes no parameter and no moment (it does count).
    capturable=True counts the steps of a parameter group on the device, so that step() can be captured into a graph and
    replayed (without it a captured step is refused): run one step outside of the capture first, with gradients of the same parameters, and give lr as a float32 tensor there if it is to change between replays.
    Parameters' version counters are moved, so that copies of weights kept by the layers are renewed."""

    def __init__(self, params, lr=1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_norm: Optional[float] = None, seed: int = 0, capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32; got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative; got {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError(f"betas must lie in [0, 1), eps and weight_decay must not be negative; got {betas}, {eps}, {weight_decay}")
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError(f"max_norm must not be negative; got {max_norm}")
        self.max_norm, self.seed, self.grad_norm = max_norm, seed, None
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay, "state_bits": state_bits, "capturable": capturable})

    def __getstate__(self):
        return super().__getstate__() | {"max_norm": self.max_norm, "seed": self.seed, "grad_norm": None}

    def _state_of(self, p, group):
        state = self.state[p]
        if not state:
            state["step"] = 0
            if group["state_bits"] == 8 and p.numel() >= LEAST_8_BIT:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
                    state[name + "_scale"] = torch.zeros(-(-p.numel() // 256), device=p.device)
            else:
                state["exp_avg"], state["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32) for _ in range(2))
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo = [(group, [p for p in group["params"] if p.grad is not None]) for group in self.param_groups]
        if _capturing():
            self._check_capture(todo)
        scale = None
        if self.max_norm is not None:
            grads = [p.grad for _, params in todo for p in params]
            if grads:
                self.grad_norm, scale = ops.grad_norm(grads, self.max_norm)
        for group, params in todo:
            if not group["capturable"]:
                self._count_here(group)
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and not lr.is_cuda:
                lr = float(lr)
            calls = {}
            for p in params:
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW takes no sparse gradients")
                state = self._state_of(p, group)
                if group["capturable"]:
                    t = None
                else:
                    t = state["step"] = state["step"] + 1
                calls.setdefault((p.device, t, "exp_avg_scale" in state), []).append((p, state))
            counted = {}
            for (device, t, bits8), some in calls.items():
                if t is None:
                    t = counted.get(device)
                    if t is None:
                        t = counted[device] = self._count_of(group, device).add_(1)
                lists = [[p for p, _ in some], [p.grad for p, _ in some]] + [[s[name] for _, s in some] for name in ("exp_avg", "exp_avg_sq")]
                if bits8:
                    lists += [[s[name + "_scale"] for _, s in some] for name in ("exp_avg", "exp_avg_sq")]
                ops.adamw_step(*lists, step=t, lr=lr, betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], grad_scale=scale, seed=self.seed)
        return loss

    def _check_capture(self, todo):
        """Before anything is recorded: a count on the host would be the same in each replay, and a state made here would be cleared by each."""
        for group, params in todo:
            if params and not group["capturable"]:
                raise RuntimeError("AdamW: a parameter group whose step is captured has to be capturable")
            counts = group.get("step_on_device", {})
            if any(not self.state.get(p) or str(p.device) not in counts for p in params):
                raise RuntimeError("AdamW: run one step outside of the capture first, with gradients of the same parameters")

    def _count_of(self, group, device):
        """The group's number of steps on the device."""
        counts = group.setdefault("step_on_device", {})
        if str(device) not in counts:
            # (steps that were counted one by one, before the group became capturable)
            done = max((self.state[p]["step"] for p in group["params"] if p.device == device and p in self.state), default=0)
            counts[str(device)] = torch.full((), done, dtype=torch.int64, device=device)
        return counts[str(device)]

    def _count_here(self, group):
        """Steps that the device has counted so far, back to the parameters' own numbers."""
        counts = group.pop("step_on_device", {})
        for p in group["params"]:
            if p in self.state and str(p.device) in counts:
                self.state[p]["step"] = int(counts[str(p.device)])

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch.optim's, but states keep the types they were saved in (8 bits among them; others are fp32).  Takes torch.optim.AdamW's too."""
        if any(group.get("amsgrad") or group.get("maximize") for group in state_dict["param_groups"]):
            raise ValueError("AdamW has neither amsgrad nor maximize")
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if name in ("exp_avg", "exp_avg_sq") and value.dtype != torch.float8_e4m3fn and value.shape == p.shape:
                    # (torch holds them in the parameter's type; they lie as the parameter does, whichever way it lay when they were saved)
                    self.state[p][name] = torch.empty_like(p, dtype=torch.float32).copy_(value)
                elif isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().to(p.device).clone(memory_format=torch.preserve_format)
            if "step" in self.state.get(p, {}):
                self.state[p]["step"] = int(self.state[p]["step"])
        for group in self.param_groups:
            for name in ("state_bits", "capturable"):
                group.setdefault(name, self.defaults[name])
            counts = group.pop("step_on_device", {})  # (by the devices of the program that saved them, which these parameters need not be on)
            for p in group["params"]:
                if counts and p in self.state:
                    self.state[p]["step"] = int(counts[str(p.device)] if str(p.device) in counts else max(counts.values()))
                    if group["capturable"]:
                        self._count_of(group, p.device)
