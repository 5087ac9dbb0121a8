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
    root), rounded stochastically; bf16 parameters are rounded stochastically too (vig_amd.adamw_step says how), by numbers that go on over all groups.  Two runs with the same `seed` give the same bits.
    max_norm clips the gradients of all parameters, which must lie on one device, to that norm; `grad_norm` holds it afterwards, as a
    number on the device.  A step whose norm is not finite changes no parameter and no moment (it does count).
    capturable=True counts a parameter group's steps on the device, so that step() can be captured into a graph and
    replayed (without it a captured step is refused): run one step outside of the capture first, with gradients of the same parameters, and give lr as a float32 tensor there if it is to change between replays.
    Each parameter counts the steps in which it had a gradient; those that a graph counts together have to go on together.
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
        if any(p.grad.is_sparse for _, params in todo for p in params):
            raise RuntimeError("AdamW takes no sparse gradients")
        if _capturing():
            self._check_capture(todo)
        elif self._captured and any(self._shared(group, params) & {id(t) for t in self._captured} for group, params in todo if group["capturable"]):
            raise RuntimeError("AdamW: parameters whose steps a captured step counts together have gradients in different steps; load the states anew to count them apart")
        scale = None
        if self.max_norm is not None:
            grads = [p.grad for _, params in todo for p in params]
            if grads:
                self.grad_norm, scale = ops.grad_norm(grads, self.max_norm)
        numbers = None
        for group, params in todo:
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and not lr.is_cuda:
                lr = float(lr)
            states = [self._state_of(p, group) for p in params]
            capturable = group["capturable"]
            if capturable:
                self._count_there(group, params, states)
            else:
                self._count_here(group)
            calls = {}
            for p, state in zip(params, states):
                if capturable:
                    t = id(state["step"])
                else:
                    t = state["step"] = state["step"] + 1
                calls.setdefault((p.device, t, "exp_avg_scale" in state), []).append((p, state))
            for (_, _, bits8), some in calls.items():
                lists = [[p for p, _ in some], [p.grad for p, _ in some]] + [[s[name] for _, s in some] for name in ("exp_avg", "exp_avg_sq")]
                if bits8:
                    lists += [[s[name + "_scale"] for _, s in some] for name in ("exp_avg", "exp_avg_sq")]
                first = None
                if bits8 or any(p.dtype == torch.bfloat16 for p, _ in some):  # (what is rounded by random words)
                    numbers = numbers or self._numbers()
                    first = [numbers[p] for p, _ in some]
                ops.adamw_step(*lists, step=some[0][1]["step"], lr=lr, betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], grad_scale=scale, seed=self.seed,
                               first=first)
        return loss

    def _numbers(self):
        """The number of each parameter's first element: they go on over all groups in blocks of 256, so that no two elements of a step are rounded by the same word,
        and stay a parameter's own whichever others have gradients."""
        numbers, n = {}, 0
        for group in self.param_groups:
            for p in group["params"]:
                numbers[p] = n
                n += -(-p.numel() // 256) * 256
        return numbers

    # Steps are counted for each parameter: state["step"] is a number on the host or, in a capturable group, one on the device, the same tensor for all that have had
    # gradients in the same steps.  group["step_on_device"] lists those.

    _captured = ()  # counts that a captured step moves

    def _check_capture(self, todo):
        """Before anything is recorded: a count on the host would be the same in each replay, and a state or a count made here would be made anew by each."""
        for group, params in todo:
            if params and not group["capturable"]:
                raise RuntimeError("AdamW: a parameter group whose step is captured has to be capturable")
            if any(not self.state.get(p) or not isinstance(self.state[p]["step"], torch.Tensor) for p in params) or self._shared(group, params):
                raise RuntimeError("AdamW: run one step outside of the capture first, with gradients of the same parameters")
        self._captured += tuple({id(t): t for _, params in todo for t in (self.state[p]["step"] for p in params)}.values())

    def _shared(self, group, params):
        """The counts (by id) of parameters some of which have a gradient and some have none."""
        if len(params) == len(group["params"]):
            return set()
        left = {id(self.state[p]["step"]) for p in group["params"] if p.grad is None and self.state.get(p) and isinstance(self.state[p]["step"], torch.Tensor)}
        return left & {id(self.state[p]["step"]) for p in params if self.state.get(p)}

    def _count_there(self, group, params, states):
        """The parameters' counts on the device, one further."""
        shared = self._shared(group, params)
        if shared or not all(isinstance(s["step"], torch.Tensor) for s in states):
            self._move_there(group)
            shared, apart = self._shared(group, params), {}
            for state in states:
                t = state["step"]
                if id(t) in shared:
                    if id(t) not in apart:
                        apart[id(t)] = t.clone()
                    state["step"] = apart[id(t)]
            self._list_counts(group)
        for t in {id(s["step"]): s["step"] for s in states}.values():
            t.add_(1)

    def _move_there(self, group):
        """Counts on the host, as those of states just made, onto the device."""
        made = {}
        for p in group["params"]:
            state = self.state.get(p)
            if state and not isinstance(state["step"], torch.Tensor):
                key = (p.device, state["step"])
                if key not in made:
                    made[key] = torch.full((), state["step"], dtype=torch.int64, device=p.device)
                state["step"] = made[key]

    def _list_counts(self, group):
        group["step_on_device"] = listed = {}
        for t in {id(t): t for t in (self.state[p]["step"] for p in group["params"] if self.state.get(p))}.values():
            name, k = str(t.device), 1
            while name in listed:
                k += 1
                name = f"{t.device} {k}"
            listed[name] = t

    def _count_here(self, group):
        """Steps that the device has counted so far, back to numbers on the host."""
        if group.pop("step_on_device", None) is None:
            return
        known = {}
        for p in group["params"]:
            t = self.state[p]["step"] if self.state.get(p) else 0
            if isinstance(t, torch.Tensor):
                if id(t) not in known:
                    known[id(t)] = (int(t), t)
                self.state[p]["step"] = known[id(t)][0]

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch.optim's, but states keep the types they were saved in (8 bits among them; others are fp32).  Takes torch.optim.AdamW's too."""
        if any(group.get("amsgrad") or group.get("maximize") for group in state_dict["param_groups"]):
            raise ValueError("AdamW has neither amsgrad nor maximize")
        super().load_state_dict(state_dict)
        self._captured = ()
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        alone = set()  # parameters whose count is their group's
        for i, p in zip(ids, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if name in ("exp_avg", "exp_avg_sq") and value.dtype != torch.float8_e4m3fn and value.shape == p.shape:
                    # (torch holds them in the parameter's type; they lie as the parameter does, whichever way it lay when they were saved)
                    self.state[p][name] = torch.empty_like(p, dtype=torch.float32).copy_(value)
                elif name == "step":
                    self.state[p][name] = int(value)
                    if not isinstance(value, torch.Tensor):
                        alone.add(p)
                elif isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().to(p.device).clone(memory_format=torch.preserve_format)
        for group in self.param_groups:
            for name in ("state_bits", "capturable"):
                group.setdefault(name, self.defaults[name])
            counts = group.pop("step_on_device", {})  # (by the devices of the program that saved them, which these parameters need not be on)
            for p in group["params"]:
                if counts and p in alone:  # (a group's steps were once counted by one number for all)
                    self.state[p]["step"] = int(counts[str(p.device)]) if str(p.device) in counts else max(map(int, counts.values()))
            if group["capturable"]:
                self._move_there(group)
                self._list_counts(group)
