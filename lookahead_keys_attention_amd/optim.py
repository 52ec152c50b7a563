"""`AdamW`: a torch.optim.Optimizer over ops.adamw_step, the optimiser of the reference's training script (Adam with clipped
gradients, train_triton.py:219-259) as a few launches for all parameters of a group.

    AdamW(params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, state_bits=32, stochastic_rounding=True, seed=None)

state_bits 8 keeps both moments as e4m3 numbers with an exponent for each 256 of them, 2 bytes a parameter instead of 8.  Those
are rounded by chance; `stochastic_rounding` says whether parameters of 16 bits are too (of 32 bits they are exact).  `seed`, a whole
number of 64 bits, decides the random numbers: replicas that are to stay alike, as those of data-parallel processes, need the same.
Without it one is drawn from the generator of the CPU, which `torch.manual_seed` sets, whenever parameters have their first gradient.  `max_norm`
clips the gradients of all groups by their common norm; it is left in `grad_norm`, a number on the GPU, behind each step.  A saved
state brings it along, as it does the options of the groups.

Steps are counted on the GPU, for each parameter those in which it had a gradient, and nothing is read back, so a step can be
captured into a graph once one of the same parameters has been taken; `lr` of a group may be a float32 tensor of one element on the
GPU, which a replay reads anew.  A graph counts for the parameters that shared a count when it was recorded: where some of them
have paused since, it is recorded again.
"""
from __future__ import annotations

import operator

import torch

from . import ops

_MOMENTS = ("exp_avg", "exp_avg_sq")
_ODD = 6364136223846793005   # (seeds go round 64 bits)


def _order(t):
    """The steps of a dense tensor's axes, but for those of one element, which say nothing."""
    return [(n, s) for n, s in zip(t.shape, t.stride()) if n != 1] if t.numel() else []


class AdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, state_bits=32, stochastic_rounding=True, seed=None):
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32:
                raise ValueError("AdamW: a learning rate in a tensor is one float32 number")
        elif not lr >= 0:
            raise ValueError(f"AdamW: the learning rate is not negative, got {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"AdamW: betas are in [0, 1), got {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"AdamW: eps and weight_decay are not negative, got {eps} and {weight_decay}")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"AdamW: max_norm is not negative, got {max_norm}")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: states of 8 or 32 bits, got {state_bits}")
        if seed is not None:
            if not hasattr(type(seed), "__index__") or isinstance(seed, torch.Tensor) or not -2 ** 63 <= (number := operator.index(seed)) < 2 ** 64:
                raise ValueError(f"AdamW: a seed is a whole number of 64 bits, got {seed!r}")
            seed = number
        self.max_norm, self.grad_norm = max_norm, None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, stochastic_rounding=stochastic_rounding, seed=seed))

    def __getstate__(self):   # (of copies and pickles)
        return super().__getstate__() | dict(max_norm=self.max_norm, grad_norm=None)

    def state_dict(self):
        return super().state_dict() | dict(max_norm=self.max_norm)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = [call for group in self.param_groups for call in self._calls(group)]
        self.grad_norm = norm = None
        if not calls:
            return loss
        if self.max_norm is not None and len(calls) > 1:
            norm = self._norm([p.grad for _, params in calls for p in params])
        for group, params in calls:
            first = self.state[params[0]]
            small = group["state_bits"] == 8
            chance = small or (group["stochastic_rounding"] and params[0].dtype != torch.float32)
            states = {k: [self.state[p][k] for p in params] for k in first if k not in ("step", "seed")}
            got = ops.adamw_step(params, [p.grad for p in params], states["exp_avg"], states["exp_avg_sq"], first["step"], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                                 weight_decay=group["weight_decay"], max_norm=self.max_norm, norm=None if norm is None else norm.to(params[0].device), seed=first["seed"] if chance else None,
                                 exp_avg_exponents=states.get("exp_avg_exponents"), exp_avg_sq_exponents=states.get("exp_avg_sq_exponents"))
            self.grad_norm = got
        return loss

    @staticmethod
    def _norm(grads):
        """Of gradients of all types together."""
        kinds = {}
        for g in grads:
            kinds.setdefault((g.dtype, g.device), []).append(g)
        norms = [ops.gradient_norm(k).to(grads[0].device) for k in kinds.values()]
        return norms[0] if len(norms) == 1 else torch.linalg.vector_norm(torch.stack(norms).double()).float()

    def _calls(self, group):
        """(group, parameters) for each call of a step: parameters of one type that have had a gradient in the same steps."""
        new, calls, paused = {}, {}, set()
        for p in group["params"]:
            if p.grad is None:
                if self.state.get(p):
                    paused.add(id(self.state[p]["step"]))
                continue
            if p.grad.is_sparse:
                raise RuntimeError("AdamW: gradients are dense")
            if not p.is_cuda:
                raise RuntimeError(f"AdamW: the HIP kernels need parameters on the GPU (got {p.device})")
            if not self.state[p]:
                new.setdefault((p.dtype, p.device), []).append(p)
        for (dtype, device), params in new.items():
            self._begin(params, device, group["state_bits"], group.get("seed"))
        for p in group["params"]:
            if p.grad is not None:
                calls.setdefault((p.dtype, id(self.state[p]["step"])), (group, []))[1].append(p)
        for (_, count), (_, params) in calls.items():
            if count in paused:
                self._part(params)
            paused.add(count)   # (each call counts: of two types that began as one, the second goes its own way)
        return list(calls.values())

    def _part(self, params):
        """Parameters that go on without others of their count: from here on they have one of their own, and a seed."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: some parameters have no gradient, or another type, that were in one call with others so far; take such a step before one is captured")
        first = self.state[params[0]]
        step, seed = first["step"].clone(), first["seed"] * _ODD + self._place(params[0])   # (another one for each place, as no parameter parts from the same seed twice)
        for p in params:
            self.state[p]["step"], self.state[p]["seed"] = step, seed

    def _place(self, param):
        """Which of all parameters it is, from one."""
        return next(i for i, p in enumerate((p for group in self.param_groups for p in group["params"]), 1) if p is param)

    def _begin(self, params, device, bits, seed):
        """States of parameters that have a gradient for the first time: one count of steps and one seed for all of them."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take a step before one is captured (states that begin inside a graph would begin again at every replay)")
        step = torch.zeros(1, dtype=torch.int64, device=device)
        if seed is None:
            seed = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,)).to(device)
        else:   # (one for each place: sets of parameters that begin apart have numbers apart)
            number = (seed * _ODD + self._place(params[0])) % 2 ** 64
            seed = torch.tensor([number - 2 ** 64 if number >= 2 ** 63 else number], device=device)
        for p in params:
            state = self.state[p]
            state["step"], state["seed"] = step, seed
            for name in _MOMENTS:
                if bits == 8:
                    state[name] = torch.empty_like(p, dtype=torch.float8_e4m3fn)
                    state[name].view(torch.uint8).zero_()
                    state[name + "_exponents"] = torch.zeros((p.numel() + 255) // 256, dtype=torch.int8, device=device)
                else:
                    state[name] = torch.zeros_like(p, dtype=torch.float32)

    def load_state_dict(self, state_dict):
        """States come back in the types that they were saved in (torch.optim.Optimizer casts them to their parameters'); those that counted alike share one count again."""
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        if any("state_bits" not in group for group in state_dict["param_groups"]):
            raise ValueError("AdamW: these states were not saved by this optimizer")
        for i, p in zip(saved, params):
            for key in _MOMENTS if i in state_dict["state"] else ():
                value = state_dict["state"][i][key]
                if value.shape != p.shape:
                    raise ValueError("AdamW: a saved state has another shape than its parameter")
                if value.dtype != torch.float32 and _order(value) != _order(torch.empty_like(p, device="meta")):
                    raise ValueError("AdamW: a saved state of 8 bits has another order in memory than its parameter, and its exponents go by that")
        super().load_state_dict(state_dict)
        self.max_norm = state_dict.get("max_norm", self.max_norm)   # (like the options of the groups)
        shared = {}
        for i, p in zip(saved, params):
            if i not in state_dict["state"]:
                continue
            state = {}
            for key, value in state_dict["state"][i].items():
                if key in _MOMENTS:
                    state[key] = torch.empty_like(p, dtype=value.dtype)
                    # (numbers of 8 bits are copied as bytes)
                    same = value.dtype if value.dtype == torch.float32 else torch.uint8
                    state[key].view(same).copy_(value.view(same))
                elif key in ("step", "seed"):
                    number = int(value)
                    state[key] = (key, number, p.device, p.dtype)
                else:
                    state[key] = value.to(device=p.device, copy=True)
            begun = (state["step"], state["seed"])
            if begun not in shared:
                shared[begun] = [torch.full((1,), k[1], dtype=torch.int64, device=p.device) for k in begun]
            state["step"], state["seed"] = shared[begun]
            self.state[p] = state

