"""The Muon optimiser on the kernels of fc3d.ops.muon_step: momentum, orthogonalisation of the update by
Newton-Schulz products and the weights' update for all matrices of a parameter group in one sequence of launches.
For hidden weights of two axes or more; biases, norms, the first layer and the head are usually left to Adam
(split_parameters)."""
from __future__ import annotations

import torch

from . import ops


def split_parameters(modules, leave=()):
    """(matrices, others): the modules' weights of two axes or more, which Muon takes, and all other parameters, among
    them everything below a submodule that `leave` names (the first layer, the head).  Each parameter once, in order."""
    modules = [modules] if isinstance(modules, torch.nn.Module) else list(modules)
    # a shared parameter goes by all its names, in all modules
    named = [(name, p) for module in modules for name, p in module.named_parameters(remove_duplicate=False)]
    kept = {id(p) for name, p in named if any(name == n or name.startswith(n + ".") for n in leave)}
    matrices, others, seen = [], [], set()
    for _, p in named:
        if id(p) not in seen:
            seen.add(id(p))
            (others if id(p) in kept or p.dim() < 2 else matrices).append(p)
    return matrices, others


class Muon(torch.optim.Optimizer):
    """lr, momentum, nesterov, weight_decay, steps, coefficients, eps, scale: as for fc3d.ops.muon_step, per group.
    The momentum is float32 whatever the weights' type.  step() can be captured into a graph once every weight has been
    stepped outside of one; the replays keep the rates they were captured with."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients=ops.NS_COEFFICIENTS, eps: float = 1e-7, scale: str = "spectral"):
        if not lr >= 0.0:
            raise ValueError(f"lr must not be negative (got {lr})")
        if not 0.0 <= momentum <= 1.0:
            raise ValueError(f"momentum must be in [0, 1] (got {momentum})")
        if not weight_decay >= 0.0:
            raise ValueError(f"weight_decay must not be negative (got {weight_decay})")
        ops._ns_arguments(steps, coefficients, eps)
        ops.muon_scale((1, 1), scale)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, scale=scale))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError(f"Muon is for weights of two axes or more, got one of shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: take one step before capturing one into a graph (a momentum made during the "
                                           "capture would be cleared by every replay)")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
                lists = by_device.setdefault(p.device, ([], [], []))
                for to, t in zip(lists, (p, p.grad, state["momentum_buffer"])):
                    to.append(t)
            for p, g, m in by_device.values():
                ops.muon_step(p, g, m, **{k: v for k, v in group.items() if k in _STEP})
        return loss

    def load_state_dict(self, state_dict):
        """The base class casts a state to its weight's type; the momenta are taken over as they were saved."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, mine):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None:
                self.state[p]["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32).copy_(m)


_STEP = ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps", "scale")
