"""AdamW whose step is one pass over all tensors, with gradient clipping and, on request, states in 8 bits.

What the reference's trainer does per tensor in PyTorch (trainers/base_trainer_accelerate.py:367-388: clip_grad_norm_, optimizer.step)
becomes ``ops.grad_norm`` and ``ops.adamw_step``; nothing is read back to the host, so that a step can be captured in a graph.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import ops


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` for CUDA parameters (fp32, bf16 or fp16, contiguous).

    ``max_norm``: gradients are scaled by ``min(1, max_norm / (norm + 1e-6))``, norm taken over all parameters; a step whose norm is
    not finite is left out.  ``state_bits=8``: tensors of at least ``min_8bit_size`` elements keep their moments in 8 bits
    (``ops.adamw_state`` says what the codes stand for), rounded stochastically with ``seed``; ``seed=None`` rounds to nearest, with
    which a second moment hardly follows gradients that shrink.  bf16 parameters are rounded the same way, by all bits that they
    drop; fp16 parameters to nearest.  ``lr`` may be a 0-dim
    fp32 tensor on the device, which a captured step reads anew each time.

    Parameters are counted from the first step in which they had a gradient, as PyTorch does."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 max_norm: Optional[float] = None, state_bits: int = 32, min_8bit_size: int = 4096, seed: Optional[int] = 0):
        if not isinstance(lr, Tensor) and not lr >= 0:
            raise ValueError(f"lr {lr}")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"betas {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"eps {eps}, weight_decay {weight_decay}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm {max_norm}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: 8 or 32")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size, seed=seed))
        self.max_norm = max_norm
        self.grad_norm: Optional[Tensor] = None       # of the last step with max_norm, 0-dim on the device

    def __getstate__(self):
        """PyTorch's keeps three attributes; copies and pickles clip as well."""
        return {**super().__getstate__(), "max_norm": self.max_norm, "grad_norm": None}

    @staticmethod
    def _outside_of_a_graph(what: str) -> None:
        """What makes states once would make them anew in every replay."""
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"AdamW: {what} cannot be captured: take a step with the same gradients outside of the graph first")

    def _new_state(self, group, p, step):
        if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
            codes = lambda: torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
            scales = torch.full((2, -(-p.numel() // 256)), 27, dtype=torch.uint8, device=p.device)
            return dict(step=step, exp_avg=codes(), exp_avg_sq=codes(), scales=scales)
        zeros = lambda: torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return dict(step=step, exp_avg=zeros(), exp_avg_sq=zeros())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # with a number over all groups, so that its random numbers do not depend on which others have a gradient
        first, work = 0, []
        for g in self.param_groups:
            work.append((g, [(i, p) for i, p in enumerate(g["params"], first) if p.grad is not None]))
            first += len(g["params"])
        for _, params in work:
            for _, p in params:
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
        norm = None
        if self.max_norm is not None:
            grads = [p.grad for _, params in work for _, p in params]
            if grads:
                norm = self.grad_norm = ops.grad_norm(grads)
        for group, params in work:
            # Parameters that have always stepped together share one count (and one launch); those that begin now begin together, and
            # where some of a count's parameters have no gradient this time, the others go on with a count of their own.
            counts: dict = {}
            fresh = None
            for i, p in params:
                st = self.state[p]
                if not st:
                    self._outside_of_a_graph("a parameter's first step")
                    if fresh is None or fresh.device != p.device:
                        fresh = torch.zeros((), dtype=torch.int64, device=p.device)
                    st.update(self._new_state(group, p, fresh))
                _, together, numbers = counts.setdefault(id(st["step"]), (st["step"], [], []))
                together.append(p)
                numbers.append(i)
            if counts and len(params) < len(group["params"]):
                present = {id(p) for _, p in params}
                for key in {id(self.state[p]["step"]) for p in group["params"] if id(p) not in present and self.state.get(p)} & counts.keys():
                    self._outside_of_a_graph("a step from which a parameter is left out for the first time")
                    step, together, numbers = counts[key]
                    step = step.clone()
                    for p in together:
                        self.state[p]["step"] = step
                    counts[key] = (step, together, numbers)
            for step, together, numbers in counts.values():
                states = [self.state[p] for p in together]
                ops.adamw_step(together, [p.grad for p in together], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], step,
                               lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], grad_norm=norm,
                               max_norm=self.max_norm, scales=[s.get("scales") for s in states], seed=group["seed"],
                               numbers=None if group["seed"] is None else numbers)
        return loss

    def load_state_dict(self, state_dict):
        """A state dict of this class or of ``torch.optim.AdamW`` (whose states become fp32; ``maximize`` and ``amsgrad`` raise).  States keep
        their own type where PyTorch casts them to their parameter's; what a group does not say stays as it is; counts that were shared
        are again."""
        for g in state_dict["param_groups"]:
            for name in ("maximize", "amsgrad"):
                if g.get(name):
                    raise RuntimeError(f"AdamW: a state dict with {name} belongs to another optimiser")
        mine = [dict(g) for g in self.param_groups]
        super().load_state_dict(state_dict)
        for old, g in zip(mine, self.param_groups):
            for name, value in old.items():
                g.setdefault(name, value)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                self.state[p] = self._loaded(p, state_dict["state"][i])
        for g in self.param_groups:
            shared: dict = {}
            for p in g["params"]:
                st = self.state.get(p)
                if st:
                    st["step"] = shared.setdefault((p.device, int(st["step"])), st["step"])

    @staticmethod
    def _loaded(p: Tensor, st: dict) -> dict:
        if not st:
            return {}
        types = dict(step=torch.int64, scales=torch.uint8)
        types["exp_avg"] = types["exp_avg_sq"] = torch.uint8 if st.get("scales") is not None else torch.float32
        return {k: torch.as_tensor(st[k]).detach().to(device=p.device, dtype=t, copy=True).contiguous() for k, t in types.items() if st.get(k) is not None}
