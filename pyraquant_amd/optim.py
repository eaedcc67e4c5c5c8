"""AdamW over the tensors of a model in one launch for MI355X (gfx950), with states in 32 bits or in 8.

  AdamW(params, lr, betas, eps, weight_decay, bits=32, max_norm=None, seed=0)

A torch.optim.Optimizer for what Mxfp4Linear and LowRankAdapters tune: many small tensors of bf16, fp16 or fp32 values. Everything
is computed in fp32 and rounded to the parameter's type once. One launch takes 448 tensors; two with ``max_norm``, which holds the norm of all
gradients to a limit as torch.nn.utils.clip_grad_norm_ does, without the host and without writing the gradients: ``grad_norm`` is a
tensor on the GPU. A norm that is infinite or NaN leaves parameters, states and counts as they were.

``bits=8`` keeps two bytes a value and two more for each 128: the mean of the gradients with 3 mantissa bits, the root of the mean of their squares
with 4, over 16 powers of two below the block's largest. What is cut off is rounded up or down by a hash of the value's place, the
step and ``seed``, so that averages move by less than a step of the grid. Elsewhere AdamW is the usual one, but that a group's states are all there from its
first use on, in one piece; sparse gradients, several parameters in one place and, in a group, several devices are refused.

``lr`` may be a tensor of one fp32 value on the GPU, which the kernel reads: a captured step then follows it. Steps can be
captured after the first one has been taken; the step counts live on the GPU, so replays go on counting. A graph goes on with the
rate, parameters, gradients and states that it was captured with: capture again where they are replaced (load_state_dict, parameters that
moved), and keep the optimizer, which holds them, as long as its graphs. Gradients that were not made in the capture are the caller's to keep.
"""
from __future__ import annotations

from collections import defaultdict
from typing import List, Optional, Tuple

import torch

from . import _lib

_PARTS = {32: ("step", "exp_avg", "exp_avg_sq"), 8: ("step", "exp_avg_8bit", "exp_avg_root_8bit", "exponents")}


class AdamW(torch.optim.Optimizer):
    """AdamW (see the module). A group may have ``lr``, ``betas``, ``eps``, ``weight_decay``, ``bits`` and ``seed`` of its own;
    ``max_norm`` counts for all groups together.

    A group's states lie end to end, each parameter's from a multiple of 128 values on (``offsets``), room for every parameter, whether it gets
    gradients or not. A parameter whose entry of ``state`` is taken away begins anew. ``state[p]`` holds views of them:
    ``step`` (a count for each 1024 values, all alike), and ``exp_avg`` and ``exp_avg_sq`` in fp32, or ``exp_avg_8bit``, ``exp_avg_root_8bit``
    and ``exponents`` (pq_adamw_states of the C header)."""

    def __init__(self, params, lr=1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 *, bits: int = 32, max_norm: Optional[float] = None, seed: int = 0):
        assert max_norm is None or max_norm > 0, f"max_norm {max_norm}: a limit above 0, or None"
        self.max_norm = max_norm
        self.grad_norm: Optional[torch.Tensor] = None
        self._plans = {}
        self._in_graphs = []   # plans that were replaced and that captured graphs go on with
        self._loading = None   # the state dict that is being loaded
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, bits=bits, seed=seed))

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            assert isinstance(g["lr"], torch.Tensor) or g["lr"] >= 0, f"lr {g['lr']}"
            assert len(g["betas"]) == 2 and all(0 <= b < 1 for b in g["betas"]), f"betas {g['betas']}"
            assert g["eps"] >= 0 and g["weight_decay"] >= 0, f"eps {g['eps']}, weight decay {g['weight_decay']}"
            assert g["bits"] in _PARTS, f"states have 8 or 32 bits (got {g['bits']})"
            for p in g["params"]:
                if p.dtype not in (torch.bfloat16, torch.float16, torch.float32):
                    raise ValueError(f"unsupported dtype {p.dtype} (expected bfloat16, float16 or float32)")
        except Exception:
            self.param_groups.pop()
            raise

    def _plan(self, i: int):
        """The plan of group i, made at its first use and where its parameters, or the states that they have in ``state``, are others; states that
        are there go with them."""
        i = range(len(self.param_groups))[i]      # (from the end, too)
        g = self.param_groups[i]
        plan = self._plans.get(i)
        if plan is None or not plan.holds(g["params"], g["bits"], self.state):
            plan = _lib.load_tune().Plan(g["params"], g["bits"])
            names = _PARTS[g["bits"]]
            given = []
            for k, p in enumerate(g["params"]):
                old, new = self.state.get(p, {}), dict(zip(names, plan.of(k)))
                if old:
                    assert set(old) == set(names) and all(old[n].numel() == new[n].numel() for n in names), (
                        f"the states of a parameter of {p.numel()} values are {sorted(old)}: not those of {g['bits']} bits and its size")
                    with torch.no_grad():
                        for n in names:
                            new[n].copy_(old[n].reshape(new[n].shape))
                            if old[n].is_cuda:      # (it goes away, and may be another stream's)
                                old[n].record_stream(torch.cuda.current_stream(old[n].device))
                given.append(new)
            for p, new in zip(g["params"], given):
                self.state.pop(p, None)      # (in the parameters' order)
                self.state[p] = new
            plan.give(given)
            self._drop(i)
            self._plans[i] = plan
        return plan

    def _drop(self, *groups: int) -> None:
        self._in_graphs += [plan for plan in (self._plans.pop(i, None) for i in groups) if plan is not None and plan.captured()]

    @torch.no_grad()
    def step(self, closure=None):
        """One step over every parameter that has a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [(self._plan(i), g["lr"], *g["betas"], g["eps"], g["weight_decay"], g["seed"])
                  for i, g in enumerate(self.param_groups) if g["params"]]
        self.grad_norm = _lib.load_tune().step(groups, self.max_norm or 0.0)
        return loss

    def offsets(self, group: int = 0) -> List[int]:
        """Where each parameter of a group begins in its states and moments."""
        return self._plan(group).offsets()

    def states(self, group: int = 0):
        """The states of a group as they are kept, end to end: (exp_avg, exp_avg_sq) in fp32, or the codes of both and the exponents."""
        return self._plan(group).states()

    def moments(self, dtype: torch.dtype = torch.float32, group: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """(means of the gradients, roots of the means of their squares) of a group, end to end: new tensors of values, whatever the states'
        bits (those of 8-bit states are exact in bf16 and fp32). Zeros behind the end of each parameter."""
        return self._plan(group).moments(dtype)

    def load_moments(self, mean: torch.Tensor, root: torch.Tensor, steps: int, group: int = 0) -> None:
        """States from values, laid out as ``moments`` gives them: to go on from another optimizer's, or in other bits. 8-bit states
        take the nearest value."""
        self._plan(group).load(mean, root, steps)

    def load_state_dict(self, state_dict) -> None:
        """A state dict of this class. Groups take the bits and the seed that it was saved with."""
        def take(_, d):      # the last hook before the load: what others made of the dict (torch would cast states to the parameters' types)
            self._loading = d
            return {**d, "state": {}}

        handle = self.register_load_state_dict_pre_hook(take)
        try:
            super().load_state_dict(state_dict)
        finally:
            handle.remove()
            self._loading = None

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def __setstate__(self, state) -> None:
        loading = self.__dict__.get("_loading")
        if loading is not None:
            ids = [i for g in loading["param_groups"] for i in g["params"]]
            params = [p for g in state["param_groups"] for p in g["params"]]
            own = defaultdict(dict)
            for i, p in zip(ids, params):
                if i in loading["state"]:
                    own[p] = {k: v.detach().clone() for k, v in loading["state"][i].items()}
            state = {**state, "state": own}
        super().__setstate__(state)
        self.__dict__.setdefault("max_norm", None)
        self.grad_norm = None
        self.__dict__.setdefault("_plans", {})
        self.__dict__.setdefault("_in_graphs", [])
        self.__dict__.setdefault("_loading", None)
        self._drop(*list(self._plans))
