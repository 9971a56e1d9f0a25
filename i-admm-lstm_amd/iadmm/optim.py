"""The optimizer of the training loop (main.py:350 ``optimizer.step()``) on the multi-tensor kernel of
csrc/adamw.hip: one launch for up to 48 parameters, moments in 32 or in 8 bits, clipping by the global
norm in the same pass."""
from __future__ import annotations

import torch

from . import ops


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over fp32 or bf16 parameters on the GPU.

    ``state_bits=8`` keeps the two moments as 8-bit codes with two shared exponents per 256 elements
    (:func:`iadmm.ops.adamw_step`): 2 bytes a parameter instead of 8.  Codes, and bf16 parameters, are rounded
    up or down at random by ``seed``, the step and the parameter's place: a run repeats bit for bit, and ranks
    that step with the same gradients stay equal.

    ``max_norm``: gradients count as scaled by min(1, max_norm / (norm + 1e-6)), norm over all gradients of all
    groups; ``norm`` holds the last one (0-dim device tensor).  ``.grad`` is not changed.

    ``capturable=True`` counts the steps on the device, so that a step captured into a graph counts its
    replays; make one step before the capture (the state is allocated there), and load a state before it (a loaded
    state is other tensors than a captured step's).  A captured step keeps the ``lr`` of its capture unless ``lr`` is
    a 1-element fp32 device tensor.

    Parameters without a gradient are left alone, as torch.optim does.  ``state_dict`` has torch.optim.AdamW's
    entries ("step", "exp_avg", "exp_avg_sq"; with 8 bits "exponents" too), and a state of torch.optim.AdamW, or of
    Adam without weight decay, loads into 32 bits."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, max_norm=None,
                 seed=0, capturable=False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        if not isinstance(lr, torch.Tensor) and not 0 <= lr < float("inf"):
            raise ValueError(f"lr must not be negative, got {lr}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0 and weight_decay >= 0):
            raise ValueError(f"betas {betas}, eps {eps} or weight_decay {weight_decay} is out of range")
        self.state_bits, self.max_norm, self.seed, self.capturable = state_bits, max_norm, int(seed), bool(capturable)
        self.norm = None
        self._counts = {}  # a group's first parameter -> int64 device tensor of the steps made, and its elements (capturable)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        """What a copy or a pickle holds: torch's entries and this optimizer's own settings (torch keeps its own alone)."""
        own = ("state_bits", "max_norm", "seed", "capturable", "norm")
        return {**super().__getstate__(), **{k: getattr(self, k) for k in own}}

    def __setstate__(self, state):
        super().__setstate__(state)  # (load_state_dict comes here too, with the state and the groups)
        self.__dict__.setdefault("_counts", {})  # (a copy's next step gathers them from the parameters' "step")

    def add_param_group(self, group):
        super().add_param_group(group)  # (params may be a generator: looked at where they are a list)
        try:
            for p in self.param_groups[-1]["params"]:
                if p.dtype not in (torch.float32, torch.bfloat16):
                    raise TypeError(f"parameters must be float32 or bfloat16, got {p.dtype}")
                if not p.is_contiguous():
                    raise ValueError(f"parameters must be contiguous, got strides {p.stride()} for {tuple(p.shape)}")
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def _state(self, p):
        """The state of one parameter, zeros at first."""
        s = self.state[p]
        if not s:
            kw = dict(device=p.device, memory_format=torch.contiguous_format)
            kind = torch.uint8 if self.state_bits == 8 else torch.float32
            s["step"] = 0
            s["exp_avg"], s["exp_avg_sq"] = (torch.zeros_like(p, dtype=kind, **kw) for _ in range(2))
            if self.state_bits == 8:
                s["exponents"] = torch.zeros(-(-p.numel() // ops.ADAM_BLOCK), 2, dtype=torch.int8, device=p.device)
        return s

    def _count(self, params):
        """The group's steps as one device tensor, whose elements the parameters' "step" entries are."""
        counts, own = self._counts.get(params[0], (None, ()))
        # (a copy of this optimizer, a changed group or a state put in from outside: entries that are not these elements)
        if len(own) != len(params) or any(self.state[p].get("step") is not c for p, c in zip(params, own)):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("make one step before the capture: the steps' counts are not on the device yet")
            made = [int(self.state[p].get("step", 0)) for p in params]
            if len(own) == len(params) and counts.device == params[0].device:  # a captured step may hold its address
                counts.copy_(torch.tensor(made))
            else:
                counts = torch.tensor(made, dtype=torch.int64, device=params[0].device)
                own = counts.unbind()
                self._counts[params[0]] = counts, own
            for p, c in zip(params, own):
                self.state[p]["step"] = c
        return counts

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        plain = lambda x: (x.resolve_neg() if x.is_neg() else x).contiguous()  # noqa: E731
        grads = [[None if p.grad is None else plain(p.grad) for p in g["params"]] for g in self.param_groups]
        every = [x for gs in grads for x in gs if x is not None]
        if not every:
            return loss
        if self.max_norm is not None:
            self.norm = ops.grad_norm(every)
        for gi, (group, gs) in enumerate(zip(self.param_groups, grads)):
            if all(x is None for x in gs):
                continue
            params = group["params"]
            if self.capturable and torch.cuda.is_current_stream_capturing() and not all(self.state[p] for p in params):
                raise RuntimeError("make one step before the capture: the moments are not allocated yet")
            # (with counts on the device every parameter has a state, also one that has had no gradient yet)
            states = [self._state(p) if self.capturable or x is not None else None for p, x in zip(params, gs)]
            if self.capturable:
                step = self._count(params)
            else:
                for s in states:
                    if s is not None and not isinstance(s["step"], int):
                        s["step"] = int(s["step"])
                step = [1 if x is None else s["step"] + 1 for s, x in zip(states, gs)]
            of = lambda k: [None if s is None else s[k] for s in states]  # noqa: E731
            ops.adamw_step(params, gs, of("exp_avg"), of("exp_avg_sq"), step, group["lr"], group["betas"], group["eps"],
                           group["weight_decay"], of("exponents") if self.state_bits == 8 else None, self.norm
                           if self.max_norm is not None else None, self.max_norm, self.seed + gi)
            if not self.capturable:
                for s, x in zip(states, gs):
                    if x is not None:
                        s["step"] += 1
        return loss

    def moments(self, p, dtype=torch.float32):
        """(exp_avg, exp_avg_sq) of a parameter as numbers, whatever their form."""
        s = self._state(p)
        if self.state_bits == 8:
            return ops.adamw_decode8(s["exp_avg"], s["exp_avg_sq"], s["exponents"], dtype)
        return s["exp_avg"].to(dtype), s["exp_avg_sq"].to(dtype)

    def load_state_dict(self, state_dict):
        """As torch.optim's, but the moments keep their own type (torch casts a state to its parameter's).  A
        state with 32 bits does not load into 8; one with 8 bits loads into 32."""
        of = [(p, state_dict["state"].get(i)) for group, saved in zip(self.param_groups, state_dict["param_groups"])
              for p, i in zip(group["params"], saved["params"])]
        if any(g.get("maximize") or g.get("amsgrad") for g in state_dict["param_groups"]):
            raise ValueError("a state of an optimizer with maximize or amsgrad does not load")
        if any(g.get("weight_decay") and g.get("decoupled_weight_decay", True) is False for g in state_dict["param_groups"]):
            raise ValueError("a state of Adam with a weight decay inside its gradients does not load: the decay is decoupled here")
        for p, s in of:
            if s is None or not s:
                continue
            if not {"step", "exp_avg", "exp_avg_sq"} <= set(s) or "max_exp_avg_sq" in s:
                raise ValueError(f"not a state of AdamW or Adam (without amsgrad): {sorted(s)}")
            if self.state_bits == 8 and "exponents" not in s:
                raise ValueError("a state with 32 bits does not load into an optimizer with 8")
            if s["exp_avg"].shape != p.shape or s["exp_avg_sq"].shape != p.shape:
                raise ValueError(f"a state of {tuple(s['exp_avg'].shape)} does not fit a parameter of {tuple(p.shape)}")
            if "exponents" in s and ([s[k].dtype for k in ("exp_avg", "exp_avg_sq", "exponents")] !=
                                     [torch.uint8, torch.uint8, torch.int8]
                                     or s["exponents"].numel() != -(-p.numel() // ops.ADAM_BLOCK) * 2):
                raise ValueError("not the codes and exponents of 8-bit moments (another optimizer may have cast them)")
        super().load_state_dict(state_dict)
        for g in self.param_groups:  # (Adam's mark: without a decay it loads, and the group is AdamW's from here on)
            g.pop("decoupled_weight_decay", None)
        for p, s in of:
            if s is None or not s:
                continue
            new = {"step": int(s["step"])}
            if "exponents" in s:
                codes = [s[k].to(p.device, copy=True).contiguous() for k in ("exp_avg", "exp_avg_sq", "exponents")]
                if self.state_bits == 8:
                    new["exp_avg"], new["exp_avg_sq"], new["exponents"] = codes
                else:
                    new["exp_avg"], new["exp_avg_sq"] = (t.clone() for t in ops.adamw_decode8(*codes, torch.float32))
            else:
                new["exp_avg"], new["exp_avg_sq"] = (s[k].to(p.device, torch.float32, copy=True).contiguous()
                                                     for k in ("exp_avg", "exp_avg_sq"))
            self.state[p] = new
