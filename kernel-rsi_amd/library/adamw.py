"""AdamW over all of a model's tensors in a few launches, on gfx950 (MI355X) HIP kernels, with states in 32 bits or
in 8: adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr=...), grad_norm(grads), and AdamW, a
torch.optim.Optimizer on them.

For every tensor with a gradient, in fp32, with t the count of its steps:
  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
  w = w (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
All tensors of a call are changed in place by one launch for each 60 to 80 of them, after one that forms
the step's factors; clipping adds the gradients' norm, a launch for each 160. The counts live on
the device (steps, int32, one per tensor), and the rate may (a float32 tensor of one number), so a captured step goes on
counting and can be given another rate between replays.
  masters    fp32 copies of 16-bit parameters: they are stepped, and each parameter is overwritten with their rounding,
             whatever it holds (AdamW, below, looks for changed ones). Without masters steps below half a rounding
             of a parameter are lost.
  max_norm   gradients are scaled to this norm over all tensors where theirs is larger: the norm is computed first
             (or given, as norm: one of several shards). Where it is not finite nothing changes, counts neither.
  scales     8-bit states: exp_avgs and exp_avg_sqs are float8_e4m3fn codes of m and of sqrt(v), scales float32
             [2, ceil(n / 256)], one for each 256 elements of m and of the root. New codes are rounded up or down at random, m
             right on average and the root in its square (rounded to nearest, v would stand still: it changes by 1 - b2 in a
             step). The random numbers follow from seed, t, the tensor's place in the list and the element's.
Parameters, states and gradients are contiguous (a gradient that is not is copied), of bf16, fp16 or fp32, gradients of the
parameters' type or fp32. Nothing is recorded for a backward; what a graph has saved of the tensors that are stepped counts
as changed.
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
import _hip  # noqa: E402


def grad_norm(grads):
    """The root of the sum of squares of all gradients (None has no part): a float32 scalar on their device, the same
    bits each time."""
    grads = list(grads)
    norm = _hip.native().grad_norm(grads)
    return _hip.grad_norm(grads) if norm is None else norm


def _check_numbers(lr, betas, eps, weight_decay, max_norm):
    b1, b2 = betas
    if not isinstance(lr, torch.Tensor) and not 0 <= lr < float("inf"):
        raise ValueError(f"lr={lr} is not a rate")
    if not (0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError(f"betas={betas} are not in [0, 1)")
    if not 0 <= eps < float("inf") or not 0 <= weight_decay < float("inf"):
        raise ValueError(f"eps={eps}, weight_decay={weight_decay}: not negative, and finite")
    if 0 < eps < 2.0 ** -126:  # 1 / eps overflows, and an element without any gradient would step by 0 * infinity
        raise ValueError(f"eps={eps}: zero, or a normal number of fp32 (2^-126 at least)")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"max_norm={max_norm} is not a norm")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               masters=None, scales=None, max_norm=None, norm=None, seed=0):
    """One step of all tensors, in place (see the module); returns the norm that it went by, or None."""
    _check_numbers(lr, betas, eps, weight_decay, max_norm)
    if norm is not None and max_norm is None:
        raise ValueError("a norm without max_norm")
    args = (params, grads, exp_avgs, exp_avg_sqs, steps, lr, float(betas[0]), float(betas[1]), float(eps),
            float(weight_decay), masters, scales, None if max_norm is None else float(max_norm), norm, int(seed))
    done = _hip.native().adamw_step(*args)
    return _hip.adamw_step(*args) if done is None else done[0]


def _marks(params):
    """What differs once a parameter was changed in place or given other data."""
    try:
        return [(p._version, p.data_ptr()) for p in params]
    except RuntimeError:  # a tensor of inference mode has no version
        return [(0 if p.is_inference() else p._version, p.data_ptr()) for p in params]


def _follow(master, p):
    """The master of a parameter that may have been changed: taken anew where p is no longer its rounding."""
    master.copy_(torch.where(master.to(p.dtype) == p, master, p.float()))


class AdamW(torch.optim.Optimizer):
    """AdamW on these kernels. state_bits: 32 or 8. masters: whether 16-bit parameters have fp32 masters (None: yes).
    max_norm: of all gradients together. A group's lr may be a float32 tensor on the device. The state of a parameter:
    step, exp_avg, exp_avg_sq and, where they are used, master and scales; it begins with the first gradient.
    A parameter that was changed in place (loaded, clamped, averaged) goes on from there: its master is taken from it where it
    is no longer the master's rounding. Changes that torch does not count, through .data or between the replays of a captured
    step, need masters_from_parameters(), or the next step undoes them. Loaded masters stand.
    A step that makes states cannot be captured into a graph; others can, with gradients that stay where they are, and so
    can the first after states were loaded, but not a copy's first. Each step goes by what `param_groups` and
    `state` hold at the time. Where that is not what a captured step had (loaded or replaced states, another group or
    parameter, a first gradient), capture again, after a step that is not captured."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32, masters=None,
                 max_norm=None, seed=0):
        _check_numbers(lr, betas, eps, weight_decay, max_norm)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.state_bits, self.masters, self.max_norm, self.seed = state_bits, masters, max_norm, seed
        self._lists, self._held, self._ids = None, [], []
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "masters": self.masters, "max_norm": self.max_norm,
                "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._lists, self._held, self._ids = None, [], []

    def _new_state(self, p):
        _hip._dtype("parameters", p)
        if not p.is_contiguous():
            raise ValueError(f"parameters must be contiguous, got one of shape {tuple(p.shape)} with strides {p.stride()}")
        state = {"step": torch.zeros((), device=p.device, dtype=torch.int32)}
        kind = torch.float32 if self.state_bits == 32 else _hip.E4M3
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros(p.shape, device=p.device, dtype=kind)
        if self.state_bits == 8:
            state["scales"] = torch.zeros(2, -(-p.numel() // _hip.BLOCK_8BIT), device=p.device, dtype=torch.float32)
        if p.dtype != torch.float32 and self.masters in (None, True):
            state["master"] = p.detach().float()
        return state

    def _made_lists(self, fresh):
        """Per group, the lists of a call for each device and type of its parameters with a state, those with a master
        (loaded states may be of either kind) apart from those without. The steps of a list are one tensor, of which each
        parameter's state has a view. The last entry: the marks of parameters with masters after the step before (None: not
        known)."""
        known = {p: mark for _, ps, *_, marks in self._lists or () for p, mark in zip(ps, marks)}
        known.update(zip(fresh, _marks(fresh)))
        lists = []
        for group in self.param_groups:
            parts = {}
            for p in group["params"]:
                if self.state.get(p):
                    parts.setdefault((p.device, p.dtype, "master" in self.state[p]), []).append(p)
            for ps in parts.values():
                states = [self.state[p] for p in ps]
                steps = torch.stack([s["step"].reshape(()) for s in states])
                for s, step in zip(states, steps):
                    s["step"] = step
                lists.append((group, ps, steps, *([s[k] for s in states] if k in states[0] else None
                                                  for k in ("exp_avg", "exp_avg_sq", "master", "scales")),
                              [known.get(p) for p in ps if "master" in states[0]]))
        return lists

    def _current(self):
        """The groups, their parameters that have a state or now get one, and the tensors of their states: what the lists
        are made of."""
        held, state_of = [], self.state.get
        for group in self.param_groups:
            held.append(group)
            for p in group["params"]:
                state = state_of(p)
                if state:
                    held.append(p)
                    held.extend(state.values())
                elif p.grad is not None:
                    held.append(p)
        return held

    def _make_lists(self, fresh):
        """fresh: parameters whose masters are new or loaded, and stand."""
        self._lists = self._made_lists(fresh)
        self._held = self._current()  # kept, so that no other object comes to one's identity
        self._ids = [*map(id, self._held)]

    def _bring_lists_up_to_date(self):
        """Not in a capture, whose replays would clear new states and form the steps from the old ones again."""
        if self._lists is not None and self._ids == [*map(id, self._current())]:
            return
        params = [p for group in self.param_groups for p in group["params"] if p.grad is not None or self.state.get(p)]
        _hip._on_gpu(*params)
        if params and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW makes its states and their counts in its first step, and where parameters or states "
                               "have changed or got their first gradient: that step must not be captured, a replay would "
                               "set them back")
        new = [p for p in params if not self.state.get(p)]
        for p in new:
            self.state[p] = self._new_state(p)
        self._make_lists(new)

    @torch.no_grad()
    def masters_from_parameters(self):
        """Takes every master from its parameter, where that is no longer the master's rounding."""
        for group in self.param_groups:
            for p in group["params"]:
                if "master" in self.state.get(p, ()):
                    _follow(self.state[p]["master"], p)

    def _norm(self):
        """Of all gradients, on the device of the first; None without any."""
        parts = {}
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    parts.setdefault((p.device, p.grad.dtype), []).append(p.grad)
        if not parts:
            return None
        norms = [grad_norm(g) for g in parts.values()]
        return norms[0] if len(norms) == 1 else torch.linalg.vector_norm(torch.stack([n.to(norms[0].device) for n in norms]))

    @torch.compiler.disable
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._bring_lists_up_to_date()
        norm = None if self.max_norm is None else self._norm()
        for group, ps, steps, m, v, masters, scales, marks in self._lists:
            if masters is not None and marks != (now := _marks(ps)):
                for p, master, before, mark in zip(ps, masters, marks, now):
                    if mark != before:
                        _follow(master, p)
            grads = [p.grad for p in ps]
            kinds = {g.dtype for g in grads if g is not None}
            for kind in kinds:
                some = grads if len(kinds) == 1 else [g if g is not None and g.dtype == kind else None for g in grads]
                adamw_step(ps, some, m, v, steps, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], masters=masters, scales=scales,
                           max_norm=None if norm is None else self.max_norm,
                           norm=None if norm is None else norm.to(ps[0].device), seed=self.seed)
            if masters is not None:
                marks[:] = _marks(ps)
        return loss

    def load_state_dict(self, state_dict):
        """States keep the types that they were saved with (torch would cast them to the parameters')."""
        if any(("scales" in state) != (self.state_bits == 8) for state in state_dict["state"].values()):
            raise ValueError(f"the saved states are not those of {self.state_bits} bits")
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            if i not in state_dict["state"]:
                continue
            self.state[p] = {k: t.detach().to(p.device, copy=True) for k, t in state_dict["state"][i].items()}
        self._make_lists(self.state)  # so that the next step may be captured


def reference(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01):
    """The new (params, exp_avgs, exp_avg_sqs) of fp32 states, by elementary operations."""
    out = []
    for p, g, m, v, t in zip(params, grads, exp_avgs, exp_avg_sqs, (steps + 1).double()):
        m = betas[0] * m + (1 - betas[0]) * g.float()
        v = betas[1] * v + (1 - betas[1]) * g.float().square()
        rate, root = (lr / (1 - betas[0] ** t)).float(), (1 - betas[1] ** t).sqrt().float()
        out.append(((p.float() * (1 - lr * weight_decay) - rate * m / (v.sqrt() / root + eps)).to(p.dtype), m, v))
    return tuple(map(list, zip(*out)))


def selftest():
    from _harness import compare, time_ab, significance, versions  # noqa: PLC0415

    shapes = [(32128, 1024)] + 4 * [(1024,), (1024, 1024), (2048, 1024), (5632, 1024), (1024, 2816)]
    params = [torch.randn(s, device="cuda") for s in shapes]
    grads = [1e-2 * torch.randn(s, device="cuda") for s in shapes]
    m, v = [0.3 * g for g in grads], [g.square() for g in grads]
    steps = torch.full((len(shapes),), 10, dtype=torch.int32, device="cuda")
    hyper = {"lr": 1e-3}
    want = reference(params, grads, m, v, steps, **hyper)
    own = [[t.clone() for t in ts] for ts in (params, m, v)]
    adamw_step(own[0], grads, own[1], own[2], steps.clone(), **hyper)
    checks = compare(want, want, own)
    t = time_ab({"reference": [lambda: reference(params, grads, m, v, steps, **hyper)],
                 "kernel": [lambda: adamw_step(params, grads, m, v, steps, **hyper)]}, rounds=3, graph=False)
    us = {name: round(x["device_ms"] * 1e3, 1) for name, x in t.items()}
    return {"pass": checks["pass"], "checks": checks, **versions(), "reference_us": us["reference"],
            "kernel_us": us["kernel"], "speedup": round(us["reference"] / us["kernel"], 2),
            "significance": significance(t["reference"], t["kernel"]),
            "compiled": {"error": "an optimizer's step is not compiled"}}


if __name__ == "__main__":
    print(selftest())
