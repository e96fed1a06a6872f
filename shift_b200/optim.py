"""AdamW over many tensors at once, with moments in 32 or in 8 bits.

``AdamWMany`` updates lists of tensors with one kernel launch per 320 of them
(``csrc/adamw_many.cu``), in place.  It stands beside
``ops.functional.adamw_step``, which updates one flat buffer of a fixed layout
from one state generation into the next: use that one where the parameters
live in ``parallel.flat.FlatParams``, and this one for parameters that are
tensors of their own (an ordinary module, a model that is not ours).

8-bit moments take 2 + 1/64 bytes per parameter instead of 8.  ``exp_avg`` and
the square root of ``exp_avg_sq`` are e4m3 codes with one power-of-two scale
per 128 consecutive elements, rounded stochastically from ``seed``.  The codes
span 18 binades: an element whose gradients are smaller than 4e-6 of its
block's largest is updated as if its root were that large, so by less than with
32-bit moments.
"""
from __future__ import annotations

import math
import operator
from typing import NamedTuple

import torch

from .ops import reference as ref
from .ops._ext import ext

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class State8(NamedTuple):
    """One moment of a tensor of n elements: ``code`` float8_e4m3fn [n], ``scale`` float8_e8m0fnu [ceil(n / 128)].
    For ``exp_avg_sq`` the codes hold its square root."""
    code: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def zeros(cls, param: torch.Tensor) -> "State8":
        n = param.numel()
        return cls(torch.zeros(n, dtype=torch.uint8, device=param.device).view(torch.float8_e4m3fn),
                   torch.zeros(-(-n // 128), dtype=torch.uint8, device=param.device).view(torch.float8_e8m0fnu))

    def values(self) -> torch.Tensor:
        """fp32 [n]; of ``exp_avg_sq`` its square root."""
        return ref.moment_decode(self.code, self.scale)


def _fail(cond: bool, text: str):
    if not cond:
        raise ValueError("AdamWMany: " + text)


class AdamWMany:
    """``params``: contiguous fp32 / bf16 / fp16 tensors on one device, updated in place.
    ``exp_avg`` / ``exp_avg_sq``: per parameter an fp32 tensor, or a ``State8``
    (one kind for all).  ``masters``: optional fp32 tensors that hold the exact
    weights; a parameter then is their rounded copy.  Without them a bf16 or
    fp16 parameter is itself the weight, and each step rounds it."""

    def __init__(self, params, exp_avg, exp_avg_sq, masters=None):
        self.params, self.exp_avg, self.exp_avg_sq = list(params), list(exp_avg), list(exp_avg_sq)
        self.masters = None if masters is None else list(masters)
        n = len(self.params)
        _fail(n <= 0x7FFF, f"{n} tensors, at most {0x7FFF}")
        _fail(len(self.exp_avg) == n and len(self.exp_avg_sq) == n
              and (self.masters is None or len(self.masters) == n), "lists of different lengths")
        self.eight = n > 0 and isinstance(self.exp_avg[0], State8)
        self.device = self.params[0].device if n > 0 else None
        self._check()
        own = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size())
                     for p, *state in zip(self.params, *self._states()) for x in (p, *state) if x.numel())
        _fail(all(end <= start for (_, end), (start, _) in zip(own, own[1:])), "a tensor is there twice, or two share memory")
        self._plan = None
        if n > 0 and self.params[0].is_cuda:
            lists = self._states()
            m, ms, v, vs = lists[:4] if self.eight else (lists[0], [], lists[1], [])
            self._plan = ext().adamw_many_plan(self.params, self.masters or [], m, ms, v, vs)

    def _check(self):
        """Types, sizes and places of all tensors; a step looks again (the extension's itself on the GPU), since a tensor
        can be given other memory."""
        for t, p in enumerate(self.params):
            _fail(p.dtype in _FLOATS, f"parameter {t} is {p.dtype}")
            same = [p]
            for s in (self.exp_avg[t], self.exp_avg_sq[t]):
                _fail(isinstance(s, State8) == self.eight, "moments in 8 bits and in 32 bits are mixed")
                if self.eight:
                    _fail(s.code.dtype == torch.float8_e4m3fn and s.code.numel() == p.numel(),
                          f"tensor {t}: {p.numel()} codes of float8_e4m3fn are expected")
                    _fail(s.scale.dtype == torch.float8_e8m0fnu and s.scale.numel() == -(-p.numel() // 128),
                          f"tensor {t}: {-(-p.numel() // 128)} scales of float8_e8m0fnu are expected")
                    same += [s.code, s.scale]
                else:
                    _fail(s.dtype == torch.float32 and s.numel() == p.numel(),
                          f"tensor {t}: fp32 moments of {p.numel()} elements are expected")
                    same.append(s)
            if self.masters is not None:
                w = self.masters[t]
                _fail(w.dtype == torch.float32 and w.numel() == p.numel(),
                      f"tensor {t}: an fp32 master of {p.numel()} elements is expected")
                same.append(w)
            _fail(torch.is_inference_mode_enabled() or not any(x.is_inference() for x in same),
                  f"tensor {t} or its state was made in inference mode")
            _fail(all(x.is_contiguous() for x in same), f"tensor {t} or its state is not contiguous")
            _fail(all(x.device == self.device for x in same), f"tensor {t} or its state is on another device")

    def check(self, grads):
        """Raises what ``step`` would of these gradients, and of the tensors as they are by now."""
        if self._plan is not None:
            ext().adamw_many_check(self._plan, grads)
            return
        if len(grads) != len(self.params):
            raise ValueError(f"AdamWMany: {len(grads)} gradients for {len(self.params)} parameters")
        self._check()
        for t, (g, p) in enumerate(zip(grads, self.params)):
            if g.dtype not in _FLOATS or g.numel() != p.numel() or not g.is_contiguous() or g.device != self.device:
                raise ValueError(f"AdamWMany: gradient {t}: contiguous, {p.numel()} elements, fp32 / bf16 / fp16, on {self.device}")

    def _states(self):
        """The lists of tensors that a step writes beside the parameters."""
        lists = [self.exp_avg, self.exp_avg_sq]
        if self.eight:
            lists = [[s[i] for s in x] for x in lists for i in (0, 1)]
        return lists + ([] if self.masters is None else [self.masters])

    def step(self, grads, lr: float = 1.0e-4, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1.0e-8,
             wd: float = 0.01, step: int = 1, grad_scale: float = 1.0, seed: int | None = None, step_dev=None,
             skip=None, nonfinite=None):
        """One update.  ``grads``: contiguous tensors like the parameters, fp32, bf16 or fp16.

        ``step`` counts from 1.  ``seed`` (8-bit moments) chooses the random
        bits; by default it is ``step``.  ``step_dev``: int32 [>= 4] on the
        device with seed, and lr, 1 - beta1^t, sqrt(1 - beta2^t) as float
        bits, which replace the arguments (a replayed graph's step;
        ``engine.StepBlock`` writes that layout).  ``skip``: int32 on the
        device; where it is not zero nothing changes.  ``nonfinite``: int32
        flag, set where a scaled gradient is not finite.  ``skip`` is read
        while ``nonfinite`` is written: not the same word."""
        if step < 1:
            raise ValueError(f"AdamWMany: step {step}: counted from 1")
        seed = (step if seed is None else seed) & 0xFFFFFFFF
        if self._plan is not None:
            ext().adamw_many(self._plan, grads if isinstance(grads, list) else list(grads), lr, beta1, beta2, eps, wd,
                             step, grad_scale, seed, step_dev, skip, nonfinite)
            return
        grads = list(grads)
        self.check(grads)
        dev = self.device
        for name, x, least in (("step_dev", step_dev, 4), ("skip", skip, 1), ("nonfinite", nonfinite, 1)):
            if x is not None and (x.dtype != torch.int32 or x.numel() < least or x.device != dev):
                raise ValueError(f"AdamWMany: {name}: int32 [{least}] on {dev}")
        if nonfinite is not None and any(x is not None and x.data_ptr() <= nonfinite.data_ptr() < x.data_ptr() + 4 * n
                                         for x, n in ((skip, 1), (step_dev, 4))):
            raise ValueError("AdamWMany: nonfinite is a word that the step reads")
        self._cpu_step(grads, lr, beta1, beta2, eps, wd, step, grad_scale, seed, step_dev, skip, nonfinite)

    def _cpu_step(self, grads, lr, beta1, beta2, eps, wd, step, grad_scale, seed, step_dev, skip, nonfinite):
        if skip is not None and int(skip.view(-1)[0]) != 0:
            return
        c1, c2 = 1.0 - beta1 ** step, math.sqrt(1.0 - beta2 ** step)
        if step_dev is not None:
            seed = int(step_dev.view(-1)[0])
            lr, c1, c2 = step_dev.view(-1)[1:4].view(torch.float32).tolist()
        for t, (p, g) in enumerate(zip(self.params, grads)):
            g = g.detach().reshape(-1).float() * grad_scale
            if nonfinite is not None and not bool(torch.isfinite(g).all()):
                nonfinite.view(-1)[0] = 1
            w = (p if self.masters is None else self.masters[t]).detach().view(-1)
            m, v = self.exp_avg[t], self.exp_avg_sq[t]
            m32 = m.values() if self.eight else m.view(-1)
            v32 = v.values().square() if self.eight else v.view(-1)
            m32 = m32 + (g - m32) * (1.0 - beta1)
            v32 = v32 * beta2 + (1.0 - beta2) * g * g
            r = v32.double().sqrt().float()            # rounded correctly: fp32's own root here is a bit off at times
            new = w.float() * (1.0 - lr * wd) - (lr / c1) * (m32 / (r / c2 + eps))
            if self.eight:
                u = ref.moment_draws(g.numel(), seed, t)
                for s, x, bits, root in ((m, m32, u & 0xFFFF, False), (v, r, u >> 16, True)):
                    code, scale = ref.moment_encode(x, bits, root)
                    s.code.view(-1).copy_(code)
                    s.scale.copy_(scale)
            else:
                m.view(-1).copy_(m32)
                v.view(-1).copy_(v32)
            w.copy_(new)
            if self.masters is not None:
                p.detach().view(-1).copy_(new)


class AdamW(torch.optim.Optimizer):
    """``AdamWMany`` as a ``torch.optim`` optimizer: a script's ``torch.optim.AdamW`` with its state in 8 bits
    (``state_bits=8``: 2 + 1/64 bytes per parameter, where 32 bits take 8) or 32, updated by one kernel per group.

    ``master_weights`` keeps fp32 weights beside bf16 or fp16 parameters.  Under ``ft.transparent`` it is adopted like
    any other optimizer: its state is part of ``state_dict`` and heals with it.  State tensors are made at a
    parameter's first gradient; a parameter without a gradient is left alone in that step.  State is row-major whatever
    a parameter's layout; a parameter that is not (channels_last, transposed) is copied to that order and back."""

    def __init__(self, params, lr: float = 1.0e-3, betas=(0.9, 0.999), eps: float = 1.0e-8, weight_decay: float = 1.0e-2,
                 state_bits: int = 8, master_weights: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state in 8 or 32 bits, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights))
        self._lists = None                             # what was handed over, and what that hangs on
        self._packed: dict = {}                        # row-major copies of parameters of another layout

    def __setstate__(self, state):
        super().__setstate__(state)
        self._lists, self._packed = None, {}           # a copy or an unpickled optimizer has tensors of its own

    def _init_state(self, p, group):
        st = self.state[p]
        st["step"] = 0
        for name in ("exp_avg", "exp_avg_sq"):
            if group["state_bits"] == 8:
                code, scale = State8.zeros(p)
                # as bytes: what copies or ships a state dict need not know the 8-bit types
                st[name], st[name + "_scale"] = code.view(torch.uint8), scale.view(torch.uint8)
            else:
                st[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"]:
            st["master"] = p.detach().to(torch.float32, memory_format=torch.contiguous_format, copy=True)

    def _flat(self, p):
        return p if p.is_contiguous() else self._packed[p]

    def _moment(self, p, name, group):
        st = self.state[p]
        if group["state_bits"] == 8:
            return State8(st[name].view(torch.float8_e4m3fn), st[name + "_scale"].view(torch.float8_e8m0fnu))
        return st[name]

    def load_state_dict(self, state_dict):
        """Takes what this class saved, and what ``torch.optim.AdamW`` did: the group then keeps this optimizer's
        ``state_bits`` and ``master_weights``, moments are rounded to nearest and master weights start from the
        parameters.  Saved state of another rule (``amsgrad``, ``maximize``, coupled weight decay) is refused."""
        kinds = [{name: g[name] for name in ("state_bits", "master_weights")} for g in self.param_groups]
        saved, groups = state_dict["state"], state_dict["param_groups"]
        for g in groups:
            other = [name for name in ("amsgrad", "maximize") if g.get(name)]
            if g.get("weight_decay") and not g.get("decoupled_weight_decay", True):
                other.append("coupled weight decay")
            other += ["no " + name for name in ("lr", "betas", "eps", "weight_decay") if name not in g]
            if other:
                raise ValueError(f"AdamW: a saved state with {', '.join(other)}")
            for i in () if "state_bits" in g else g["params"]:
                if i in saved and not {"step", "exp_avg", "exp_avg_sq"} <= saved[i].keys():
                    raise ValueError(f"AdamW: saved state with {sorted(saved[i])}, not step, exp_avg and exp_avg_sq")
        super().load_state_dict(state_dict)
        for mine, theirs, kind in zip(self.param_groups, groups, kinds):
            mine.update({name: x for name, x in kind.items() if name not in theirs})
            for i, p in zip(theirs["params"], mine["params"]):
                if i not in saved:
                    continue
                if "state_bits" not in theirs:
                    self._take(p, mine, saved[i])
                    continue
                # the base class casts floating-point and byte states to the parameter's type: put back what was saved
                for name, x in saved[i].items():
                    self.state[p][name] = x.to(p.device, copy=True) if isinstance(x, torch.Tensor) else x
        self._lists = None

    def _take(self, p, group, saved):
        """State of ``p`` from that of torch.optim.AdamW: moments of the parameter's shape in any floating type."""
        self.state.pop(p, None)
        self._init_state(p, group)
        st = self.state[p]
        st["step"] = int(saved["step"])
        m, v = (saved[name].to(p.device, torch.float32).contiguous() for name in ("exp_avg", "exp_avg_sq"))
        if group["state_bits"] == 32:
            st["exp_avg"].copy_(m)
            st["exp_avg_sq"].copy_(v)
            return
        half = torch.full((p.numel(),), 0x8000, device=p.device)
        for name, x, root in (("exp_avg", m, False), ("exp_avg_sq", v.sqrt(), True)):
            code, scale = ref.moment_encode(x.view(-1), half, root)
            st[name].copy_(code.view(torch.uint8))
            st[name + "_scale"].copy_(scale.view(torch.uint8))

    @torch.no_grad()
    def step(self, closure=None):
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            # a replay would repeat this step's bias corrections and random bits and leave the counts behind
            raise RuntimeError("AdamW: step() cannot be captured into a graph; AdamWMany.step takes step_dev for that")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        live = [[(p, g) for p in group["params"] if (g := p.grad) is not None] for group in self.param_groups]
        made = []
        try:                                           # all that may be refused comes before the first update
            jobs = self._jobs(live, made)
        except Exception:
            for p in made:
                del self.state[p]
            self._lists = None
            raise
        for (k, ps, states, many, _, place), t, grads in jobs:
            group = self.param_groups[k]
            moved = [p for p in ps if p in self._packed] if self._packed else ()
            for p in moved:
                self._packed[p].copy_(p)
            beta1, beta2 = group["betas"]
            # the random bits hang on the seed and on a tensor's number in its list: each list has a seed of its own
            many.step(grads, lr=float(group["lr"]), beta1=beta1, beta2=beta2, eps=group["eps"],
                      wd=group["weight_decay"], step=t, seed=t + 0x9E3779B1 * place)
            for p in moved:
                p.copy_(self._packed[p])
            for st in states:
                st["step"] = t
        return loss

    def _used(self, live):
        """What the lists handed over hang on: objects, and the addresses of state tensors (``None`` where a state is
        not as this class makes it).  State can be cleared, or given other tensors or other memory."""
        objects, places = [*self.state, *self.state.values()], []
        for group, pairs in zip(self.param_groups, live):
            objects += (group["state_bits"], group["master_weights"], None)
            for p, _ in pairs:
                objects += (p, p.is_contiguous())
        for st in self.state.values():
            if not isinstance(st, dict) or next(iter(st), None) != "step":
                return objects, None
            tensors = [x for x in st.values() if x.__class__ is not int]
            objects += tensors
            try:
                places += [x.data_ptr() for x in tensors]
            except AttributeError:
                return objects, None
        return objects, places

    def _jobs(self, live, made):
        """(list handed over, step, gradients) of every update; parameters with new state are added to ``made``."""
        for p, g in (pair for pairs in live for pair in pairs):
            if g.layout is not torch.strided:
                raise ValueError(f"AdamW: gradient of layout {g.layout} of a parameter {tuple(p.shape)}: dense ones only")
        objects, places = self._used(live)
        held = self._lists
        if (held is None or places is None or places != held[1] or len(objects) != len(held[0])
                or not all(map(operator.is_, objects, held[0]))
                or any(st["step"] != states[0]["step"] for _, _, states, *_ in held[2] for st in states)):
            lists = self._hand_over(live, made)
            held = self._lists = (*self._used(live), lists)
        jobs = []
        for one in held[2]:
            k, ps, states, many, index, _ = one
            grads = [live[k][i][1].contiguous() for i in index]
            for p in ps if self._packed else ():
                if p in self._packed and self._packed[p].shape != p.shape:
                    raise ValueError(f"AdamW: a parameter has changed its shape to {tuple(p.shape)}")
            many.check(grads)
            jobs.append((one, int(states[0]["step"]) + 1, grads))
        return jobs

    def _hand_over(self, live, made):
        """The lists that are updated by one call each: (group, parameters, their state, AdamWMany, their places among
        the group's live ones, the first one's number in the optimizer)."""
        place = {p: i for i, p in enumerate(p for group in self.param_groups for p in group["params"])}
        lists = []
        for k, (group, pairs) in enumerate(zip(self.param_groups, live)):
            by_step: dict = {}
            for i, (p, _) in enumerate(pairs):
                if "step" not in self.state[p]:
                    made.append(p)
                    self._init_state(p, group)
                held = self._packed.get(p)
                if p.is_contiguous():
                    self._packed.pop(p, None)
                elif held is None or (held.shape, held.dtype, held.device) != (p.shape, p.dtype, p.device):
                    self._packed[p] = torch.empty(p.shape, dtype=p.dtype, device=p.device)
                by_step.setdefault((int(self.state[p]["step"]), p.device), []).append((i, p))
            for some in by_step.values():
                index, ps = zip(*some)
                many = AdamWMany([self._flat(p) for p in ps], [self._moment(p, "exp_avg", group) for p in ps],
                                 [self._moment(p, "exp_avg_sq", group) for p in ps],
                                 [self.state[p]["master"] for p in ps] if group["master_weights"] else None)
                lists.append((k, ps, [self.state[p] for p in ps], many, index, place[ps[0]]))
        return lists
