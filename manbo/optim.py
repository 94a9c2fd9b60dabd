"""Optimisers on the B200 step kernels: Adan (mirrors manbo/optim.py:10-190)
and AdamW over all parameters at once.

``Adan`` has the same constructor, validation, state (``exp_avg``, ``exp_avg_sq``,
``exp_avg_diff``, ``neg_pre_grad`` per parameter), ``restart_opt`` and global
gradient-norm clipping as the reference; every parameter's update is one
``cs_adan_step`` launch.  Like the reference, clipping (max_grad_norm > 0)
reads the norm on the host, once per step.

``AdamW`` (no counterpart in the reference) moves several hundred parameters a
launch, with its moments in 32 bits or in 8 (manbo/ops/adamw.py), clips by the
global gradient norm without reading it back, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import collections
import math

import torch
from torch.optim.optimizer import Optimizer

from repo_b200 import _ext

from .ops.adamw import ADAMW8_BLOCK, adamw8_moments, adamw8_state, grad_norm
from .ops.optim import adan_step_from_grad_kernel

DEFAULT_TILELANG_THREADS = 256
_STATE_KEYS = ("exp_avg", "exp_avg_sq", "exp_avg_diff", "neg_pre_grad")


class Adan(Optimizer):
    """Adan (adaptive Nesterov momentum) with decoupled or proximal weight decay."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.98, 0.92, 0.99), eps: float = 1e-8,
                 weight_decay: float = 0.0, max_grad_norm: float = 0.0, no_prox: bool = False,
                 tilelang_threads: int = DEFAULT_TILELANG_THREADS):
        if not 0.0 <= max_grad_norm:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i in range(3):
            if not 0.0 <= betas[i] < 1.0:
                raise ValueError(f"Invalid beta parameter at index {i}: {betas[i]}")
        if tilelang_threads <= 0:
            raise ValueError(f"Invalid tilelang_threads: {tilelang_threads}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      max_grad_norm=max_grad_norm, no_prox=no_prox,
                                      tilelang_threads=tilelang_threads))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("no_prox", False)
            group.setdefault("tilelang_threads", DEFAULT_TILELANG_THREADS)

    @torch.no_grad()
    def restart_opt(self):
        """Zero the step count and every moment (the reference's restart)."""
        for group in self.param_groups:
            group["step"] = 0
            for p in group["params"]:
                if p.requires_grad:
                    st = self.state[p]
                    for k in _STATE_KEYS:
                        st[k] = torch.zeros_like(p)

    def _clip_factor(self) -> float:
        max_norm = self.defaults["max_grad_norm"]
        if max_norm <= 0:
            return 1.0
        dev = self.param_groups[0]["params"][0].device
        sq = torch.zeros(1, device=dev)
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    sq.add_(p.grad.pow(2).sum())
        eps = self.param_groups[0]["eps"]
        factor = torch.clamp(torch.tensor(max_norm, device=dev) / (torch.sqrt(sq) + eps), max=1.0)
        return float(factor.item())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        clip = self._clip_factor()
        for group in self.param_groups:
            b1, b2, b3 = group["betas"]
            group["step"] = group.get("step", 0) + 1
            t = int(group["step"])
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            no_prox = bool(group["no_prox"])
            key = (int(group["tilelang_threads"]), no_prox)
            if group.get("_b200_kernel_key") != key:
                group["_b200_kernel"] = adan_step_from_grad_kernel(threads=key[0], no_prox=no_prox)
                group["_b200_kernel_key"] = key
            kernel = group["_b200_kernel"]
            bc1, bc2, bc3_sqrt = 1.0 - b1 ** t, 1.0 - b2 ** t, math.sqrt(1.0 - b3 ** t)
            for p in params:
                if p.dtype != torch.float32:
                    raise ValueError("TileLang Adan currently expects float32 params")
                if not p.is_contiguous():
                    raise ValueError("TileLang Adan expects contiguous params")
                st = self.state[p]
                if not st:
                    for k in _STATE_KEYS:
                        st[k] = torch.zeros_like(p)
                moments = [st[k] for k in _STATE_KEYS]
                if any(m.dtype != torch.float32 or not m.is_contiguous() for m in moments):
                    raise ValueError("TileLang Adan expects contiguous float32 states")
                g = p.grad
                if g.dtype != torch.float32 or g.device != p.device or not g.is_contiguous():
                    buf = st.get("_grad_buf")
                    if buf is None or buf.shape != p.shape:
                        buf = torch.empty_like(p)
                        st["_grad_buf"] = buf
                    buf.copy_(g)
                    g = buf
                n = p.numel()
                kernel(p.view(n), g.view(n), *(m.view(n) for m in moments), t, b1, b2, b3, bc1,
                       bc2, bc3_sqrt, group["lr"], group["weight_decay"], group["eps"], clip)
        return loss


_ADAMW_MAX_GROUPS = 16  # hyper-parameter groups of one launch


def _order(t):
    """A tensor's strides where they matter: of sizes above 1."""
    return [s for n, s in zip(t.shape, t.stride()) if n > 1]


class AdamW(Optimizer):
    """Adam with decoupled weight decay, several hundred parameters a launch.

    A launch holds one device, ``state_bits``, ``seed`` and ``capturable``, and up to
    16 pairs of group and step number.

    ``state_bits`` 32 keeps ``exp_avg`` and ``exp_avg_sq`` as float32 in the
    parameter's layout, 8 as one byte an element with a scale byte for each 256
    elements (see ``manbo.ops.adamw8_step``; ``seed`` feeds its rounding).
    ``max_grad_norm`` > 0 clips by the global norm of all gradients, which stays
    on the device (``grad_norm`` holds the last one); it is the same in every group,
    so that it is saved and loaded with them.  Parameters are float32,
    bfloat16 or float16, non-overlapping and dense.

    Steps are counted per parameter, those at which it has a gradient.  With
    ``capturable`` the counts live on the device, so that a captured step counts on
    every replay; a group's ``lr`` may then be a float32 device scalar that a
    schedule writes to.  Take one step before the capture, so that the state exists.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, max_grad_norm: float = 0.0, state_bits: int = 32,
                 capturable: bool = False, seed: int = 0):
        if not 0.0 <= max_grad_norm:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        if isinstance(lr, torch.Tensor):
            if not capturable:
                raise ValueError("lr as a tensor needs capturable=True")
        elif not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i in range(2):
            if not 0.0 <= betas[i] < 1.0:
                raise ValueError(f"Invalid beta parameter at index {i}: {betas[i]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      max_grad_norm=max_grad_norm, state_bits=state_bits,
                                      capturable=capturable, seed=seed))
        self.grad_norm = None

    def __setstate__(self, state):
        if self.__dict__.get("_loaded") is not None:  # of a load
            state = {**state, "state": self._loaded}
        super().__setstate__(state)
        self.__dict__.setdefault("grad_norm", None)
        own = set()  # an optimiser stored by an earlier version shares counters
        for st in self.state.values():
            step = st.get("step")
            if isinstance(step, torch.Tensor):
                if id(step) in own:
                    st["step"] = step.clone()
                own.add(id(st["step"]))
        for group in self.param_groups:
            for key, value in self.defaults.items():
                group.setdefault(key, value)
        # one value for all groups, those that are added later among them
        if len({group["max_grad_norm"] for group in self.param_groups}) == 1:
            self.defaults["max_grad_norm"] = self.param_groups[0]["max_grad_norm"]

    def _new_state(self, p, group, capturing):
        if capturing:
            raise RuntimeError("AdamW: take one step before capturing, so that the state exists")
        st = {}
        if group["state_bits"] == 8:
            (st["exp_avg"], st["exp_avg_scales"], st["exp_avg_sq"],
             st["exp_avg_sq_scales"]) = adamw8_state(p)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                st[k] = torch.zeros_like(p, dtype=torch.float32,
                                         memory_format=torch.preserve_format)
        st["step"] = (torch.zeros((), dtype=torch.int64, device=p.device) if group["capturable"]
                      else 0)
        return st

    def _plan(self):
        """{(device index, state_bits, seed, capturable): [(group, step, parameters,
        gradients, states)]} of this step, the parameters of an entry at the same step
        (counted on the device, step is None and they may be at any)."""
        plan = {}
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for group in self.param_groups:
            cohorts = {}
            eight, capturable = group["state_bits"] == 8, bool(group["capturable"])
            if capturing and not capturable:
                raise RuntimeError("AdamW: a captured step needs capturable=True")
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                device = p.get_device()
                if device < 0:
                    raise ValueError("AdamW parameters must be CUDA tensors")
                st = self.state[p]
                if not st:
                    st.update(self._new_state(p, group, capturing))
                if ("exp_avg_scales" in st) != eight:
                    raise ValueError(f"AdamW state is not of state_bits={group['state_bits']}")
                step = st["step"]
                if isinstance(step, torch.Tensor) != capturable:
                    raise ValueError("AdamW state was made with another value of capturable")
                if capturable:
                    step = None
                key = (device, step)
                cohort = cohorts.get(key)
                if cohort is None:
                    cohort = cohorts[key] = (group, step, [], [], [])
                    launch = (device, group["state_bits"], group["seed"] if eight else 0,
                              capturable)
                    plan.setdefault(launch, []).append(cohort)
                cohort[2].append(p)
                cohort[3].append(grad)
                cohort[4].append(st)
        return plan

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        plan = self._plan()
        if not plan:
            return loss
        norm = scale = None
        max_norm = self.param_groups[0]["max_grad_norm"]
        if any(group["max_grad_norm"] != max_norm for group in self.param_groups):
            raise ValueError("AdamW: max_grad_norm must be the same in every group")
        if max_norm != 0:
            if len({device for device, *_ in plan}) > 1:
                raise ValueError("max_grad_norm needs every parameter on one device")
            grads = [g for parts in plan.values() for part in parts for g in part[3]]
            norm, scale = grad_norm(grads, max_norm=max_norm)
        calls, counted = [], []
        places = {}  # 8-bit parameters already stepped with a seed, which draw other bits
        for (_, bits, seed, capturable), parts in plan.items():
            for at in range(0, len(parts), _ADAMW_MAX_GROUPS):
                some = parts[at:at + _ADAMW_MAX_GROUPS]
                groups = [(len(ps), g["lr"], g["betas"][0], g["betas"][1], g["eps"],
                           g["weight_decay"], 1 if capturable else step + 1)
                          for g, step, ps, _, _ in some]
                if len(some) == 1:
                    params, grads, states = some[0][2:]
                else:
                    params, grads, states = ([x for part in some for x in part[k]]
                                             for k in (2, 3, 4))
                m = [s["exp_avg"] for s in states]
                v = [s["exp_avg_sq"] for s in states]
                steps = [s["step"] for s in states] if capturable else None
                if bits == 8:
                    ms = [s["exp_avg_scales"] for s in states]
                    vs = [s["exp_avg_sq_scales"] for s in states]
                    seed &= 0xFFFFFFFF
                    first = places.get(seed, 0)
                    places[seed] = first + len(params)
                    calls.append((params, grads, m, v, groups, steps, ms, vs, seed, first))
                else:
                    calls.append((params, grads, m, v, groups, steps))
                if not capturable:
                    counted += some
        _ext.load().adamw_steps(calls, scale)  # all are checked before one runs
        if norm is not None:
            self.grad_norm = norm
        for _, step, _, _, states in counted:
            for st in states:
                st["step"] = step + 1
        return loss

    @torch.no_grad()
    def moments(self, p):
        """(exp_avg, exp_avg_sq) of a parameter as new float32 tensors."""
        st = self.state.get(p)
        if not st:
            raise ValueError("the parameter has no state yet: it has not taken a step")
        if "exp_avg_scales" not in st:
            return st["exp_avg"].clone(), st["exp_avg_sq"].clone()
        m, v = adamw8_moments([st["exp_avg"]], [st["exp_avg_scales"]], [st["exp_avg_sq"]],
                              [st["exp_avg_sq_scales"]])
        return m[0], v[0]

    @torch.no_grad()
    def restart_opt(self):
        """Zero every moment and step count in place, so that a step captured before
        goes on from there.  A state made with other ``state_bits`` or ``capturable``
        than its group has now is dropped."""
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p)
                if not st:
                    continue
                if (("exp_avg_scales" in st) != (group["state_bits"] == 8)
                        or isinstance(st["step"], torch.Tensor) != bool(group["capturable"])):
                    del self.state[p]
                    continue
                for x in st.values():
                    if isinstance(x, torch.Tensor):
                        x.zero_()
                if not group["capturable"]:
                    st["step"] = 0

    def load_state_dict(self, state_dict):
        """As the base class, except that moments keep their own types (the base
        class casts them to the parameter's) and are copies of the given ones.
        States of ``torch.optim.AdamW`` load too, into groups of 32-bit moments;
        what this class does not compute (``maximize``, ``amsgrad``, Adam's coupled
        decay) and moments of other ``state_bits`` than the group's are refused.  A
        refused load changes nothing.  A step captured before a load has to be
        captured again: its moments, counts and hyper-parameters are the old ones."""
        # behind the user's own hooks, so that it sees what they return
        hook = self.register_load_state_dict_pre_hook(AdamW._take_state)
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
            self._loaded = None

    def _take_state(self, state_dict):
        """Pre-hook of a load: keeps the parameters' new states for ``__setstate__`` and
        leaves none for the base class to cast."""
        saved = state_dict["param_groups"]
        for group in saved:
            if (group.get("maximize") or group.get("amsgrad")
                    or not group.get("decoupled_weight_decay", True)):
                raise ValueError("AdamW does not support maximize, amsgrad or coupled weight decay")
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            return None  # which the base class refuses
        loaded = collections.defaultdict(dict)
        for group, own in zip(saved, self.param_groups):
            bits, capturable = (group.get(k, self.defaults[k])
                                for k in ("state_bits", "capturable"))
            for i, p in zip(group["params"], own["params"]):
                if i in state_dict["state"]:
                    loaded[p] = self._own_state(p, state_dict["state"][i], bits,
                                                capturable)
        rates = {}  # groups that shared a tensor go on sharing one
        groups = []
        for group, own in zip(saved, self.param_groups):
            lr = group.get("lr")
            if isinstance(lr, torch.Tensor):
                if not group.get("capturable", self.defaults["capturable"]):
                    lr = float(lr)
                elif own["params"]:
                    device = own["params"][0].device
                    lr = rates.setdefault((id(lr), device),
                                          lr.detach().to(device, torch.float32, copy=True))
                group = {**group, "lr": lr}
            groups.append(group)
        self._loaded = loaded
        return {**state_dict, "state": {}, "param_groups": groups}

    @staticmethod
    def _own_state(p, state, bits, capturable):
        """Copies of a parameter's saved moments and step count, on its device, as a
        step takes them: 32-bit moments in float32 (torch keeps them in the
        parameter's type), 8-bit ones as they are."""
        if not state:
            return {}
        names = ("exp_avg", "exp_avg_sq")
        scales = ("exp_avg_scales", "exp_avg_sq_scales") if bits == 8 else ()
        missing = [k for k in (*names, *scales, "step") if k not in state]
        if not all(state[k].dtype == torch.uint8 if bits == 8 else state[k].is_floating_point()
                   for k in names if k in state):
            raise ValueError(f"AdamW state is not of state_bits={bits}")
        if missing:
            raise ValueError(f"AdamW state lacks {', '.join(missing)}")
        blocks = -(-p.numel() // ADAMW8_BLOCK)
        st = {}
        for k, x in state.items():
            if k in names:
                if x.shape != p.shape:
                    raise ValueError(f"{k} must have its parameter's shape")
                if bits == 8 and _order(x) != _order(p):
                    raise ValueError("8-bit moments need the strides of the parameter they were "
                                     "saved with (their blocks follow its storage)")
                kind = torch.uint8 if bits == 8 else torch.float32
                st[k] = torch.empty_like(p, dtype=kind).copy_(x)
            elif k in scales:
                if x.dtype != torch.uint8 or x.numel() != blocks:
                    raise ValueError(f"{k} must be {blocks} uint8 scales")
                st[k] = torch.empty(blocks, dtype=torch.uint8, device=p.device).copy_(x.view(-1))
            elif k == "step":
                st[k] = (torch.as_tensor(x).reshape(()).to(p.device, torch.int64, copy=True)
                         if capturable else int(x))
            else:
                st[k] = x.to(p.device, copy=True) if isinstance(x, torch.Tensor) else x
        return st


__all__ = ["Adan", "AdamW"]
