"""AdamW over many tensors at once, with states in 32 or in 8 bits, on the HIP kernels.

`AdamW` is torch.optim.AdamW's update (decoupled weight decay) in one launch for
48 tensors, whatever their sizes:

    m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
    p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)

in float32. A state of 32 bits holds m and v ("exp_avg", "exp_avg_sq"). One of 8
bits holds m and r = sqrt(v) as e4m3 numbers ("exp_avg", "exp_root") times a
float32 step for each 256 numbers in a row of the tensor ("exp_avg_scale",
"exp_root_scale": the block's largest / 448): 2 bytes a number instead of 8. The
rounding is dithered over the steps, so that small changes are kept on average,
and the same on every run. Blocks whose largest number is below 2^-110 are held
as zeros.

16-bit weights lose updates below half their spacing; `master_weights=True` keeps a
float32 copy ("master") that the update is made to, the weight its rounding: who
changes such a weight otherwise changes its master too, or the next step undoes it.

Steps are counted on the device, one counter a tensor, and nothing synchronises: a
step can be captured into a graph (after a first one, or a loaded state, has made
the states) and counts on with every replay. lr may be a float32 number on the
device, read when the step runs.

Supported: float32, bfloat16 and float16 parameters on the GPU, contiguous, with
dense gradients of their type; anything else raises NotImplementedError. There is
no CPU path: CPU tensors raise.
"""
from __future__ import annotations

import itertools
import math
import operator

import numpy as np
import torch
from torch import Tensor

from . import _lib
from .embedding_bag import _require_device

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_BLOCK = 256
_CODES = torch.float8_e4m3fn
_FIELDS = 9  # words of pkm_adamw_tensor_t
_GRAD = 1  # the gradient's
_DTYPE = operator.attrgetter("dtype")


def _names(bits: int, master: bool) -> tuple[str, ...]:
    """A tensor's states in the order of pkm_adamw_tensor_t: first moment, second, their steps, master."""
    names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "exp_root", "exp_avg_scale", "exp_root_scale")
    return (*names, "master") if master else names


class _Plan:
    """What a step passes for tensors of one type and kind: their pointers, of which the gradients' change."""

    def __init__(self, params: list, states: list[dict], bits: int, master: bool):
        self.params, self.states, self.bits = params, states, bits
        self.names = (*_names(bits, master), "step")
        self.take = operator.itemgetter(*self.names)
        self.held = [self.take(s) for s in states]
        self.table = (_lib.AdamWTensor * len(params))()
        self.words = np.frombuffer(self.table, dtype=np.int64).reshape(len(params), _FIELDS)
        self.places = self._places()
        for row, p, s in zip(self.table, params, states):
            row.param, row.exp_avg, row.step, row.numel = p.data_ptr(), s["exp_avg"].data_ptr(), s["step"].data_ptr(), p.numel()
            row.second = s["exp_avg_sq" if bits == 32 else "exp_root"].data_ptr()
            if bits == 8:
                row.exp_avg_scale, row.second_scale = s["exp_avg_scale"].data_ptr(), s["exp_root_scale"].data_ptr()
            if master:
                row.master = s["master"].data_ptr()
        self.device, self.dtype = params[0].device, _lib.dtype_code(params[0])
        self.grads_are = [*map(Tensor.numel, params), *map(Tensor.get_device, params), *map(_DTYPE, params)]
        self.ws_bytes = _lib.load().pkm_adamw_workspace_size(len(params))

    def _places(self) -> list:
        """Where weights and states lie (an address is of one device), which an assignment to their `data` changes too, and
        what the weights are: another type may have the same memory (a view, or a copy that was put where the weight had been)."""
        params, states = self.params, itertools.chain.from_iterable(map(self.take, self.states))
        return [*map(Tensor.data_ptr, params), *map(Tensor.numel, params), *map(Tensor.is_contiguous, params),
                *map(_DTYPE, params), *map(Tensor.data_ptr, states)]

    def stands(self) -> bool:
        """Whether the weights and states are what and where they were: what is held here keeps its place to itself."""
        return self._places() == self.places


class AdamW(torch.optim.Optimizer):
    """AdamW(params, lr, betas, eps, weight_decay, state_bits=32 or 8, master_weights=False); every option may differ
    between parameter groups."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = False):
        self._plans: dict = {}
        self._planned: list = []  # the parameters' states when the plans were made
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:  # of an optimizer without these options
            for name, value in self.defaults.items():
                group.setdefault(name, value)
        self._plans, self._planned = {}, []

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check(group)
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group: dict) -> None:
        lr = group["lr"]
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1:
                raise ValueError(f"AdamW: lr as a tensor has to be one float32 number, got {lr.dtype} {tuple(lr.shape)}")
        elif not (isinstance(lr, (int, float)) and math.isfinite(lr) and lr >= 0):
            raise ValueError(f"AdamW: lr {lr!r} has to be at least 0")
        if len(group["betas"]) != 2 or not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError(f"AdamW: betas {group['betas']!r} have to lie in [0, 1)")
        for name in ("eps", "weight_decay"):
            if not (math.isfinite(group[name]) and group[name] >= 0):
                raise ValueError(f"AdamW: {name} {group[name]!r} has to be at least 0")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"AdamW: state_bits {group['state_bits']!r} has to be 8 or 32")

    def _new_state(self, p: torch.Tensor, bits: int, master: bool) -> dict:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the states of a captured step have to be there before: take a step, or load a state")
        zeros = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device=p.device)
        held = torch.float32 if bits == 32 else _CODES
        state = {"step": zeros((), torch.float32), "exp_avg": zeros(p.shape, held)}
        if bits == 32:
            state["exp_avg_sq"] = zeros(p.shape, held)
        else:
            blocks = -(-p.numel() // _BLOCK)
            state["exp_root"] = zeros(p.shape, held)
            state["exp_avg_scale"], state["exp_root_scale"] = (zeros(blocks, torch.float32) for _ in range(2))
        if master:
            state["master"] = p.detach().float().clone()
        return state

    @staticmethod
    def _check_state(state: dict, p: torch.Tensor, bits: int, master: bool) -> None:
        wide = torch.float32
        kinds = {"exp_avg": wide if bits == 32 else _CODES, "exp_avg_sq": wide, "exp_root": _CODES, "exp_avg_scale": wide,
                 "exp_root_scale": wide, "master": wide, "step": wide}
        for name in (*_names(bits, master), "step"):
            x = state.get(name)
            n = 1 if name == "step" else -(-p.numel() // _BLOCK) if name.endswith("scale") else p.numel()
            if not isinstance(x, torch.Tensor) or x.dtype != kinds[name] or x.numel() != n or x.device != p.device \
                    or not x.is_contiguous():
                raise ValueError(f"AdamW: the state {name!r} of a parameter {tuple(p.shape)} has to be {n} contiguous numbers "
                                 f"of {kinds[name]} on {p.device}, with state_bits={bits}, master_weights={master}")

    def _plans_of(self, params: list, bits: int, master: bool) -> list[_Plan]:
        kinds: dict = {}
        for p in params:
            if p.dtype not in _DTYPES or not p.is_contiguous():
                raise NotImplementedError(f"AdamW: a parameter {tuple(p.shape)} of {p.dtype}, strides {p.stride()} is not "
                                          "supported (contiguous float32, bfloat16 and float16 are)")
            if p.grad.shape != p.shape:  # of before the weight's data were exchanged
                raise ValueError(f"AdamW: a gradient {tuple(p.grad.shape)} of a parameter {tuple(p.shape)}")
            _require_device(p)
            # a float32 weight is its own master
            kinds.setdefault((p.device, p.dtype, master and p.dtype != torch.float32), []).append(p)
        plans = []
        for (_, _, with_master), some in kinds.items():
            for p in some:
                if not self.state[p]:
                    self.state[p] = self._new_state(p, bits, with_master)
                self._check_state(self.state[p], p, bits, with_master)
            plans.append(_Plan(some, [self.state[p] for p in some], bits, with_master))
        return plans

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: torch.Tensor | None = None):
        """One step of every parameter that has a gradient. grad_scale: one float32 number on the device that the
        gradients are multiplied by (a loss scale's inverse, a clipping factor)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grad_scale is not None and (grad_scale.dtype != torch.float32 or grad_scale.numel() != 1):
            raise ValueError(f"AdamW.step: grad_scale has to be one float32 number, got {grad_scale.dtype} "
                             f"{tuple(grad_scale.shape)}")
        if len(self.state) != len(self._planned) or not all(map(operator.is_, self.state.values(), self._planned)):
            self._plans = {}
        for i, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            self._check(group)
            bits, master = group["state_bits"], bool(group["master_weights"])
            held = self._plans.get(i)
            if held is None or held[0] != (bits, master) or len(held[1]) != len(params) \
                    or not all(map(operator.is_, held[1], params)) or not all(plan.stands() for plan in held[2]):
                held = self._plans[i] = ((bits, master), params, self._plans_of(params, bits, master))
                self._planned = list(self.state.values())
            for plan in held[2]:
                self._launch(plan, group, grad_scale)
        return loss

    @staticmethod
    def _gradients(plan: _Plan) -> list[torch.Tensor]:
        """The gradients of a plan's weights, contiguous. Anything may have come to lie in their `data` since the last step."""
        grads = [p.grad for p in plan.params]
        whole = all(map(Tensor.is_contiguous, grads))  # which sparse ones are not
        if not whole or [*map(Tensor.numel, grads), *map(Tensor.get_device, grads), *map(_DTYPE, grads)] != plan.grads_are:
            for p, g in zip(plan.params, grads):
                if g.dtype != p.dtype or g.layout is not torch.strided:
                    raise NotImplementedError(f"AdamW: a gradient of {g.dtype}, {g.layout} for a parameter of {p.dtype} is not "
                                              "supported (dense ones of the parameter's type are)")
                if g.shape != p.shape or g.device != p.device:
                    raise ValueError(f"AdamW: a gradient {tuple(g.shape)} on {g.device} of a parameter {tuple(p.shape)} on {p.device}")
        return grads if whole else [g.contiguous() for g in grads]

    def _launch(self, plan: _Plan, group: dict, grad_scale) -> None:
        grads = self._gradients(plan)
        lr = group["lr"]
        lr_device = lr if isinstance(lr, torch.Tensor) and lr.is_cuda else None
        if lr_device is not None or grad_scale is not None:
            _require_device(plan.params[0], lr_device, grad_scale)
        plan.words[:, _GRAD] = list(map(Tensor.data_ptr, grads))
        ws = torch.empty(plan.ws_bytes, dtype=torch.uint8, device=plan.device)
        _lib.call_on(plan.device, "pkm_adamw_step", plan.table, len(grads), plan.dtype, plan.bits,
                     0.0 if lr_device is not None else float(lr), _lib.ptr(lr_device), *group["betas"], group["eps"],
                     group["weight_decay"], _lib.ptr(grad_scale), _lib.ptr(ws), plan.ws_bytes, _lib.stream_of(plan.device))
        torch.autograd.graph.increment_version(plan.params)  # as an update in place does

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's; states keep their types (torch's would take that of the weight)."""
        super().load_state_dict({**state_dict, "state": {}})
        self._plans = {}
        self.state.clear()
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for (group, p), i in zip(((g, p) for g in self.param_groups for p in g["params"]), ids):
            saved = state_dict["state"].get(i)
            if not saved:
                continue
            state = {n: x.to(device=p.device).contiguous() if isinstance(x, torch.Tensor) else x for n, x in saved.items()}
            state["step"] = torch.as_tensor(state["step"], dtype=torch.float32, device=p.device).reshape(())
            self._check_state(state, p, group["state_bits"], bool(group["master_weights"]) and p.dtype != torch.float32)
            self.state[p] = state


__all__ = ["AdamW"]
