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
as zeros. A gradient that is infinite or NaN makes its block's step so: all 256
weights of the block are NaN from the next step on (with 32 bits only its own).
Nothing on the device leaves such a step out: whoever scales a loss looks at its
gradients before the step, and does not capture that step into a graph.

16-bit weights lose updates below half their spacing; `master_weights=True` keeps a
float32 copy ("master") that the update is made to, the weight its rounding: who
changes such a weight otherwise changes its master too, or the next step undoes it.

Steps are counted on the device, one counter a tensor, and nothing synchronises: a
step can be captured into a graph (after a first one, or a loaded state, has made
the states) and counts on with every replay. lr may be a float32 number on the
device, read when the step runs.

Supported: float32, bfloat16 and float16 parameters on the GPU, contiguous, with
dense gradients of their type; anything else raises NotImplementedError. There is
no CPU path: CPU tensors raise. The parameters of a group are updated at once: one
that is there twice, and parameters or states that share memory, raise ValueError.
"""
from __future__ import annotations

import collections
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
_IN_CODES = ("exp_avg", "exp_root")
_FIELDS = 9  # words of pkm_adamw_tensor_t
_PARAM, _GRAD, _NUMEL = 0, 1, 8
_COLUMNS = {"exp_avg": 2, "exp_avg_sq": 3, "exp_root": 3, "exp_avg_scale": 4, "exp_root_scale": 5, "master": 6, "step": 7}
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
        self.grads_at = self.words[:, _GRAD]
        self.places = self._places()
        columns = (_PARAM, *(_COLUMNS[n] for n in self.names))
        for column, tensors in zip(columns, zip(*((p, *held) for p, held in zip(params, self.held)))):
            self.words[:, column] = list(map(Tensor.data_ptr, tensors))
        self.words[:, _NUMEL] = list(map(Tensor.numel, params))
        if self._shares_memory(params[0].element_size(), master):
            raise ValueError(f"AdamW: parameters of one group, or their states, share memory (of {len(params)} of {params[0].dtype}):"
                             " they would be updated at once")
        self.device, self.dtype = params[0].device, _lib.dtype_code(params[0])
        self.grads_are = [*map(Tensor.numel, params), *map(Tensor.get_device, params), *map(_DTYPE, params)]
        self.ws_bytes = _lib.load().pkm_adamw_workspace_size(len(params))

    def _shares_memory(self, item: int, master: bool) -> bool:
        """Whether anything that a step writes lies in two places of the table: its rows are worked on at once."""
        n, held = self.words[:, _NUMEL:], self.bits // 8
        sizes = n * np.array([item, 0, held, held, 0, 0, 4 * master, 0])
        if self.bits == 8:
            sizes[:, 4:6] = -(-n // _BLOCK) * 4
        sizes[:, 7] = 4
        begins, sizes = self.words[:, :_NUMEL].flatten(), sizes.ravel()
        begins[sizes == 0] = 0
        order = np.argsort(begins)
        begins = begins[order]
        ends = begins + sizes[order]
        return bool((ends[:-1] > begins[1:]).any())

    def _places(self) -> list:
        """Where weights and states lie (an address is of one device), which an assignment to their `data` changes too, and
        what the weights are: another type may have the same memory (a view, or a copy that was put where the weight had been).
        What the states are is looked at where their places change: five more questions a weight would take 15 % of a small step."""
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
        if "_loading" in self.__dict__:
            state = {**state, "state": self.__dict__.pop("_loading")}
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
            if len(set(map(id, group["params"]))) != len(group["params"]):  # torch warns only
                raise ValueError("AdamW: a parameter group holds a parameter more than once")
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
        for name in ("amsgrad", "maximize", "differentiable"):  # torch's
            if group.get(name):
                raise NotImplementedError(f"AdamW: {name} is not supported")
        if not group.get("decoupled_weight_decay", True) and group["weight_decay"]:
            raise NotImplementedError("AdamW: decoupled_weight_decay=False, decay in the gradient, is not supported")

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
    def _check_states(states: list[dict], params: list, bits: int, master: bool) -> None:
        numels, places = list(map(Tensor.numel, params)), list(map(Tensor.get_device, params))
        blocks = [-(-n // _BLOCK) for n in numels]
        for name in (*_names(bits, master), "step"):
            kind = _CODES if bits == 8 and name in _IN_CODES else torch.float32
            sizes = [1] * len(params) if name == "step" else blocks if name.endswith("scale") else numels
            for p, x, n, place in zip(params, (s.get(name) for s in states), sizes, places):
                if not isinstance(x, Tensor) or x.dtype is not kind or x.numel() != n or not x.is_contiguous() \
                        or x.get_device() != place:
                    raise ValueError(f"AdamW: the state {name!r} of a parameter {tuple(p.shape)} has to be {n} contiguous numbers "
                                     f"of {kind} on {p.device}, with state_bits={bits}, master_weights={master}")

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
            states = [self.state[p] for p in some]
            for i, p in enumerate(some):
                if not states[i]:
                    states[i] = self.state[p] = self._new_state(p, bits, with_master)
            self._check_states(states, some, bits, with_master)
            plans.append(_Plan(some, states, bits, with_master))
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
        work = []  # all groups are looked at before the first runs: a step that is refused changes nothing
        for i, group in enumerate(self.param_groups):
            grads = [p.grad for p in group["params"]]
            params = [p for p, g in zip(group["params"], grads) if g is not None]
            if not params:
                continue
            if len(params) != len(grads):
                grads = [g for g in grads if g is not None]
            self._check(group)
            bits, master = group["state_bits"], bool(group["master_weights"])
            held = self._plans.get(i)
            if held is None or held[0] != (bits, master) or len(held[1]) != len(params) \
                    or not all(map(operator.is_, held[1], params)) or not all(plan.stands() for plan in held[2]):
                held = self._plans[i] = ((bits, master), params, self._plans_of(params, bits, master))
                self._planned = list(self.state.values())
            for plan in held[2]:
                own = grads if len(held[2]) == 1 else [p.grad for p in plan.params]
                work.append((plan, group, self._checked(plan, own), self._rate(plan, group, grad_scale)))
        for plan, group, grads, rate in work:
            self._launch(plan, group, grads, rate, grad_scale)
        return loss

    @staticmethod
    def _checked(plan: _Plan, grads: list) -> list[torch.Tensor]:
        """The gradients of a plan's weights, contiguous. Anything may have come to lie in their `data` since the last step."""
        whole = all(map(Tensor.is_contiguous, grads))  # which sparse ones are not
        if not whole or [*map(Tensor.numel, grads), *map(Tensor.get_device, grads), *map(_DTYPE, grads)] != plan.grads_are:
            for p, g in zip(plan.params, grads):
                if g.dtype != p.dtype or g.layout is not torch.strided:
                    raise NotImplementedError(f"AdamW: a gradient of {g.dtype}, {g.layout} for a parameter of {p.dtype} is not "
                                              "supported (dense ones of the parameter's type are)")
                if g.shape != p.shape or g.device != p.device:
                    raise ValueError(f"AdamW: a gradient {tuple(g.shape)} on {g.device} of a parameter {tuple(p.shape)} on {p.device}")
        return grads if whole else [g.contiguous() for g in grads]

    @staticmethod
    def _rate(plan: _Plan, group: dict, grad_scale) -> tuple:
        """The rate as a number, and as one on the device."""
        lr = group["lr"]
        on_device = lr if isinstance(lr, Tensor) and lr.is_cuda else None
        if on_device is not None or grad_scale is not None:
            _require_device(plan.params[0], on_device, grad_scale)
        return (float(lr), None) if on_device is None else (0.0, on_device)

    def _launch(self, plan: _Plan, group: dict, grads: list, rate: tuple, grad_scale) -> None:
        plan.grads_at[:] = list(map(Tensor.data_ptr, grads))
        ws = torch.empty(plan.ws_bytes, dtype=torch.uint8, device=plan.device)
        _lib.call_on(plan.device, "pkm_adamw_step", plan.table, len(grads), plan.dtype, plan.bits, rate[0],
                     _lib.ptr(rate[1]), *group["betas"], group["eps"], group["weight_decay"], _lib.ptr(grad_scale),
                     _lib.ptr(ws), plan.ws_bytes, _lib.stream_of(plan.device))
        torch.autograd.graph.increment_version(plan.params)  # as an update in place does

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's; states keep their types (torch's would take that of the weight). One that is refused changes nothing."""

        def take(_, loaded: dict) -> dict:  # the last of the hooks before: what the others have made of it
            self._loading = self._states_of(loaded)
            return {**loaded, "state": {}}

        handle = self.register_load_state_dict_pre_hook(take)
        try:
            super().load_state_dict(state_dict)  # which hands on to __setstate__
        finally:
            handle.remove()
            self.__dict__.pop("_loading", None)

    def _states_of(self, loaded: dict) -> collections.defaultdict:
        """What is loaded as the parameters' states, on their devices."""
        states, names = collections.defaultdict(dict), set()
        for group, saved in zip(self.param_groups, loaded["param_groups"]):
            options = {**self.defaults, **saved}
            self._check(options)
            for p, i in zip(group["params"], saved["params"]):
                names.add(i)
                if not loaded["state"].get(i):
                    continue
                state = {n: x.to(device=p.device).contiguous() if isinstance(x, Tensor) else x
                         for n, x in loaded["state"][i].items()}
                if "step" in state:  # a counter of its own, which saved ones may share
                    state["step"] = torch.as_tensor(state["step"], dtype=torch.float32, device=p.device).reshape(()).clone()
                with_master = bool(options["master_weights"]) and p.dtype != torch.float32
                self._check_states([state], [p], options["state_bits"], with_master)
                states[p] = state
        states.update((i, x) for i, x in loaded["state"].items() if i not in names)  # of no parameter: as torch's
        return states


__all__ = ["AdamW"]
