"""AdamW: arguments that are refused and states that do not fit, on the CPU before any kernel runs."""
from __future__ import annotations

import ctypes

import pytest
import torch

from modelos_amd import _lib, build_lib
from modelos_amd.adamw import AdamW
from oracle import adamw as oracle

P = 1 << 20


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    return _lib.load()


def _param(*shape, dtype=torch.float32, grad=True):
    p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype))
    if grad:
        p.grad = torch.zeros_like(p)
    return p


@pytest.mark.parametrize("options", [
    {"lr": -1.0}, {"lr": float("nan")}, {"lr": "fast"}, {"lr": torch.zeros(2)}, {"lr": torch.zeros((), dtype=torch.float64)},
    {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"betas": (0.9,)}, {"eps": -1e-8}, {"weight_decay": float("inf")},
    {"state_bits": 16},
])
def test_refused_options(options):
    with pytest.raises(ValueError):
        AdamW([_param(3)], **options)
    opt = AdamW([_param(3)])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [_param(4)], **options})
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("p,error", [
    (_param(4), RuntimeError),  # CPU
    (_param(4, dtype=torch.float64), NotImplementedError),
])
def test_refused_parameters(p, error):
    with pytest.raises(error):
        AdamW([p]).step()


def test_refused_strides():
    p = torch.zeros(4, 6).T.requires_grad_()
    p.grad = torch.zeros_like(p)
    with pytest.raises(NotImplementedError, match="contiguous"):
        AdamW([p]).step()


def test_grad_scale_is_one_number():
    for scale in (torch.ones(2), torch.ones((), dtype=torch.float64)):
        with pytest.raises(ValueError, match="grad_scale"):
            AdamW([_param(3)]).step(grad_scale=scale)


def test_nothing_to_do():
    opt = AdamW([_param(3, grad=False)])
    assert opt.step(lambda: 5) == 5
    assert not opt.state


def _state(bits=32, n=300, with_master=False, **other):
    s = {"step": torch.tensor(3.0), "exp_avg": torch.zeros(n, dtype=torch.float32 if bits == 32 else torch.float8_e4m3fn)}
    if bits == 32:
        s["exp_avg_sq"] = torch.zeros(n)
    else:
        s.update(exp_root=torch.zeros(n, dtype=torch.float8_e4m3fn), exp_avg_scale=torch.zeros(2), exp_root_scale=torch.zeros(2))
    if with_master:
        s["master"] = torch.zeros(n)
    return {**s, **other}


@pytest.mark.parametrize("bits", [8, 32])
def test_load_state(bits):
    opt = AdamW([_param(300, dtype=torch.bfloat16), _param(2)], state_bits=bits, master_weights=True)
    groups = opt.state_dict()["param_groups"]
    state = _state(bits, with_master=True)
    opt.load_state_dict({"state": {0: state}, "param_groups": groups})
    got = opt.state_dict()["state"]
    assert set(got) == {0} and all(got[0][n].dtype == x.dtype and torch.equal(got[0][n].float(), x.float()) for n, x in state.items())
    for wrong in (_state(40 - bits, with_master=True), _state(bits), _state(bits, n=299, with_master=True),
                  _state(bits, with_master=True, exp_avg=torch.zeros(300, dtype=torch.bfloat16)),
                  _state(bits, with_master=True, master=torch.zeros(300, dtype=torch.bfloat16))):
        with pytest.raises(ValueError, match="state"):
            opt.load_state_dict({"state": {0: wrong}, "param_groups": groups})


def _tensors(n, **fields):
    full = dict(param=P, grad=P, exp_avg=P, second=P, exp_avg_scale=P, second_scale=P, master=None, step=P, numel=8)
    return (_lib.AdamWTensor * n)(*(_lib.AdamWTensor(**{**full, **(fields if i == n - 1 else {})}) for i in range(n)))


@pytest.mark.parametrize("tensors,count,dtype,bits,ws,status", [
    (_tensors(1), -1, 0, 32, 1 << 20, 1), (_tensors(1), 1, 5, 32, 1 << 20, 1), (_tensors(1), 1, 0, 4, 1 << 20, 1),
    (None, 1, 0, 32, 1 << 20, 1), (_tensors(2, param=None), 2, 0, 32, 1 << 20, 1), (_tensors(2, grad=None), 2, 0, 32, 1 << 20, 1),
    (_tensors(2, step=None), 2, 0, 32, 1 << 20, 1), (_tensors(2, numel=-1), 2, 0, 32, 1 << 20, 1),
    (_tensors(2, second_scale=None), 2, 0, 8, 1 << 20, 1), (_tensors(2, master=P), 2, 0, 32, 1 << 20, 1),
    (_tensors(2, numel=1 << 35), 2, 0, 32, 1 << 20, 2), (_tensors(2), 2, 0, 32, 31, 3), (None, 0, 0, 32, 0, 0),
])
def test_entry(lib, tensors, count, dtype, bits, ws, status):
    got = lib.pkm_adamw_step(tensors, count, dtype, bits, 1e-3, None, 0.9, 0.99, 1e-8, 0.0, None, ctypes.c_void_p(P), ws, None)
    assert got == status


def test_workspace_size(lib):
    assert [lib.pkm_adamw_workspace_size(n) for n in (0, 1, 100, -1)] == [0, 16, 1600, 0]


def test_oracle_dither_loses_nothing():
    """Numbers between two codes become either, in shares that keep their mean as far as the dither runs evenly through
    [0, 1): over N steps, the share of dithers in [x, 1) is off by at most max |x_(i) - i / N| + 1 / N (their star
    discrepancy, x_(i) in order), which the continued fraction 1 / (1 + 1 / (1 + 1 / (10 + ...))) of 2246822519 / 2^32 keeps
    to a few N-ths."""
    a = torch.tensor([448.0, 3.3, 0.001, 100.9]).repeat(64)
    N = 4096
    dithers = torch.stack([oracle.dither(256, t)[0] for t in range(N)])
    off = (dithers.sort(0).values - torch.arange(N)[:, None] / N).abs().amax(0) + 1 / N
    assert off.max() <= 16 / N
    held = torch.stack([oracle.hold(a, u, 0.0)[0] for u in dithers]).mean(0)
    spacing = torch.tensor([32.0, 2.0**-2, 2.0**-9, 2.0**3]).repeat(64)
    assert ((held - a).abs() <= spacing * off + a * 2.0**-20).all()


def test_load_groups_of_another_optimizer():
    """torch's own AdamW has other options: those that are missing keep their defaults."""
    p = _param(3)
    opt = AdamW([p], state_bits=8)
    opt.load_state_dict(torch.optim.AdamW([_param(3)], lr=0.5).state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["state_bits"] == 8 and not opt.param_groups[0]["master_weights"]


def test_gradient_of_data_that_was_exchanged():
    p = _param(4)
    p.data = torch.zeros(9)
    with pytest.raises(ValueError, match=r"gradient \(4,\) of a parameter \(9,\)"):
        AdamW([p]).step()


@pytest.mark.parametrize("bits", [8, 32])
def test_hooks_of_loading_see_the_states(bits):
    """As with torch's optimizers: a hook before sees, and may change, what is loaded; one behind finds it loaded."""
    opt = AdamW([_param(300)], state_bits=bits)
    seen = []

    def before(optimizer, loaded):
        seen.append((len(optimizer.state), set(loaded["state"][0])))
        return {**loaded, "state": {0: {**loaded["state"][0], "step": torch.tensor(9.0)}}}

    def behind(optimizer):
        (state,) = optimizer.state.values()
        seen.append((state["step"].item(), state["exp_avg"].dtype))

    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(behind)
    state = _state(bits)
    opt.load_state_dict({"state": {0: state}, "param_groups": opt.state_dict()["param_groups"]})
    assert seen == [(0, set(state)), (9.0, state["exp_avg"].dtype)]


@pytest.mark.parametrize("wrong", ["state", "of another kind", "groups", "sizes", "option"])
def test_a_refused_load_changes_nothing(wrong):
    p, q = _param(300), _param(2)
    opt = AdamW([{"params": [p]}, {"params": [q], "lr": 0.25}], betas=(0.5, 0.5))
    groups = opt.state_dict()["param_groups"]
    opt.load_state_dict({"state": {0: _state(), 1: _state(n=2)}, "param_groups": groups})
    held = {t: dict(s) for t, s in opt.state.items()}
    new = [{**g, "lr": 0.125} for g in groups]
    states = {0: _state(step=torch.tensor(8.0)), 1: _state(n=2)}
    if wrong == "state":
        states[1] = _state(n=3)
    elif wrong == "of another kind":
        new[1]["state_bits"] = 8
    elif wrong == "groups":
        new = new[:1]
    elif wrong == "sizes":
        new[1] = {**new[1], "params": [1, 2]}
    else:
        new[1]["weight_decay"] = -1.0
    with pytest.raises(ValueError):
        opt.load_state_dict({"state": states, "param_groups": new})
    assert [g["lr"] for g in opt.param_groups] == [1e-3, 0.25] and opt.param_groups[1]["state_bits"] == 32
    assert set(opt.state) == {p, q} and all(opt.state[t][n] is x for t, s in held.items() for n, x in s.items())


def test_loaded_options_decide_what_states_are():
    """Those that are loaded, not those that the optimizer had."""
    opt = AdamW([_param(300)])
    saved = AdamW([_param(300)], state_bits=8).state_dict()["param_groups"]
    opt.load_state_dict({"state": {0: _state(8)}, "param_groups": saved})
    assert opt.param_groups[0]["state_bits"] == 8 and "exp_root" in opt.state[opt.param_groups[0]["params"][0]]


def test_copies():
    import copy

    opt = AdamW([_param(300, dtype=torch.bfloat16)], state_bits=8)
    opt.load_state_dict({"state": {0: _state(8)}, "param_groups": opt.state_dict()["param_groups"]})
    twin = copy.deepcopy(opt)
    (s,), (t,) = opt.state.values(), twin.state.values()
    assert set(s) == set(t) and all(x.dtype == t[n].dtype and torch.equal(x.float(), t[n].float()) for n, x in s.items())
    assert twin.param_groups[0]["state_bits"] == 8


def test_loaded_counters_are_their_own():
    opt = AdamW([_param(300), _param(300)])
    one = torch.tensor(4.0)
    opt.load_state_dict({"state": {0: _state(step=one), 1: _state(step=one)}, "param_groups": opt.state_dict()["param_groups"]})
    a, b = (s["step"] for s in opt.state.values())
    assert a.item() == b.item() == 4.0 and len({x.data_ptr() for x in (a, b, one)}) == 3
    without = _state()
    del without["step"]
    with pytest.raises(ValueError, match="step"):
        opt.load_state_dict({"state": {0: without}, "param_groups": opt.state_dict()["param_groups"]})


@pytest.mark.parametrize("option", [{"amsgrad": True}, {"maximize": True}, {"differentiable": True},
                                    {"decoupled_weight_decay": False}])
def test_options_of_torchs_that_are_not_there(option):
    """Of a group that is given or loaded: not silently left out."""
    with pytest.raises(NotImplementedError, match=next(iter(option))):
        AdamW([{"params": [_param(3)], **option}])
    opt = AdamW([_param(3)])
    (group,) = opt.state_dict()["param_groups"]
    with pytest.raises(NotImplementedError, match=next(iter(option))):
        opt.load_state_dict({"state": {}, "param_groups": [{**group, **option}]})
    opt.param_groups[0].update(option)
    with pytest.raises(NotImplementedError, match=next(iter(option))):
        opt.step()
    AdamW([{"params": [_param(3)], **option, "weight_decay": 0.0}] if "decoupled_weight_decay" in option else [_param(3)])
