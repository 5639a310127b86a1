"""AdamW's plan of a step, on the CPU with the launch taken out: what is passed on after weights, states and gradients were
exchanged for others, and what is refused before anything runs."""
from __future__ import annotations

import pytest
import torch

from modelos_amd import _lib, adamw, build_lib
from modelos_amd.adamw import AdamW

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def launches(monkeypatch):
    """The launches of the steps that follow: (dtype, state bits, the tensors' fields)."""
    if not _lib.LIB_PATH.exists():
        build_lib.build(verbose=False)
    made = []

    def call_on(device, name, table, count, dtype, bits, *rest):
        assert name == "pkm_adamw_step" and len(table) == count
        made.append((dtype, bits, [{n: getattr(row, n) for n, _ in row._fields_} for row in table]))

    monkeypatch.setattr(_lib, "call_on", call_on)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(adamw, "_require_device", lambda *tensors: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return made


def _param(*shape, dtype=F32):
    p = torch.nn.Parameter(torch.zeros(shape, dtype=dtype))
    p.grad = torch.zeros_like(p)
    return p


def _steps(params, launches, **options):
    opt = AdamW(params, **options)
    opt.step()
    opt.step()
    assert launches
    launches.clear()
    return opt


@pytest.mark.parametrize("bits", [8, 32])
def test_a_weight_viewed_as_another_type(bits, launches):
    """The same memory and as many numbers, of the other type of 16 bits: the step's type follows."""
    p = _param(6, 50, dtype=BF16)
    opt = _steps([p], launches, state_bits=bits)
    p.grad, p.data = None, p.data.view(F16)
    p.grad = torch.zeros_like(p)
    opt.step()
    assert [x[0] for x in launches] == [_lib.DTYPE_CODES[F16]]


def test_a_weight_of_another_type_in_the_same_place(launches):
    """A float32 weight's memory taken by one of 16 bits and as many numbers: nothing may be written as float32 there. With
    masters it then needs one."""
    p = _param(40)
    opt = _steps([p], launches, master_weights=True)
    p.grad, p.data = None, p.data.view(BF16)[:40]
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError, match="master"):
        opt.step()
    assert not launches


@pytest.mark.parametrize("data", [torch.zeros(39), torch.zeros(41), torch.zeros(0)], ids=["shorter", "longer", "none"])
@pytest.mark.parametrize("which", [0, 2])
def test_a_gradient_exchanged_for_one_that_does_not_fit(which, data, launches):
    """Through its `data`, which torch lets pass, between two steps of one plan."""
    params = [_param(40), _param(3), _param(40)]
    opt = _steps(params, launches)
    params[which].grad.data = data
    with pytest.raises(ValueError, match="gradient"):
        opt.step()
    assert not launches


def test_gradients_in_other_places_and_orders(launches):
    """Every step's own gradients are passed on, those of other strides as copies in the weight's order."""
    params = [_param(4, 6), _param(3), _param(4, 6)]
    opt = _steps(params, launches)
    for _ in range(2):
        for p in params:
            p.grad = torch.zeros_like(p)
        params[2].grad = torch.zeros(6, 4).T
        opt.step()
        ((_, _, rows),) = launches
        launches.clear()
        assert [r["grad"] for r in rows[:2]] == [p.grad.data_ptr() for p in params[:2]]
        assert rows[2]["grad"] != params[2].grad.data_ptr()


@pytest.mark.parametrize("grad", [torch.zeros(4, 6).to_sparse(), torch.zeros(4, 6, dtype=BF16)], ids=["sparse", "bf16"])
def test_gradients_of_another_kind(grad, launches):
    p = _param(4, 6)
    opt = _steps([p], launches)
    if grad.dtype == p.dtype:
        p.grad = grad
    else:
        p.grad.data = grad
    with pytest.raises(NotImplementedError, match="gradient"):
        opt.step()
    assert not launches


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
def test_one_weight_twice(launches):
    """Two rows of one launch would update the same numbers at once."""
    p, q = _param(40), _param(3)
    with pytest.raises(ValueError, match="more than once"):
        AdamW([p, q, p])
    opt = AdamW([q])
    with pytest.raises(ValueError, match="more than once"):
        opt.add_param_group({"params": [p, p]})
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("bits", [8, 32])
def test_weights_that_share_memory(bits, launches):
    """Of one launch; those that lie side by side in one tensor do not."""
    flat = torch.zeros(600)
    a, b, c = (torch.nn.Parameter(flat[i:j]) for i, j in ((0, 300), (300, 600), (299, 301)))
    for p in (a, b, c):
        p.grad = torch.zeros_like(p)
    AdamW([b, a], state_bits=bits).step()
    assert len(launches) == 1
    for pair in ([a, c], [c, b], [a, b, c]):
        with pytest.raises(ValueError, match="share memory"):
            AdamW(pair, state_bits=bits).step()
    assert len(launches) == 1
    AdamW([{"params": [a]}, {"params": [c]}], state_bits=bits).step()  # one after the other
    assert len(launches) == 3


@pytest.mark.parametrize("name", ["exp_avg", "exp_root", "exp_avg_scale", "master", "step"])
def test_states_that_share_memory(name, launches):
    params = [_param(300, dtype=BF16), _param(300, dtype=BF16), _param(0, dtype=BF16)]
    opt = _steps(params, launches, state_bits=8, master_weights=True)
    opt.state[params[1]][name] = opt.state[params[0]][name]
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    assert not launches


@pytest.mark.parametrize("what", ["sparse", "shorter", "rate", "option", "state", "scale"])
def test_a_refused_step_changes_nothing(what, launches, monkeypatch):
    """A group that cannot be stepped: neither are the groups before it."""
    a, b, c = _param(40), _param(40, dtype=BF16), _param(5)
    opt = _steps([{"params": [a, b]}, {"params": [c]}], launches)
    if what == "sparse":
        c.grad = torch.zeros(5).to_sparse()
    elif what == "shorter":
        c.grad.data = torch.zeros(4)
    elif what == "option":
        opt.param_groups[1]["betas"] = (0.9, 1.0)
    elif what == "state":
        opt.state[c]["exp_avg"] = torch.zeros(4)
    elif what == "rate":
        opt.param_groups[1]["lr"] = torch.zeros(2)

    def require(*tensors):
        if any(t is not None and t.dim() == 1 and t.numel() == 1 for t in tensors):
            raise RuntimeError("elsewhere")

    monkeypatch.setattr(adamw, "_require_device", require)
    scale = torch.ones(1) if what == "scale" else None
    with pytest.raises((ValueError, NotImplementedError, RuntimeError)):
        opt.step(grad_scale=scale)
    assert not launches
