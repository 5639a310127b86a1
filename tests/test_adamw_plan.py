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
