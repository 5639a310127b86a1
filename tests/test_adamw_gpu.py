"""AdamW against the formulas in 64 bits, its 8-bit states bit for bit."""
from __future__ import annotations

import copy

import pytest
import torch

from modelos_amd.adamw import AdamW
from oracle import adamw as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SIZES = [(1,), (0,), (255,), (16, 16), (257,), (64, 64), (4097,), (3, 5, 7), (100, 333)]
HYPER = dict(lr=3e-3, betas=(0.8, 0.96), eps=1e-6, weight_decay=0.2)


def _params(gen, dtype, device, sizes=SIZES, offset=0):
    out = []
    for s in sizes:
        n = int(torch.tensor(s).prod())
        flat = torch.zeros(n + offset, dtype=dtype, device=device)
        p = flat[offset:].view(s)
        p.copy_(torch.randn(s, generator=gen))
        out.append(p.requires_grad_())
    return out


def _grads(gen, params, offset=0):
    for p in params:
        size = 1e-2 * torch.exp(2 * torch.randn((), generator=gen))
        flat = torch.zeros(p.numel() + offset, dtype=p.dtype, device=p.device)
        p.grad = flat[offset:].view(p.shape)
        p.grad.copy_(size * torch.randn(p.shape, generator=gen))


def _check_step(before, after, p0, p, g, t, bits, hyper=HYPER):
    """One step of one tensor from the state `before`, all on the CPU."""
    betas = hyper["betas"]
    if bits == 32:
        m0, v0 = before["exp_avg"], before["exp_avg_sq"]
    else:
        m0 = oracle.numbers(before["exp_avg"], before["exp_avg_scale"])
        r0 = oracle.numbers(before["exp_root"], before["exp_root_scale"])
        v0 = r0 * r0
    m, v = oracle.moments(g.float(), m0, v0, betas)
    if bits == 32:
        assert torch.equal(after["exp_avg"], m) and torch.equal(after["exp_avg_sq"], v)
    else:
        root = v.double().sqrt().float()  # rounded once, which torch's float32 root on the CPU is not
        for name, x, u, least in zip(("exp_avg", "exp_root"), (m, root), oracle.dither(m.numel(), t), (0.0, 2.0**-9)):
            held, steps = oracle.hold(x, u, least)
            assert torch.equal(after[name + "_scale"], steps), name
            assert torch.equal(after[name].float(), held), name
    master = before.get("master")
    want, _, _ = oracle.step(p0 if master is None else master, g, m0, v0, t, **{"decay" if k == "weight_decay" else k: x
                                                                              for k, x in hyper.items()})
    # float32: m, v and the update's own 6 roundings, v_rcp_f32 and v_sqrt_f32 an ulp each; p (1 - lr decay) and the sum
    start = (p0 if master is None else master).double()
    bound = 2.0**-24 * (3 * start.abs() + 20 * (want - start).abs() + want.abs()) + 1e-30
    if master is not None:
        assert ((after["master"].double() - want).abs() <= bound).all()
        assert torch.equal(after["master"].to(p.dtype), p)
    u, tiny = torch.finfo(p.dtype).eps / 2, torch.finfo(p.dtype).smallest_normal * torch.finfo(p.dtype).eps / 2
    err = (p.double() - want).abs()
    assert (err <= bound + u * (want.abs() + bound) + tiny).all(), err.max()


def _cpu(state):
    return {k: x.detach().cpu().clone() for k, x in state.items()}


@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("master", [False, True], ids=["", "master"])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
def test_steps(dtype, bits, master, offset, device):
    gen = torch.Generator().manual_seed(bits + offset)
    params = _params(gen, dtype, device, offset=offset)
    opt = AdamW(params, **HYPER, state_bits=bits, master_weights=master)
    for t in range(1, 5):
        _grads(gen, params, offset)
        if t == 1:
            before = [{"exp_avg": torch.zeros(p.shape), "exp_avg_sq": torch.zeros(p.shape), "exp_root": torch.zeros(p.shape),
                       "exp_avg_scale": torch.zeros(-(-p.numel() // 256)), "exp_root_scale": torch.zeros(-(-p.numel() // 256)),
                       **({"master": p.detach().cpu().float()} if master and dtype != F32 else {})} for p in params]
        else:
            before = [_cpu(opt.state[p]) for p in params]
        old = [p.detach().cpu().clone() for p in params]
        version = [p._version for p in params]
        opt.step()
        assert all(p._version > v for p, v in zip(params, version))
        for p, p0, s in zip(params, old, before):
            after = _cpu(opt.state[p])
            assert after["step"] == t
            assert ("master" in after) == (master and dtype != F32)
            _check_step(s, after, p0, p.detach().cpu(), p.grad.cpu(), t, bits)


def test_many_tensors(device):
    """More tensors than a launch takes, and than one counts the steps of; some without a gradient."""
    gen = torch.Generator().manual_seed(1)
    params = _params(gen, F32, device, [(1 + i % 37,) for i in range(600)])
    opt = AdamW(params, **HYPER)
    _grads(gen, params)
    for p in params[::5]:
        p.grad = None
    for t in (1, 2):
        before = [(p.detach().cpu().clone(), _cpu(opt.state[p]) if t == 2 and p.grad is not None else
                   {"exp_avg": torch.zeros(p.shape), "exp_avg_sq": torch.zeros(p.shape)}) for p in params]
        opt.step()
        for p, (p0, s) in zip(params, before):
            if p.grad is None:
                assert p not in opt.state and torch.equal(p.detach().cpu(), p0)
            else:
                _check_step(s, _cpu(opt.state[p]), p0, p.detach().cpu(), p.grad.cpu(), t, 32)


def test_groups_scale_and_rate(device):
    """Groups of their own options; the rate and the gradients' scale on the device, a gradient of other strides."""
    gen = torch.Generator().manual_seed(2)
    a, b, c = _params(gen, BF16, device, [(40, 24), (300,), (64,)])
    (d,) = _params(gen, F32, device, [(77,)])
    rate = torch.tensor(2.0**-7, device=device)
    opt = AdamW([{"params": [a, d], "state_bits": 8, "lr": rate, "weight_decay": 0.0}, {"params": [b, c], "master_weights": True}],
                lr=2.0**-8, betas=(0.5, 0.75), eps=0.0, weight_decay=0.5)
    scale = torch.tensor(0.25, device=device)
    for t in (1, 2):
        _grads(gen, [a, b, c, d])
        a.grad = torch.randn((24, 40), generator=gen).to(BF16).to(device).T
        params = [a, b, c, d]
        bits = [8, 32, 32, 8]
        zeros = lambda p: {"exp_avg": torch.zeros(p.shape), "exp_avg_sq": torch.zeros(p.shape), "exp_root": torch.zeros(p.shape),
                           "exp_avg_scale": torch.zeros(-(-p.numel() // 256)), "exp_root_scale": torch.zeros(-(-p.numel() // 256)),
                           **({"master": p.detach().cpu().float()} if p is b or p is c else {})}
        before = [(p.detach().cpu().clone(), zeros(p) if t == 1 else _cpu(opt.state[p])) for p in params]
        opt.step(grad_scale=scale)
        for p, (p0, s), n in zip(params, before, bits):
            hyper = dict(lr=2.0**-7 if n == 8 else 2.0**-8, betas=(0.5, 0.75), eps=0.0, weight_decay=0.0 if n == 8 else 0.5)
            _check_step(s, _cpu(opt.state[p]), p0, p.detach().cpu(), p.grad.cpu().float() * 0.25, t, n, hyper)
        rate.fill_(2.0**-7)


@pytest.mark.parametrize("bits", [8, 32])
def test_state_goes_on_after_loading(bits, device):
    gen = torch.Generator().manual_seed(4)
    params = _params(gen, BF16, device)
    opt = AdamW(params, **HYPER, state_bits=bits, master_weights=True)
    for _ in range(2):
        _grads(gen, params)
        opt.step()
    twins = [p.detach().clone().requires_grad_() for p in params]
    other = AdamW(twins, state_bits=bits, master_weights=True)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    _grads(gen, params)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        assert all(torch.equal(x.float(), other.state[q][n].float()) for n, x in opt.state[p].items())


def test_weights_and_states_that_move(device):
    """A step follows weights and states that were put elsewhere since the last one."""
    gen = torch.Generator().manual_seed(6)
    (p,) = _params(gen, F32, device, [(500,)])
    opt = AdamW([p], **HYPER)
    _grads(gen, [p])
    opt.step()
    p.data = p.data.clone()
    opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"] * 2
    before, p0 = _cpu(opt.state[p]), p.detach().cpu().clone()
    opt.step()
    _check_step(before, _cpu(opt.state[p]), p0, p.detach().cpu(), p.grad.cpu(), 2, 32)


@pytest.mark.parametrize("bits", [8, 32])
def test_captured(bits, device):
    """A captured step counts on, reads the rate and the gradients of each replay."""
    gen = torch.Generator().manual_seed(7)
    params = _params(gen, BF16, device)
    twins = [p.detach().clone().requires_grad_() for p in params]
    rate, rate2 = (torch.tensor(1e-2, device=device) for _ in range(2))
    opt = AdamW(params, lr=rate, state_bits=bits, master_weights=True)
    other = AdamW(twins, lr=rate2, state_bits=bits, master_weights=True)

    def grads():
        for p, q in zip(params, twins):
            if p.grad is None:
                p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
            p.grad.copy_(torch.randn(p.shape, generator=gen))
            q.grad.copy_(p.grad)

    grads()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="states of a captured step"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    other.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        grads()
        rate.fill_(1e-2 / (k + 1))
        rate2.copy_(rate)
        graph.replay()
        other.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q) and opt.state[p]["step"].item() == k + 2
            assert all(torch.equal(x.float(), other.state[q][n].float()) for n, x in opt.state[p].items())


def test_what_is_not_a_number_stays_in_its_block(device):
    gen = torch.Generator().manual_seed(8)
    (p,) = _params(gen, F32, device, [(1024,)])
    opt = AdamW([p], state_bits=8)
    _grads(gen, [p])
    p.grad[300] = float("nan")
    opt.step()
    state = opt.state[p]
    assert state["exp_avg_scale"].isnan().tolist() == [False, True, False, False]
    assert p.isnan().nonzero().tolist() == [[300]]
    assert not oracle.numbers(state["exp_avg"].cpu(), state["exp_avg_scale"].cpu())[512:].isnan().any()


def test_small_numbers_of_a_block(device):
    """A block with numbers far apart: roots above 0 stay above 0, a block of nothing but zeros or of the smallest numbers
    is held as zeros."""
    p = torch.zeros(768, device=device, requires_grad=True)
    p.grad = torch.zeros(768, device=device)
    p.grad[:256] = 1e-6
    p.grad[0] = 1e6
    p.grad[256:512] = 1e-38
    opt = AdamW([p], lr=1e-3, state_bits=8)
    opt.step()
    s = opt.state[p]
    assert (s["exp_root"][:256].float() >= 2.0**-9).all()
    assert s["exp_root_scale"].tolist()[1:] == [0.0, 0.0] and s["exp_avg_scale"].tolist()[1:] == [0.0, 0.0]
    assert not s["exp_root"][256:].float().any() and not s["exp_avg"][256:].float().any()
    assert p.isfinite().all() and (p[512:] == 0).all()


def test_states_in_8_bits_forget(device):
    """Beside a number that stays, those without a gradient fall by sqrt(b2) a step, in the mean: nearest rounding would
    hold them where they are, as a step moves them by 0.05 % of themselves where codes lie 7 to 12 % apart. Over 1000 steps
    (a fall by 39 %) a number goes down some 5 codes, give or take 2.3: 0.2 of itself, the mean of 65280 of them 0.1 %."""
    n = 1 << 16
    gen = torch.Generator().manual_seed(9)
    root = torch.randn(n, generator=gen).abs() + 0.5
    root[::256] = 10.0
    held, steps = oracle.hold(root, torch.full((n,), 0.5), 2.0**-9)
    p = torch.zeros(n, device=device, requires_grad=True)
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), state_bits=8)
    codes = held.to(torch.float8_e4m3fn)
    opt.load_state_dict({"state": {0: {"step": 5.0, "exp_avg": torch.zeros_like(codes.float()).to(codes.dtype), "exp_root": codes,
                                       "exp_avg_scale": torch.zeros_like(steps), "exp_root_scale": steps}},
                         "param_groups": opt.state_dict()["param_groups"]})
    p.grad = torch.zeros(n, device=device)
    p.grad[::256] = 10.0

    def mean():
        r = oracle.numbers(opt.state[p]["exp_root"].cpu(), opt.state[p]["exp_root_scale"].cpu()).double()
        r = r.view(-1, 256)
        assert ((r[:, 0] / 10 - 1).abs() < 1e-3).all()
        return r[:, 1:].mean().item()

    start = mean()
    for _ in range(1000):
        opt.step()
    assert abs(mean() / (start * 0.999**500) - 1) < 0.01


def test_other_stream(device):
    gen = torch.Generator().manual_seed(10)
    params = _params(gen, F32, device)
    twins = [p.detach().clone().requires_grad_() for p in params]
    _grads(gen, params)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    AdamW(params).step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        AdamW(twins).step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(p, q) for p, q in zip(params, twins))


def test_blocks_of_any_size(device):
    """Gradients from 1e-25 to 1e15: at the top the codes' scale leaves float32's full numbers, at the bottom the second moments
    do; another way is taken there."""
    p = torch.zeros(256 * 41, device=device, requires_grad=True)
    gen = torch.Generator().manual_seed(11)
    size = 10.0 ** torch.arange(-25, 16).double()
    g = (torch.randn((41, 256), generator=gen).double() * size[:, None]).float().flatten()
    opt = AdamW([p], **HYPER, state_bits=8)
    for t in (1, 2):
        before, p0 = ({"exp_avg": torch.zeros(p.shape), "exp_root": torch.zeros(p.shape), "exp_avg_scale": torch.zeros(41),
                       "exp_root_scale": torch.zeros(41)} if t == 1 else _cpu(opt.state[p])), p.detach().cpu().clone()
        p.grad = g.to(device)
        opt.step()
        after = _cpu(opt.state[p])
        m0 = oracle.numbers(before["exp_avg"], before["exp_avg_scale"])
        r0 = oracle.numbers(before["exp_root"], before["exp_root_scale"])
        m, v = oracle.moments(g, m0, r0 * r0, HYPER["betas"])
        for name, x, u, least in zip(("exp_avg", "exp_root"), (m, v.double().sqrt().float()), oracle.dither(g.numel(), t), (0.0, 2.0**-9)):
            held, steps = oracle.hold(x, u, least)
            assert torch.equal(after[name + "_scale"], steps), name
            assert torch.equal(after[name].float(), held), name


def test_more_numbers_than_32_bits_count(device):
    """One tensor of more than 2^32 numbers. A first step moves a weight by lr against its gradient's sign; blocks of 256 end
    at multiples of 256, so the last 44 are one of their own."""
    n = (1 << 32) + 300
    p = torch.zeros(n, dtype=BF16, device=device)
    at = torch.tensor([0, 5, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1], device=device)
    p[at] = 1.0
    p.requires_grad_()
    p.grad = torch.zeros_like(p)
    p.grad[at] = torch.tensor([2.0, -2, 2, 2, 2, 2], dtype=BF16, device=device)
    opt = AdamW([p], lr=0.25, betas=(0.5, 0.5), eps=1e-30, weight_decay=0.0, state_bits=8)
    opt.step()
    assert p[at].tolist() == [0.75, 1.25, 0.75, 0.75, 0.75, 0.75]
    state = opt.state[p]
    m = oracle.numbers(state["exp_avg"][-300:].cpu(), state["exp_avg_scale"][-2:].cpu())
    # 448 steps of (max / 448), rounded twice
    assert ((m[[0, -1]] - 1).abs() <= 2.0**-22).all() and not m[1:-1].any()
    assert p[(1 << 32) + 1 : n - 1].eq(0).all() and p[6:1000].eq(0).all()


@pytest.mark.parametrize("bits,master", [(8, True), (32, False)])
def test_data_put_elsewhere(bits, master, device):
    """A step follows states whose `data` was exchanged, and refuses weights and states that do not fit any more."""
    gen = torch.Generator().manual_seed(9)
    (p,) = _params(gen, BF16, device, [(32, 32)])
    opt = AdamW([p], **HYPER, state_bits=bits, master_weights=master)
    _grads(gen, [p])
    opt.step()
    state, old = opt.state[p], {}
    for name, x in state.items():
        old[name] = x.data
        x.data = x.data.clone()
    before, p0, kept = _cpu(state), p.detach().cpu().clone(), _cpu(old)
    opt.step()
    _check_step(before, _cpu(state), p0, p.detach().cpu(), p.grad.cpu(), 2, bits)
    assert all(torch.equal(x.cpu().float(), kept[n].float()) for n, x in old.items())
    whole = p.data
    p.grad, p.data = None, whole[:8]
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="has to be 1024 contiguous|has to be 256 contiguous|has to be 1 contiguous"):
        opt.step()
    p.grad, p.data = None, whole.t()
    p.grad = torch.ones_like(p)
    with pytest.raises(NotImplementedError, match="contiguous"):
        opt.step()
    p.grad, p.data = None, whole
    p.grad = torch.ones_like(p)
    opt.step()
    state["exp_avg"].data = state["exp_avg"].data.cpu()
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()


@pytest.mark.parametrize("how", ["clear", "another", "one", "put back"])
def test_states_taken_away(how, device):
    """A step begins anew where a state is gone, and uses the one that is put in its place."""
    gen = torch.Generator().manual_seed(10)
    params = _params(gen, F32, device, [(300,), (20,)])
    opt = AdamW(params, **HYPER)
    _grads(gen, params)
    opt.step()
    held = copy.deepcopy([opt.state[p] for p in params])
    opt.step()
    if how == "clear":
        opt.state.clear()
    elif how == "another":
        opt.state = type(opt.state)(dict)
    elif how == "one":
        del opt.state[params[1]]
    else:
        for p, s in zip(params, held):
            opt.state[p] = s
    gone = {"clear": [0, 1], "another": [0, 1], "one": [1], "put back": []}[how]
    before = [{k: torch.zeros_like(x) for k, x in _cpu(s).items()} if i in gone else
              _cpu(s if how == "put back" else opt.state[params[i]]) for i, s in enumerate(held)]
    p0 = [p.detach().cpu().clone() for p in params]
    opt.step()
    for i, p in enumerate(params):
        t = 1 if i in gone else 2 if how == "put back" else 3
        assert opt.state[p]["step"].item() == t
        _check_step(before[i], _cpu(opt.state[p]), p0[i], p.detach().cpu(), p.grad.cpu(), t, 32)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_weight_viewed_as_another_type(bits, device):
    """The same memory as the other type of 16 bits between two steps."""
    gen = torch.Generator().manual_seed(12)
    (p,) = _params(gen, BF16, device, [(40, 50)])
    opt = AdamW([p], **HYPER, state_bits=bits)
    for _ in range(2):
        _grads(gen, [p])
        opt.step()
    p.grad, p.data = None, p.data.view(F16)
    _grads(gen, [p])
    before, p0 = _cpu(opt.state[p]), p.detach().cpu().clone()
    opt.step()
    assert p.dtype == F16 and p0.isfinite().all()
    _check_step(before, _cpu(opt.state[p]), p0, p.detach().cpu(), p.grad.cpu(), 3, bits)


def test_a_gradient_moved_to_the_host(device):
    """torch lets a gradient's data be exchanged for one elsewhere: refused before anything runs."""
    gen = torch.Generator().manual_seed(13)
    params = _params(gen, F32, device, [(40,), (7,)])
    opt = AdamW(params, **HYPER)
    for _ in range(2):
        _grads(gen, params)
        opt.step()
    _grads(gen, params)
    params[1].grad.data = params[1].grad.data.cpu()
    held = copy.deepcopy([p.detach() for p in params]), [_cpu(opt.state[p]) for p in params]
    with pytest.raises(ValueError, match="on cpu of a parameter"):
        opt.step()
    for p, p0, s in zip(params, *held):
        assert torch.equal(p, p0) and all(torch.equal(x, s[n]) for n, x in _cpu(opt.state[p]).items())
