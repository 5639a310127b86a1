"""Timed cases of a language model's two ends and its update: token embedding, the loss over the vocabulary, AdamW.

listed() names the cases, draw() gives more of the same ranges, prepare() makes
a case's inputs on the GPU from a seed, run() takes one pass: where `own` is
true through the framework's entry points, else through plain torch operations
in 32 bits. exact() computes the same outputs from the definitions in 64 bits
and work() says what a pass cannot do without.

Embedding: out_t = scale W[id_t]; dW_v = scale * the sum of dout_t over the
tokens t with id_t = v; the row of the padding id has no gradient.

Loss: with logits l_jv = <x_j, W_v>, loss_j = log sum_v exp l_jv - l_j,y_j;
tokens of label -100 have none. The mean is over the tokens that have one.

AdamW: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps).
States in 8 bits hold m and r = sqrt(v) as e4m3 numbers times a step for each
256 of a tensor's numbers, step = max / 448. A number a >= 0 (in units of the step,
2^e <= a < 2^(e + 1), e at least -6) becomes floor(a 2^(3 - e) + u) 2^(e - 3),
at most 448, with the dither u = (x >> 12) 2^-20 for m, (x mod 2^20) 2^-20 for r,
x = (2654435761 i + 2246822519 t) mod 2^32 for number i of the tensor in step t;
an r above 0 becomes 2^-9 at least.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORED = -100
BLOCK = 256
TOP = 448.0  # e4m3's largest number
BETAS, EPS, DECAY = (0.9, 0.99), 1e-8, 0.1


def listed():
    return [
        # A training step's loss at the sizes of the small example decoder: latency.
        {"name": "loss_small", "op": "loss", "train": True, "tokens": 2048, "vocab": 64, "dim": 256, "ignored": 0.0,
         "reduction": "mean", "dtype": "bf16"},
        # A few candidate tokens are scored under the benchmark decoder's vocabulary: forward alone.
        {"name": "loss_score", "op": "loss", "train": False, "tokens": 64, "vocab": 151936, "dim": 1024,
         "ignored": 0.0, "reduction": "none", "dtype": "bf16"},
        # One sequence of the benchmark decoder, forward and backward.
        {"name": "loss_sequence", "op": "loss", "train": True, "tokens": 2048, "vocab": 151936, "dim": 1024,
         "ignored": 0.0, "reduction": "mean", "dtype": "bf16"},
        # The benchmark decoder's whole batch, 8 x 2048 tokens.
        {"name": "loss_batch", "op": "loss", "train": True, "tokens": 16384, "vocab": 151936, "dim": 1024,
         "ignored": 0.0, "reduction": "mean", "dtype": "bf16"},
        # Fine-tuning on answers: most prompt tokens have no loss, sizes of no tile, 16-bit floats, weighted tokens.
        {"name": "loss_ragged_f16", "op": "loss", "train": True, "tokens": 3001, "vocab": 32001, "dim": 1000,
         "ignored": 0.4, "reduction": "none", "dtype": "f16"},
        # The next tokens of 64 sequences that decode.
        {"name": "embed_tokens", "op": "embed", "train": False, "tokens": 64, "vocab": 151936, "dim": 1024,
         "scale": 1.0, "padding": None, "wide": True, "dtype": "bf16"},
        # The benchmark decoder's batch, scaled, with the table's gradient.
        {"name": "embed_batch", "op": "embed", "train": True, "tokens": 16384, "vocab": 151936, "dim": 1024,
         "scale": 32.0, "padding": None, "wide": True, "dtype": "bf16"},
        # Rows of no vector's size in 32 bits, 32-bit ids, a padding id.
        {"name": "embed_ragged_f32", "op": "embed", "train": True, "tokens": 5003, "vocab": 32001, "dim": 333,
         "scale": 0.5, "padding": 0, "wide": False, "dtype": "f32"},
        # The small example decoder's tensors: latency.
        {"name": "update_small", "op": "update", "vocab": 64, "hidden": 256, "layers": 2, "bits": 32, "master": False,
         "dtype": "f32"},
        # Half of the benchmark decoder: 16-bit weights with 32-bit masters and states, 127 tensors.
        {"name": "update_stack", "op": "update", "vocab": 151936, "hidden": 1024, "layers": 14, "bits": 32,
         "master": True, "dtype": "bf16"},
        # A memory's value table of 2^20 slots, states in 8 bits.
        {"name": "update_table", "op": "update", "vocab": 1 << 20, "hidden": 1024, "layers": 0, "bits": 8,
         "master": False, "dtype": "bf16"},
        # Tensors of odd sizes, 32-bit weights, states in 8 bits.
        {"name": "update_ragged", "op": "update", "vocab": 1001, "hidden": 333, "layers": 3, "bits": 8,
         "master": False, "dtype": "f32"},
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    top = {}
    for case in listed():
        for n, x in work(case).items():
            top[case["op"], n] = max(x, top.get((case["op"], n), 0))
    while True:
        case = _drawn(rng)
        if all(x <= top[case["op"], n] for n, x in work(case).items()):
            return case


def _drawn(rng):
    op = rng.choice(["loss", "loss", "embed", "update"])
    if op == "update":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        return {"op": op, "vocab": _between(rng, 1, 200000), "hidden": _between(rng, 1, 2048),
                "layers": rng.choice([0, 1, rng.randint(2, 24)]), "bits": rng.choice([8, 32]),
                "master": dtype != "f32" and rng.choice([False, True]), "dtype": dtype}
    case = {"op": op, "train": rng.choice([False, True, True]), "tokens": _between(rng, 1, 16384),
            "vocab": _between(rng, 2, 200000)}
    dim = _between(rng, 16, 4096)
    case["dim"] = rng.choice([dim, -(-dim // 8) * 8, -(-dim // 64) * 64])
    if op == "loss":
        case.update(ignored=rng.choice([0.0, 0.0, 0.1, 0.7]), reduction=rng.choice(["mean", "mean", "sum", "none"]),
                    dtype=rng.choice(["bf16", "bf16", "f16"]))
    else:
        case.update(scale=rng.choice([1.0, round(rng.uniform(0.1, 40.0), 3)]),
                    padding=rng.choice([None, 0, rng.randrange(case["vocab"])]), wide=rng.choice([False, True]),
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    return case


def _shapes(case):
    """The tensors of a decoder's table and layers."""
    H = case["hidden"]
    layer = [(2 * H, H), (H, H), (H, H), (H, 2 * H), (4 * H, H), (H, 4 * H), (H,), (H,), (128,)]
    return [(case["vocab"], H)] + layer * case["layers"]


def _starts(case):
    """Where each tensor begins in the flat buffers, and where the last one ends: whole blocks each."""
    at = [0]
    for s in _shapes(case):
        at.append(at[-1] + -(-math.prod(s) // BLOCK) * BLOCK)
    return at


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _tokens(gen, n, vocab):
    """Token ids as texts have them: the k-th most frequent about 1 / k of the time."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (float(vocab) ** u).long().clamp_(1, vocab) - 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    dtype, state = DTYPES[case["dtype"]], {"case": case}
    if case["op"] == "update":
        return _prepare_update(state, gen, randn, dtype)
    n, V, D = case["tokens"], case["vocab"], case["dim"]
    ids = _tokens(gen, n, V)
    if case["op"] == "embed":
        state["ids"] = ids if case["wide"] else ids.int()
        state["w"] = randn(V, D).mul_(0.02).to(dtype)
        if case["train"]:
            state["dout"] = randn(n, D).to(dtype)
    else:
        w = randn(V, D).mul_(0.64 * D**-0.5)
        # normed hidden states that lean towards their label's row, by 0 to 16 in the logit
        lean = 16 * torch.rand((n, 1), generator=gen, device="cuda")
        x = randn(n, D) + lean * w[ids] / w[ids].square().sum(1, keepdim=True)
        state["x"], state["w"] = x.to(dtype), w.to(dtype)
        hide = torch.rand(n, generator=gen, device="cuda") < case["ignored"]
        state["labels"] = torch.where(hide, IGNORED, ids)
        if case["train"]:
            one = case["reduction"] != "none"
            state["dloss"] = torch.ones((), device="cuda") if one else torch.rand(n, generator=gen, device="cuda")
    if own and case["train"]:
        for name in ("x", "w"):
            if name in state:
                state[name].requires_grad_()
    return state


def _prepare_update(state, gen, randn, dtype):
    case = state["case"]
    shapes, at = _shapes(case), _starts(case)
    sizes = torch.tensor([math.prod(s) for s in shapes], device="cuda")
    blocks = torch.tensor([(b - a) // BLOCK for a, b in zip(at, at[1:])], device="cuda")
    begin = torch.tensor(at[:-1], device="cuda")
    first = torch.arange(at[-1] // BLOCK, device="cuda") * BLOCK - begin.repeat_interleave(blocks)
    end = sizes.repeat_interleave(blocks)
    state["first"] = first  # of each block, its first number's place in its tensor
    there = first[:, None] + torch.arange(BLOCK, device="cuda") < end[:, None]
    flat = lambda x: torch.where(there, x, 0.0)
    spread = torch.exp(randn(there.shape[0], 1))  # gradients of blocks differ in size
    w = flat(randn(*there.shape).mul_(0.02))
    state["p"] = w.to(dtype)
    if case["master"]:
        state["master"] = w
    state["g"] = flat(1e-3 * spread * randn(*there.shape)).to(dtype)
    m = flat(3e-4 * spread * randn(*there.shape))
    r = flat(1e-3 * spread * randn(*there.shape).abs_().add_(0.1))
    state["t"] = 1000
    if case["bits"] == 32:
        state["m"], state["v"] = m, r.square_()
    else:
        state["m"], state["ms"] = _held(m, 0.5, 0.0)
        state["r"], state["rs"] = _held(r, 0.5, 2.0**-9)
    if own:
        from modelos_amd.adamw import AdamW

        cut = lambda x, i: x.view(-1)[at[i] : at[i] + math.prod(shapes[i])].view(shapes[i])
        part = lambda x, i: x[at[i] // BLOCK : at[i + 1] // BLOCK]
        params = [cut(state["p"], i) for i in range(len(shapes))]
        opt = AdamW(params, lr=5e-5, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                    master_weights=case["master"])
        held = opt.state_dict()
        for i, p in enumerate(params):
            p.grad = cut(state["g"], i)
            s = held["state"][i] = {"step": torch.tensor(float(state["t"]), device="cuda"), "exp_avg": cut(state["m"], i)}
            if case["bits"] == 32:
                s["exp_avg_sq"] = cut(state["v"], i)
            else:
                s["exp_root"] = cut(state["r"], i)
                s["exp_avg_scale"], s["exp_root_scale"] = part(state["ms"], i), part(state["rs"], i)
            if case["master"]:
                s["master"] = cut(state["master"], i)
        opt.load_state_dict(held)
        state["opt"] = opt
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return {"loss": _plain_loss, "embed": _plain_embed, "update": _plain_update}[case["op"]](state)
    if case["op"] == "update":
        state["opt"].step()
        return _updated(state)
    if case["op"] == "embed":
        from modelos_amd.token_embedding import token_embedding

        out = token_embedding(state["ids"], state["w"], scale=case["scale"], padding_idx=case["padding"])
        if not case["train"]:
            return out
        return [out.detach(), *torch.autograd.grad(out, state["w"], state["dout"])]
    from modelos_amd.linear_cross_entropy import linear_cross_entropy

    x, w = state["x"], state["w"]
    loss = linear_cross_entropy(x, w, state["labels"], ignore_index=IGNORED, reduction=case["reduction"])
    if not case["train"]:
        return loss
    return [loss.detach(), *torch.autograd.grad(loss, (x, w), state["dloss"])]


def _updated(state):
    return {n: state[n] for n in ("p", "master", "m", "v", "r", "ms", "rs") if n in state}


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_embed(state):
    case, ids, w = state["case"], state["ids"].long(), state["w"]
    out = (w[ids].float() * case["scale"]).to(w.dtype)
    if not case["train"]:
        return out
    dw = torch.zeros(w.shape, device="cuda").index_add_(0, ids, state["dout"].float()).mul_(case["scale"])
    if case["padding"] is not None:
        dw[case["padding"]] = 0
    return [out, dw.to(w.dtype)]


def _plain_loss(state):
    """Pieces of the tokens against the whole vocabulary."""
    case, labels = state["case"], state["labels"]
    x, w = state["x"].float(), state["w"].float()
    live = labels != IGNORED
    y = labels.clamp_min(0)
    count = live.sum().clamp_min(1) if case["reduction"] == "mean" else 1
    losses = torch.empty(x.shape[0], device="cuda")
    if case["train"]:
        weights = torch.where(live, state["dloss"] / count, 0.0)
        dx, dw = torch.empty_like(x), torch.zeros_like(w)
    step = 2048
    for i in range(0, x.shape[0], step):
        xs, ys = x[i : i + step], y[i : i + step, None]
        e = xs @ w.T
        target = e.gather(1, ys)
        top = e.amax(1, keepdim=True)
        e.sub_(top).exp_()
        total = e.sum(1, keepdim=True)
        losses[i : i + step] = (total.log() + (top - target)).squeeze(1)
        if case["train"]:
            e.div_(total).scatter_add_(1, ys, torch.full_like(total, -1.0)).mul_(weights[i : i + step, None])
            dx[i : i + step] = e @ w
            dw.addmm_(e.T, xs)
    losses = torch.where(live, losses, 0.0)
    loss = losses if case["reduction"] == "none" else losses.sum() / count
    if not case["train"]:
        return loss
    return [loss, dx.to(state["x"].dtype), dw.to(state["w"].dtype)]


def _held(x, u, least):
    """x [blocks, 256] in 8 bits: e4m3 numbers of x / step, rounded with the dither u, and steps [blocks]."""
    step = x.abs().amax(1) / TOP
    a = x.abs().double() / torch.where(step > 0, step, 1).double()[:, None]
    e = (torch.frexp(a).exponent - 1).clamp_min(-6)
    n = torch.floor(torch.ldexp(a, 3 - e) + u)
    held = torch.ldexp(n, e - 3).clamp_max(TOP)
    if least:
        held = torch.where(a > 0, held.clamp_min(least), 0.0)
    return torch.where(x < 0, -held, held).to(torch.float8_e4m3fn), step


def _plain_update(state):
    case, lr = state["case"], 5e-5
    state["t"] += 1
    t = state["t"]
    c1, c2 = 1 - BETAS[0] ** t, 1 - BETAS[1] ** t
    g = state["g"].float()
    if case["bits"] == 32:
        m, v = state["m"], state["v"]
        m.mul_(BETAS[0]).add_(g, alpha=1 - BETAS[0])
        v.mul_(BETAS[1]).add_(g * g, alpha=1 - BETAS[1])
    else:
        m = (state["m"].float() * state["ms"][:, None]).mul_(BETAS[0]).add_(g, alpha=1 - BETAS[0])
        v = (state["r"].float() * state["rs"][:, None]).square_().mul_(BETAS[1]).add_(g * g, alpha=1 - BETAS[1])
    root = v.sqrt()
    w = state["master"] if case["master"] else state["p"].float()
    w.mul_(1 - lr * DECAY).sub_(m / (root * c2**-0.5 + EPS), alpha=lr / c1)
    state["p"].copy_(w)
    if case["bits"] == 8:
        i = state["first"][:, None] + torch.arange(BLOCK, device="cuda")
        x = (i * 2654435761 + t * 2246822519) & 0xFFFFFFFF
        for name, values, u, least in (("m", m, x >> 12, 0.0), ("r", root, x & 0xFFFFF, 2.0**-9)):
            held, step = _held(values, u * 2.0**-20, least)
            state[name].copy_(held)
            state[name + "s"].copy_(step)
    return _updated(state)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"loss": _exact_loss, "embed": _exact_embed, "update": _exact_update}[case["op"]](state)


def _exact_embed(state):
    case, ids, w = state["case"], state["ids"].long(), state["w"].detach().double()
    out = w[ids] * case["scale"]
    if not case["train"]:
        return out
    order = torch.argsort(ids)
    rows, counts = torch.unique_consecutive(ids[order], return_counts=True)
    sums = torch.cumsum(state["dout"].double()[order], 0)
    last = torch.cumsum(counts, 0) - 1
    sums = sums[last]
    sums[1:] -= sums[:-1].clone()
    dw = torch.zeros_like(w)
    dw[rows] = sums * case["scale"]
    if case["padding"] is not None:
        dw[case["padding"]] = 0
    return [out, dw]


def _exact_loss(state):
    case, labels = state["case"], state["labels"]
    x, w = state["x"].detach().double(), state["w"].detach().double()
    kept = torch.nonzero(labels != IGNORED).squeeze(1)
    n = x.shape[0]
    scale = 1 / max(1, len(kept)) if case["reduction"] == "mean" else 1.0
    losses = torch.zeros(n, dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for part in kept.split(1024):
        logits = x[part] @ w.T
        log_p = torch.log_softmax(logits, 1)
        rows = torch.arange(len(part), device="cuda")
        losses[part] = -log_p[rows, labels[part]]
        if case["train"]:
            d = log_p.exp()
            d[rows, labels[part]] = torch.expm1(log_p[rows, labels[part]])
            d *= (state["dloss"].double() * scale).expand(n)[part, None]
            dx[part] = d @ w
            dw += d.T @ x[part]
    loss = losses if case["reduction"] == "none" else losses.sum() * scale
    return [loss, dx, dw] if case["train"] else loss


def _exact_update(state):
    case, lr, t = state["case"], 5e-5, state["t"] + 1
    g = state["g"].double()
    if case["bits"] == 32:
        m, v = state["m"].double(), state["v"].double()
    else:
        m = state["m"].double() * state["ms"].double()[:, None]
        v = (state["r"].double() * state["rs"].double()[:, None]) ** 2
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g**2
    w = state["master" if case["master"] else "p"].double()
    p = w - lr * DECAY * w - lr * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
    out = {"p": p, "m": m}
    if case["master"]:
        out["master"] = p
    if case["bits"] == 32:
        out["v"] = v
        return out
    place = (state["first"][:, None] + torch.arange(BLOCK, device="cuda")) % (1 << 32)
    x = (place * 2654435761 % (1 << 32) + t * 2246822519) % (1 << 32)
    for name, values, u in (("m", m, (x // 4096).double() / 1048576), ("r", v.sqrt(), (x % 1048576).double() / 1048576)):
        step = values.abs().amax(1) / TOP
        a = (values / step.clamp_min(1e-300)[:, None]).abs()
        grid = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0**-6))) - 3)  # the numbers' spacing at a
        held = (torch.floor(a / grid + u) * grid).clamp_max(TOP)
        if name == "r":
            held = torch.where(a > 0, held.clamp_min(2.0**-9), 0.0)
        out[name], out[name + "s"] = held * torch.sign(values), step
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "update":
        n = sum(math.prod(s) for s in _shapes(case))
        size = 4 if case["dtype"] == "f32" else 2
        states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        weights = (8 + size) if case["master"] else 2 * size  # with a master the weight itself is only written
        return {"bytes": n * (size + weights + states), "flops": 16 * n}
    n, V, D = case["tokens"], case["vocab"], case["dim"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "embed":
        bytes_ = n * (8 if case["wide"] else 4) + size * D * (min(n, V) + n)
        return {"bytes": bytes_ + (size * D * (n + V) if case["train"] else 0), "flops": (2 if case["train"] else 1) * n * D}
    live = n * (1 - case["ignored"])
    passes = 2 if case["train"] else 1  # read, and written as a gradient
    return {"bytes": passes * size * D * (live + V) + 8 * n, "flops": (6 if case["train"] else 2) * live * V * D}
