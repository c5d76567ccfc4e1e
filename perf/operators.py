"""What the feed-forward half of a decoder block costs, operator by operator.

Five kinds of pass:

* ``gated4``: one forward of a gated projection with 4-bit weights
  (``marlin.GatedLayer``): both projections, the activation and the product.
* ``gated``: the same with dense fp16 or bf16 weights (``streamk.gated``).
* ``gated_train``: that forward, and its backward pass down to the gradients of
  the input and of the weights.
* ``linear_train``: a dense linear layer (``streamk.linear``), forward and
  backward: the down projection of a block that is trained.
* ``norm``, ``norm_train``: the norms after a block and before the next one,
  with the block's gate and the residual's scale
  (``feedforward.residual_norm``), forward, or forward and backward.

Where ``own`` is false the same passes are elementary torch operations in 32
bits, rounded once at the end.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
SCALE = 0.75  # of the residual, as deep stacks use it


def _framework():
    """The modules of the package, whose folder is no identifier."""
    path = os.path.join(os.path.abspath(os.getcwd()), "awesome-cute_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import feedforward
    import marlin
    import streamk
    return marlin, streamk, feedforward


# --- the cases -----------------------------------------------------------------------------

def _gated4(m, n, k, group, act, name=None):
    return _named(name, kind="gated4", m=m, n=n, k=k, group=group, act=act)


def _gated(m, n, k, type, act, name=None):
    return _named(name, kind="gated", m=m, n=n, k=k, type=type, act=act)


def _gated_train(m, n, k, type, act, name=None):
    return _named(name, kind="gated_train", m=m, n=n, k=k, type=type, act=act)


def _linear_train(m, n, k, type, name=None):
    return _named(name, kind="linear_train", m=m, n=n, k=k, type=type)


def _norm(batch, tokens, d, type, gate, train=False, name=None):
    return _named(name, kind="norm_train" if train else "norm", batch=batch, tokens=tokens, d=d, type=type,
                  gate=gate)


def _named(name, **case):
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # one token between two blocks of a 7B model: what a call costs by itself
        _norm(1, 1, 4096, "fp16", "channel", name="norm_token"),
        # a batch of long prompts of a wide model
        _norm(1, 8192, 8192, "bf16", "channel", name="norm_prompt"),
        # a training step of four sequences, each with a gate of its own
        _norm(4, 1024, 4096, "bf16", "sequence", train=True, name="norm_train"),
        # one token through gate and up of a 7B model with 4-bit weights
        _gated4(1, 10752, 4096, 128, "silu", "gated4_token"),
        # an uneven decoding batch of a 13B model, scales per column
        _gated4(45, 13568, 5120, -1, "gelu", "gated4_batch"),
        # a prompt of 2048 tokens
        _gated4(2048, 10752, 4096, 128, "silu", "gated4_prompt"),
        # one token through dense weights, before any are quantised
        _gated(1, 10752, 4096, "fp16", "silu", "gated_token"),
        # a chunk of a prompt: rows and columns that no tile divides
        _gated(777, 5208, 4160, "bf16", "gelu", "gated_chunk"),
        # a training step of 2048 tokens through a 7B model's gate and up
        _gated_train(2048, 10752, 4096, "bf16", "silu", "gated_train"),
        # a small model's step on a ragged batch
        _gated_train(1237, 2744, 1032, "fp16", "gelu", "gated_train_ragged"),
        # the down projection of the first training step ...
        _linear_train(2048, 4096, 10752, "bf16", "linear_train"),
        # ... and of the second
        _linear_train(1237, 1032, 2744, "fp16", "linear_train_ragged"),
    ]


MOST_FLOPS = 12 * 2048 * 10752 * 4096


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def _step(rng, lo, hi, step):
    return max(lo, min(hi, step * round(_log(rng, lo, hi) / step)))


def draw(rng):
    kind = rng.choice(["gated4", "gated4", "gated", "gated", "gated_train", "linear_train", "norm", "norm_train"])
    type = rng.choice(["fp16", "bf16"])
    act = rng.choice(["silu", "gelu"])
    if kind in ("norm", "norm_train"):
        type = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        batch, tokens = _log(rng, 1, 16), _log(rng, 1, 4096)
        d = _log(rng, 64, 16384)
        d = d if rng.random() < 0.2 else max(64, 8 * round(d / 8))
        while batch * tokens * d > 8192 * 8192:
            tokens = (tokens + 1) // 2
        gate = rng.choice(["none", "channel", "sequence"])
        return _norm(batch, tokens, d, type, gate, kind == "norm_train")
    if kind == "gated4":
        return _gated4(_log(rng, 1, 2048), _step(rng, 128, 14336, 128), _step(rng, 256, 8192, 128),
                       rng.choice([128, 128, -1]), act)
    if kind == "gated":
        m, n, k = _log(rng, 1, 4096), _step(rng, 64, 14336, 8), _step(rng, 64, 8192, 8)
        while 4 * m * n * k > MOST_FLOPS:
            m = (m + 1) // 2
        return _gated(m, n, k, type, act)
    m = _log(rng, 1, 8192)
    n, k = _step(rng, 64, 11008, 8), _step(rng, 64, 8192, 8)
    while 12 * m * n * k > MOST_FLOPS:
        m = (m + 1) // 2
    return _gated_train(m, n, k, type, act) if kind == "gated_train" else _linear_train(m, n, k, type)


# --- inputs --------------------------------------------------------------------------------

def _inputs(case, seed):
    """Activations N(0, 1), 4-bit weights uniform with scales U(0.001, 0.02), dense weights
    N(0, 0.02), norms' weights and gates near one, gradients N(0, 0.01)."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def randn(*shape, type, std=1.0, mean=0.0):
        return (torch.randn(shape, device=DEV, generator=gen) * std + mean).to(type)

    kind = case["kind"]
    if kind == "gated4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = 1 if case["group"] == -1 else k // case["group"]
        return {"x": randn(m, k, type=torch.float16),
                "q": torch.randint(0, 16, (k, 2 * n), dtype=torch.uint8, device=DEV, generator=gen),
                "s": (torch.rand((groups, 2 * n), device=DEV, generator=gen) * 0.019 + 0.001).half()}
    type = TYPES[case["type"]]
    if kind in ("gated", "gated_train", "linear_train"):
        m, n, k = case["m"], case["n"], case["k"]
        inputs = {"x": randn(m, k, type=type),
                  "w": randn(n if kind == "linear_train" else 2 * n, k, type=type, std=0.02)}
        if kind != "gated":
            inputs["dy"] = randn(m, n, type=type, std=0.01)
        return inputs
    batch, tokens, d = case["batch"], case["tokens"], case["d"]
    inputs = {"block": randn(batch, tokens, d, type=type), "residual": randn(batch, tokens, d, type=type),
              "post": randn(d, type=type, std=0.1, mean=1.0), "pre": randn(d, type=type, std=0.1, mean=1.0),
              "gate": None}
    if case["gate"] == "channel":
        inputs["gate"] = randn(d, type=type, std=0.2, mean=0.5)
    elif case["gate"] == "sequence":
        inputs["gate"] = randn(batch, 1, d, type=type, std=0.2, mean=0.5)
    if kind == "norm_train":
        inputs["dy"] = randn(batch, tokens, d, type=type, std=0.01)
        inputs["dr"] = randn(batch, tokens, d, type=type, std=0.01)
    return inputs


def prepare(case, seed):
    state = _inputs(case, seed)
    state["kind"] = case["kind"]
    state["act"] = case.get("act")
    state["group"] = case.get("group")
    if not own:
        return state
    marlin, streamk, feedforward = _framework()
    state["streamk"], state["feedforward"] = streamk, feedforward
    if case["kind"] == "gated4":
        # a model is packed once, from weights that lie on the quantised grid
        n, k = case["n"], case["k"]
        q, s = state.pop("q"), state.pop("s")
        full = s.repeat_interleave(k // s.shape[0], dim=0)
        fake = ((q.half() - 8) * full).t().contiguous()
        layer = marlin.GatedLayer(k, n, case["group"], case["act"]).to(DEV)
        halves = []
        for part in (slice(0, n), slice(n, 2 * n)):
            linear = torch.nn.Linear(1, 1, bias=False)
            linear.weight = torch.nn.Parameter(fake[part].contiguous(), requires_grad=False)
            halves.append((linear, s[:, part].t().contiguous()))
        layer.pack(halves[0][0], halves[1][0], halves[0][1], halves[1][1])
        state["layer"] = layer
    elif case["kind"] in ("gated_train", "linear_train"):
        state["x"].requires_grad_()
        state["w"].requires_grad_()
    elif case["kind"] == "norm_train":
        for name in ("block", "residual", "post", "pre", "gate"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# --- one pass ------------------------------------------------------------------------------

def run(state):
    return _call(state) if own else _plain(state)


def _call(state):
    kind = state["kind"]
    if kind == "gated4":
        return state["layer"](state["x"])
    if kind == "gated":
        return state["streamk"].gated(state["x"], state["w"], state["act"])
    if kind == "gated_train":
        h = state["streamk"].gated(state["x"], state["w"], state["act"])
        dx, dw = torch.autograd.grad(h, (state["x"], state["w"]), state["dy"])
        return {"h": h.detach(), "dx": dx, "dw": dw}
    if kind == "linear_train":
        y = state["streamk"].linear(state["x"], state["w"])
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y, r = state["feedforward"].residual_norm(
        state["residual"], state["block"], post_weight=state["post"], gate=state["gate"], scale=SCALE,
        pre_weight=state["pre"], eps=EPS)
    if kind == "norm":
        return {"y": y, "r": r}
    names = [name for name in ("block", "residual", "post", "pre", "gate") if state[name] is not None]
    grads = torch.autograd.grad((y, r), [state[name] for name in names], (state["dy"], state["dr"]))
    return {"y": y.detach(), "r": r.detach(), **{"d" + name: g for name, g in zip(names, grads)}}


def _activation(g, act):
    """act(g) and its derivative"""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    s = 1 / (1 + torch.exp(-2 * c * (g + 0.044715 * g * g * g)))
    return g * s, s + g * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * g * g)


def _plain(state):
    kind = state["kind"]
    if kind == "gated4":
        q, s = state["q"], state["s"]
        w = (q.float() - 8) * s.float().repeat_interleave(q.shape[0] // s.shape[0], dim=0)
        gu = state["x"].float() @ w
        n = gu.shape[1] // 2
        return (_activation(gu[:, :n], state["act"])[0] * gu[:, n:]).half()
    if kind in ("gated", "gated_train"):
        x, w = state["x"].float(), state["w"].float()
        gu = x @ w.t()
        n = gu.shape[1] // 2
        g, u = gu[:, :n], gu[:, n:]
        value, slope = _activation(g, state["act"])
        type = state["x"].dtype
        if kind == "gated":
            return (value * u).to(type)
        dh = state["dy"].float()
        dgu = torch.cat([dh * u * slope, dh * value], dim=1)
        return {"h": (value * u).to(type), "dx": (dgu @ w).to(type), "dw": (dgu.t() @ x).to(type)}
    if kind == "linear_train":
        type = state["x"].dtype
        x, w, dy = state["x"].float(), state["w"].float(), state["dy"].float()
        return {"y": (x @ w.t()).to(type), "dx": (dy @ w).to(type), "dw": (dy.t() @ x).to(type)}
    type = state["block"].dtype
    b, r0, post, pre = (state[name].float() for name in ("block", "residual", "post", "pre"))
    gate = 1.0 if state["gate"] is None else state["gate"].float()
    rstd1 = torch.rsqrt((b * b).mean(-1, keepdim=True) + EPS)
    bh = b * rstd1
    r = SCALE * r0 + gate * (bh * post)
    rstd2 = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    rh = r * rstd2
    out = {"y": (rh * pre).to(type), "r": r.to(type)}
    if kind == "norm":
        return out
    dy = state["dy"].float()
    d = dy * pre
    dt = state["dr"].float() + rstd2 * (d - rh * (d * rh).mean(-1, keepdim=True))
    d = dt * gate * post
    out["dblock"] = (rstd1 * (d - bh * (d * bh).mean(-1, keepdim=True))).to(type)
    out["dresidual"] = (SCALE * dt).to(type)
    out["dpost"] = (dt * gate * bh).sum((0, 1)).to(type)
    out["dpre"] = (dy * rh).sum((0, 1)).to(type)
    if state["gate"] is not None:
        dgate = dt * bh * post
        out["dgate"] = (dgate.sum((0, 1)) if gate.dim() == 1 else dgate.sum(1, keepdim=True)).to(type)
    return out


def exact(case, seed):
    """The outputs in 64 bits, from the definitions: products with the weights as they are
    stored, x / (1 + exp(-x)) and x / 2 (1 + tanh ...), gradients by the chain rule."""
    data = {name: None if t is None else t.double() for name, t in _inputs(case, seed).items()}
    kind = case["kind"]

    def act(g):
        if case["act"] == "silu":
            s = torch.sigmoid(g)
            return g * s, s + g * s * (1 - s)
        z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        t = torch.tanh(z)
        return g / 2 * (1 + t), (1 + t) / 2 + g / 2 * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)

    if kind == "gated4":
        k, n = case["k"], case["n"]
        per = k // data["s"].shape[0]
        w = ((data["q"] - 8).view(-1, per, 2 * n) * data["s"].unsqueeze(1)).view(k, 2 * n)
        return act(data["x"] @ w[:, :n])[0] * (data["x"] @ w[:, n:])
    if kind in ("gated", "gated_train"):
        n = case["n"]
        wg, wu = data["w"][:n], data["w"][n:]
        g, u = data["x"] @ wg.t(), data["x"] @ wu.t()
        value, slope = act(g)
        if kind == "gated":
            return value * u
        dg, du = data["dy"] * u * slope, data["dy"] * value
        return {"h": value * u, "dx": dg @ wg + du @ wu,
                "dw": torch.cat([dg.t() @ data["x"], du.t() @ data["x"]])}
    if kind == "linear_train":
        return {"y": data["x"] @ data["w"].t(), "dx": data["dy"] @ data["w"], "dw": data["dy"].t() @ data["x"]}
    d = case["d"]
    b, gate = data["block"], data["gate"]
    n1 = ((b ** 2).sum(-1, keepdim=True) / d + EPS) ** 0.5
    p = b / n1 * data["post"]
    r = SCALE * data["residual"] + (p if gate is None else gate * p)
    n2 = ((r ** 2).sum(-1, keepdim=True) / d + EPS) ** 0.5
    out = {"y": r / n2 * data["pre"], "r": r}
    if kind == "norm":
        return out
    # v / n with n^2 = v.v / d + eps:  dv = dz / n - v (dz . v) / (d n^3)
    dz = data["dy"] * data["pre"]
    dr = data["dr"] + dz / n2 - r * (dz * r).sum(-1, keepdim=True) / (d * n2 ** 3)
    dp = dr if gate is None else dr * gate
    dz = dp * data["post"]
    out["dblock"] = dz / n1 - b * (dz * b).sum(-1, keepdim=True) / (d * n1 ** 3)
    out["dresidual"] = SCALE * dr
    out["dpost"] = (dp * b / n1).sum((0, 1))
    out["dpre"] = (data["dy"] * r / n2).sum((0, 1))
    if gate is not None:
        out["dgate"] = (dr * p).sum((0, 1)) if gate.dim() == 1 else (dr * p).sum(1, keepdim=True)
    return out


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_train"):
        rows, d = case["batch"] * case["tokens"], case["d"]
        size = 4 if case["type"] == "fp32" else 2
        gates = {"none": 0, "channel": 1, "sequence": case["batch"]}[case["gate"]]
        big = 4 if kind == "norm" else 8  # block, residual, r, y; dy, dr, dblock, dresidual
        small = (2 + gates) * (1 if kind == "norm" else 2)
        return {"bytes": float(size * d * (big * rows + small)), "flops": float(rows * d * (10 if kind == "norm" else 35))}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "gated4":
        groups = 1 if case["group"] == -1 else k // case["group"]
        return {"bytes": float(n * k + 4 * groups * n + 2 * m * (n + k)), "flops": float(4 * m * n * k)}
    if kind == "gated":
        return {"bytes": float(2 * (m * k + 2 * n * k + m * n)), "flops": float(4 * m * n * k)}
    w = n * k * (2 if kind == "gated_train" else 1)
    # x, w, dy read, the output and the gradients of x and w written
    return {"bytes": float(2 * (2 * m * k + 2 * w + 2 * m * n)), "flops": float(6 * m * w)}
