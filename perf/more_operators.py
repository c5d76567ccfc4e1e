"""What the operators of a feed-forward half with biases and dropout cost.

Four kinds of pass:

* ``linear``: one forward of a product with bias, activation, dropout and residual
  in its epilogue (``streamk.linear``), as a model is served or run for its logits.
* ``linear_train``: that forward, and its backward pass down to the gradients of
  the input, the weights, the bias and the residual.
* ``dropout``: dropout by a counter-based generator, alone or with the residual's
  addition (``feedforward.dropout``).
* ``dropout_train``: that forward, and its backward pass, which makes the mask again.

Where ``own`` is false the same passes are elementary torch operations in 32
bits, rounded once at the end.

The mask of both: element i of the result in row-major order is dropped where its 16
random bits are below T = round(65536 p), and what is kept is multiplied by 65536 /
(65536 - T).  The bits are half i % 2 (the low one first) of word i % 8 // 2 of
Philox4x32 (Salmon, Moraes, Dror and Shaw, SC 2011) of seven rounds, with the seed's
low and high words as key and the counter (low and high words of i // 8, site, 0).
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _framework():
    """The modules of the package, whose folder is no identifier."""
    path = os.path.join(os.path.abspath(os.getcwd()), "awesome-cute_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import feedforward
    import streamk
    return streamk, feedforward


# --- the cases -----------------------------------------------------------------------------

def _linear(m, n, k, type, act="none", bias=True, residual=False, p=0.0, train=False, name=None):
    return _named(name, kind="linear_train" if train else "linear", m=m, n=n, k=k, type=type, act=act, bias=bias,
                  residual=residual, p=p)


def _dropout(rows, d, type, p, residual=False, train=False, name=None):
    return _named(name, kind="dropout_train" if train else "dropout", rows=rows, d=d, type=type, p=p,
                  residual=residual)


def _named(name, **case):
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # the embeddings of a short sequence, in training: what a call costs by itself
        _dropout(64, 1024, "bf16", 0.1, name="dropout_short"),
        # a batch of long sequences after a sublayer, added to the residual
        _dropout(16384, 4096, "bf16", 0.1, residual=True, name="dropout_residual"),
        # the inner activations of a training step, forward and backward
        _dropout(2048, 10752, "bf16", 0.1, train=True, name="dropout_train"),
        # a small model in 32 bits on a ragged batch, rows that no piece divides
        _dropout(1237, 1033, "fp32", 0.25, residual=True, train=True, name="dropout_train_ragged"),
        # one token through the up projection of a 7B model without a gate
        _linear(1, 10752, 4096, "fp16", "gelu", name="linear_token"),
        # an uneven decoding batch through a 13B model's down projection, onto the residual
        _linear(45, 5120, 13568, "bf16", residual=True, name="linear_batch"),
        # a chunk of a prompt: rows and columns that no tile divides
        _linear(777, 5208, 4160, "fp16", "silu", name="linear_chunk"),
        # a prompt of 2048 tokens
        _linear(2048, 10752, 4096, "bf16", "gelu", name="linear_prompt"),
        # a batch of prompts through a square projection, onto the residual
        _linear(8192, 4096, 4096, "bf16", residual=True, name="linear_prompts"),
        # a training step of 2048 tokens through a 7B model's up projection ...
        _linear(2048, 10752, 4096, "bf16", "gelu", train=True, name="linear_train_up"),
        # ... and its down projection, with dropout before the residual's addition
        _linear(2048, 4096, 10752, "bf16", residual=True, p=0.1, train=True, name="linear_train_down"),
        # a small model's step on a ragged batch, with all there is
        _linear(1237, 2744, 1032, "fp16", "silu", residual=True, p=0.2, train=True, name="linear_train_ragged"),
    ]


MOST_FLOPS = 6 * 2048 * 10752 * 4096


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return int(round(lo * (hi / lo) ** rng.random()))


def _step(rng, lo, hi, step):
    return max(lo, min(hi, step * round(_log(rng, lo, hi) / step)))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_train", "linear_train", "dropout", "dropout_train"])
    p = rng.choice([0.05, 0.1, 0.1, 0.2, 0.5])
    if kind in ("dropout", "dropout_train"):
        type = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        rows, d = _log(rng, 1, 16384), _log(rng, 64, 16384)
        d = d if rng.random() < 0.3 else max(64, 8 * round(d / 8))
        while rows * d > 16384 * 4096:
            rows = (rows + 1) // 2
        return _dropout(rows, d, type, p, rng.random() < 0.5, kind == "dropout_train")
    type = rng.choice(["fp16", "bf16"])
    act = rng.choice(["none", "silu", "gelu", "gelu"])
    residual = rng.random() < 0.5
    train = kind == "linear_train"
    p = p if train and rng.random() < 0.5 else 0.0
    bias = rng.random() < 0.75 or not (residual or p or act != "none")
    m = _log(rng, 1, 8192)
    n, k = _step(rng, 64, 14336, 8), _step(rng, 64, 11008, 8)
    while (6 if train else 2) * m * n * k > MOST_FLOPS:
        m = (m + 1) // 2
    return _linear(m, n, k, type, act, bias, residual, p, train)


# --- inputs --------------------------------------------------------------------------------

def _inputs(case, seed):
    """Activations and residuals N(0, 1), weights such that sums are about one, biases
    N(0, 0.2), gradients N(0, 0.01)."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    type = TYPES[case["type"]]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device=DEV, generator=gen) * std).to(type)

    kind = case["kind"]
    inputs = {}
    if kind in ("dropout", "dropout_train"):
        shape = (case["rows"], case["d"])
        inputs["x"] = randn(*shape)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        shape = (m, n)
        inputs["x"], inputs["w"] = randn(m, k), randn(n, k, std=k ** -0.5)
        if case["bias"]:
            inputs["bias"] = randn(n, std=0.2)
    if case["residual"]:
        inputs["residual"] = randn(*shape)
    if kind.endswith("_train"):
        inputs["dy"] = randn(*shape, std=0.01)
    return inputs


def _mask_inputs(case, seed):
    """The seed of the mask, any 63 bits, and which of a step's masks it is."""
    return (seed * 6364136223846793005 + 1442695040888963407) % 2 ** 63, seed % 7


def prepare(case, seed):
    state = _inputs(case, seed)
    state["names"] = [name for name in ("x", "w", "bias", "residual") if name in state]
    state["kind"], state["p"] = case["kind"], case["p"]
    state["act"] = case.get("act", "none")
    state["seed"], state["site"] = _mask_inputs(case, seed)
    if not own:
        return state
    state["streamk"], state["feedforward"] = _framework()
    if case["kind"].endswith("_train"):
        # a training step that may be captured keeps its seed on the GPU
        state["seed"] = torch.tensor([state["seed"]], dtype=torch.int64, device=DEV)
        for name in state["names"]:
            state[name].requires_grad_()
    return state


# --- one pass ------------------------------------------------------------------------------

def run(state):
    return _call(state) if own else _plain(state)


def _call(state):
    if state["kind"] in ("dropout", "dropout_train"):
        y = state["feedforward"].dropout(state["x"], state["p"], state["seed"], site=state["site"],
                                         residual=state.get("residual"))
    else:
        act = state["act"]
        y = state["streamk"].linear(state["x"], state["w"], state.get("bias"), None if act == "none" else act,
                                    state.get("residual"), dropout=state["p"],
                                    seed=state["seed"] if state["p"] else None, site=state["site"])
    if not state["kind"].endswith("_train"):
        return {"y": y}
    names = state["names"]
    grads = torch.autograd.grad(y, [state[name] for name in names], state["dy"])
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(names, grads)}}


LOW = 0xffffffff


def _philox(c0, c1, c2, key):
    """Seven rounds on the counters (c0, c1, c2, 0), words in 64-bit integers."""
    k0, k1 = key & LOW, key >> 32 & LOW
    c3 = torch.zeros_like(c0)
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (modulo 2^64)
        c0, c1, c2, c3 = (b >> 32 & LOW) ^ c1 ^ k0, b & LOW, (a >> 32 & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = k0 + 0x9E3779B9 & LOW, k1 + 0xBB67AE85 & LOW
    return torch.stack([c0, c1, c2, c3], dim=1)


def _kept(state, shape):
    """Truth values of `shape`, and the factor of what is kept."""
    below = round(65536 * state["p"])
    count = math.prod(shape)
    group = torch.arange((count + 7) // 8, device=DEV, dtype=torch.int64)
    words = _philox(group & LOW, group >> 32, torch.full_like(group, state["site"]), state["seed"])
    bits = torch.stack([words & 0xffff, words >> 16], dim=2).view(-1)[:count]
    return (bits >= below).view(shape), 65536 / (65536 - below)


def _activation(z, act):
    """act(z) and its derivative"""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-2 * c * (z + 0.044715 * z * z * z)))
        return z * s, s + z * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * z * z)
    return z, None


def _plain(state):
    kind, p = state["kind"], state["p"]
    type = state["x"].dtype
    x = state["x"].float()
    zero = torch.zeros((), device=DEV)
    train = kind.endswith("_train")
    dy = state["dy"].float() if train else None
    if kind in ("dropout", "dropout_train"):
        kept, factor = _kept(state, x.shape)
        y = torch.where(kept, x * factor, zero)
        if "residual" in state:
            y = state["residual"].float() + y
        out = {"y": y.to(type)}
        if train:
            out["dx"] = torch.where(kept, dy * factor, zero).to(type)
    else:
        w = state["w"].float()
        z = x @ w.t()
        if "bias" in state:
            z = z + state["bias"].float()
        y, slope = _activation(z, state["act"])
        if p:
            kept, factor = _kept(state, y.shape)
            y = torch.where(kept, y * factor, zero)
        if "residual" in state:
            y = state["residual"].float() + y
        out = {"y": y.to(type)}
        if train:
            dz = dy
            if p:
                dz = torch.where(kept, dz * factor, zero)
            if slope is not None:
                dz = dz * slope
            out["dx"], out["dw"] = (dz @ w).to(type), (dz.t() @ x).to(type)
            if "bias" in state:
                out["dbias"] = dz.sum(0).to(type)
    if train and "residual" in state:
        out["dresidual"] = state["dy"].clone()
    return out


def _times(a, b):
    """High and low words of the product of words: by halves, so that nothing passes 2^63."""
    b0, b1 = b & 0xffff, b >> 16
    low = a * b0                              # below 2^48
    middle = a * b1 + (low >> 16)             # below 2^49
    return middle >> 16, (middle & 0xffff) << 16 | low & 0xffff


def exact(case, seed):
    """The outputs in 64 bits, from the definitions; the generator by halves of words, element by
    element."""
    data = {name: t.double() for name, t in _inputs(case, seed).items()}
    key, site = _mask_inputs(case, seed)
    train = case["kind"].endswith("_train")
    is_linear = "m" in case
    shape = (case["m"], case["n"]) if is_linear else (case["rows"], case["d"])
    factor = None
    if case["p"]:
        groups = (shape[0] * shape[1] + 7) // 8
        word = torch.zeros((4, groups), dtype=torch.int64, device=DEV)
        at = torch.arange(groups, device=DEV)
        word[0], word[1], word[2] = at % 2 ** 32, at // 2 ** 32, site
        for r in range(7):
            k0, k1 = (key + r * 0x9E3779B9) % 2 ** 32, (key // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32
            (h0, l0), (h1, l1) = _times(word[0], 0xD2511F53), _times(word[2], 0xCD9E8D57)
            word = torch.stack([h1 ^ word[1] ^ k0, l1, h0 ^ word[3] ^ k1, l0])
        drop_below = int(case["p"] * 65536 + 0.5)
        random = torch.empty((groups, 8), dtype=torch.int64, device=DEV)
        for e in range(8):
            random[:, e] = word[e // 2] // 65536 ** (e % 2) % 65536
        keep = random.view(-1)[:shape[0] * shape[1]].view(shape) >= drop_below
        factor = keep.double() / (1 - drop_below / 65536)
    slope = None
    if is_linear:
        value = data["x"] @ data["w"].t()
        if case["bias"]:
            value = value + data["bias"]
        if case["act"] == "silu":
            s = torch.sigmoid(value)
            slope = s + value * s * (1 - s)
            value = value * s
        elif case["act"] == "gelu":
            t = torch.tanh(math.sqrt(2 / math.pi) * (value + 0.044715 * value ** 3))
            slope = (1 + t) / 2 + value / 2 * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * value * value)
            value = value / 2 * (1 + t)
    else:
        value = data["x"]
    if factor is not None:
        value = value * factor
    out = {"y": value + data["residual"] if case["residual"] else value}
    if train:
        d = data["dy"]
        for part in (factor, slope):
            if part is not None:
                d = d * part
        if is_linear:
            out["dx"], out["dw"] = d @ data["w"], d.t() @ data["x"]
            if case["bias"]:
                out["dbias"] = d.sum(0)
        else:
            out["dx"] = d
        if case["residual"]:
            out["dresidual"] = data["dy"]
    return out


def work(case):
    train = case["kind"].endswith("_train")
    if "rows" in case:
        size = 4 if case["type"] == "fp32" else 2
        # x and y, the residual, dy and dx (the residual's gradient is dy itself)
        count = case["rows"] * case["d"]
        return {"bytes": float(size * count * (2 + case["residual"] + 2 * train)), "flops": float(count * (2 + train))}
    m, n, k = case["m"], case["n"], case["k"]
    small = n if case["bias"] else 0
    if not train:
        return {"bytes": float(2 * (m * k + n * k + m * n * (1 + case["residual"]) + small)),
                "flops": float(2 * m * n * k)}
    # x, w, the bias, the residual and dy read, y and the gradients of x, w and the bias written
    return {"bytes": float(2 * (2 * m * k + 2 * n * k + m * n * (2 + case["residual"]) + 2 * small)),
            "flops": float(6 * m * n * k)}
