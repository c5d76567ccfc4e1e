"""The feed-forward half of a decoder block: the norms around it, dropout, and the block as a module,
gated, dense and trained (`FeedForward`) or with 4-bit weights (`QuantizedFeedForward`), or without a
gate (`Mlp`).  The kernels of norms and dropout are in the HIP library (include/feedforward_amd.h),
the products those of `streamk` and `marlin`; no reference counterpart."""
import torch
import torch.nn as nn

import marlin
import streamk
from native import seed_parts as _seed_parts, torch_binding as _torch_binding


def residual_norm(residual, block=None, *, post_weight=None, gate=None, scale=1.0, pre_weight=None, eps=1e-6):
    """The norm after a block, its gate, the residual's scale and the norm before the next block in
    one launch: with rms(v) = v / sqrt(mean(v^2) + eps) over the last dimension,

        r = scale * residual + gate * rms(block) * post_weight,    y = rms(r) * pre_weight

    Returns (y, r).  Without `post_weight` the block is taken as it is, without `gate` the gate is 1,
    without `pre_weight` y is None; without a block (then without post_weight and gate, and whatever
    the scale) r is the residual itself.

    residual, block: (..., d), d up to 16384, torch.half, torch.bfloat16 or torch.float, weights and
    gate of that type as well.  gate: (d,), or the residual's shape with ones for its last dimensions
    but d -- (batch, 1, d): a gate for each sequence.  Inside fp32, r and y rounded once.
    Differentiable once, on the current stream of the residual's device; sums over rows are added in
    a fixed order."""
    scale, eps = float(scale), float(eps)
    if not torch.compiler.is_compiling():
        out = _torch_binding.residual_norm(residual, block, post_weight, gate, pre_weight, scale, eps)
        if out is not NotImplemented:  # (something records the dispatcher's operators)
            return out[0], residual if block is None else out[1]
    y, r, _ = torch.ops.marlin_amd.residual_norm(residual, block, post_weight, gate, pre_weight, scale, eps)
    return (None if pre_weight is None else y), (residual if block is None else r)


_Maybe = torch.Tensor | None


@torch.library.custom_op("marlin_amd::residual_norm", mutates_args=())
def _norm_op(residual: torch.Tensor, block: _Maybe, post: _Maybe, gate: _Maybe, pre: _Maybe, scale: float,
             eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    y, r, lengths = _torch_binding.norm_lengths(residual, block, post, gate, pre, scale, eps)
    return tuple(residual.new_empty(0) if t is None else t for t in (y, r, lengths))


@_norm_op.register_fake
def _norm_fake(residual, block, post, gate, pre, scale, eps):
    rows = residual.numel() // residual.shape[-1]
    return (residual.new_empty(0 if pre is None else residual.shape),
            residual.new_empty(0 if block is None else residual.shape),
            residual.new_empty((rows, 2), dtype=torch.float32))


@torch.library.custom_op("marlin_amd::norm_grads", mutates_args=())
def _norm_grads_op(dy: _Maybe, dr: _Maybe, r: torch.Tensor, block: _Maybe, post: _Maybe, gate: _Maybe, pre: _Maybe,
                   lengths: torch.Tensor, scale: float, want: list[bool]) -> list[torch.Tensor]:
    out = _torch_binding.norm_grads(dy, dr, r, block, post, gate, pre, lengths, scale, *want)
    return [r.new_empty(0) if g is None else g for g in out]


@_norm_grads_op.register_fake
def _norm_grads_fake(dy, dr, r, block, post, gate, pre, lengths, scale, want):
    return [r.new_empty(0 if t is None or not w else t.shape) for t, w in zip((r, block, post, gate, pre), want)]


def _keep_norm(ctx, inputs, output):
    residual, block, post, gate, pre, scale, _ = inputs
    ctx.save_for_backward(residual if block is None else output[1], block, post, gate, pre, output[2])
    ctx.scale = 1.0 if block is None else scale


def _norm_backward(ctx, dy, dr, _):
    r, block, post, gate, pre, lengths = ctx.saved_tensors
    want = list(ctx.needs_input_grad[:5])  # (False of what is None)
    out = torch.ops.marlin_amd.norm_grads(dy if pre is not None else None, dr if block is not None else None, r, block,
                                          post, gate, pre, lengths, ctx.scale, want)
    return (*(g if w else None for g, w in zip(out, want)), None, None)


_norm_op.register_autograd(_norm_backward, setup_context=_keep_norm)


def dropout(x, p, seed, *, site=0, residual=None):
    """Every element of x zero with probability p (whatever its value), multiplied by 1 / (1 - p)
    otherwise, and added to `residual`, if that is given; rounded once.

    x: torch.half, torch.bfloat16 or torch.float, any shape of up to 2^34 elements; residual of x's shape and type.  Strided
    tensors are copied.  p is rounded to a multiple of 2^-16.  The mask is a function of `seed`, an int of
    64 bits with its sign or one torch.int64 on x's device (which a captured graph can advance),
    of `site`, 0 to 2^32 - 1, which distinguishes masks of one seed, and of the elements' places; include/
    feedforward_amd.h says which.  It is not stored: the backward pass makes it again, and a seed that
    is a tensor must not have been written until then.  Differentiable once, on the current stream of x's
    device."""
    if not torch.compiler.is_compiling():
        y = _torch_binding.dropout(x, residual, p, seed, site)
        if y is not NotImplemented:
            return y
    number, tensor = _seed_parts(p, seed)
    return torch.ops.marlin_amd.dropout(x, residual, float(p), number, tensor, site)


@torch.library.custom_op("marlin_amd::dropout", mutates_args=())
def _dropout_op(x: torch.Tensor, residual: _Maybe, p: float, seed: int, seed_at: _Maybe, site: int) -> torch.Tensor:
    return _torch_binding.dropout(x, residual, p, seed if seed_at is None else seed_at, site, True)


@torch.library.custom_op("marlin_amd::dropout_grad", mutates_args=())
def _dropout_grad_op(dy: torch.Tensor, p: float, seed: int, seed_at: _Maybe, site: int,
                     leaves: list[torch.Tensor]) -> torch.Tensor:
    return _torch_binding.dropout_grad(dy, p, seed if seed_at is None else seed_at, site, *leaves)


@_dropout_op.register_fake
def _dropout_fake(x, residual, p, seed, seed_at, site):
    return x.new_empty(x.shape)


@_dropout_grad_op.register_fake
def _dropout_grad_fake(dy, p, seed, seed_at, site, leaves):
    return dy.new_empty(dy.shape)


def _keep_dropout(ctx, inputs, output):
    x, residual, ctx.p, ctx.seed, seed_at, ctx.site = inputs
    ctx.save_for_backward(seed_at, *streamk._leaves(x, residual))


def _dropout_backward(ctx, dy):
    seed_at, *leaves = ctx.saved_tensors
    dx = None
    if ctx.needs_input_grad[0]:
        dx = torch.ops.marlin_amd.dropout_grad(dy, ctx.p, ctx.seed, seed_at, ctx.site, leaves)
    return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


_dropout_op.register_autograd(_dropout_backward, setup_context=_keep_dropout)


def _check_widths(hidden, inner, dropout):
    if hidden % 8 or inner % 8:
        raise ValueError("hidden and inner must be multiples of 8")
    if not 0 <= dropout <= 1:
        raise ValueError("dropout must be a probability")


class _Half(nn.Module):
    """What both kinds of block share: the norms, the gate and the residual's scale."""

    def __init__(self, hidden, activation, post_norm, gate, scale, eps, dtype, device):
        super().__init__()
        streamk._activation(activation)
        self.hidden, self.activation, self.scale, self.eps = hidden, activation, float(scale), float(eps)
        like = dict(dtype=dtype, device=device)
        self.pre_weight = nn.Parameter(torch.ones(hidden, **like))
        self.post_weight = nn.Parameter(torch.ones(hidden, **like)) if post_norm else None
        self.gate = nn.Parameter(torch.ones(hidden, **like)) if gate else None

    def _products(self, y, seed, site):
        raise NotImplementedError

    def forward(self, residual, gate=None, next_weight=None, *, seed=None, site=0):
        """residual (..., hidden) -> (y, residual'): residual' = scale * residual + gate *
        post_norm(down(gated(pre_norm(residual)))), y its norm by `next_weight`, the pre_weight of
        what follows, or None without one.  `gate`, if given, takes the place of the module's own,
        one for each sequence, say.  `seed` and `site`, below 2^31, are for dropout, as `dropout` takes
        them: the number of the step, say, and that of the layer."""
        y, _ = residual_norm(residual, pre_weight=self.pre_weight, eps=self.eps)
        return self.after_norm(y, residual, gate, next_weight, seed=seed, site=site)

    def after_norm(self, y, residual, gate=None, next_weight=None, *, seed=None, site=0):
        """`forward` from y, the residual's norm by pre_weight, which the block before has written
        already where it was given this module's as its `next_weight`."""
        return residual_norm(residual, self._products(y, seed, site), post_weight=self.post_weight,
                             gate=self.gate if gate is None else gate, scale=self.scale, pre_weight=next_weight,
                             eps=self.eps)


class FeedForward(_Half):
    """The feed-forward half of a decoder block, dense, torch.half or torch.bfloat16, with gradients
    of everything: pre-norm, gated projections, down projection, post-norm, gate and residual.
    hidden and inner are multiples of 8.  `gate_up` (2 inner, hidden) holds the rows of the gate
    projection and behind them those of the up projection; `down` is (hidden, inner).  With `dropout`,
    a probability, calls in training mode need a seed: the gated projection is dropped from, and the
    down projection."""

    def __init__(self, hidden, inner, activation="silu", *, post_norm=True, gate=False, scale=1.0, eps=1e-6,
                 dropout=0.0, dtype=torch.bfloat16, device=None):
        _check_widths(hidden, inner, dropout)
        super().__init__(hidden, activation, post_norm, gate, scale, eps, dtype, device)
        self.inner, self.dropout = inner, float(dropout)
        self.gate_up = nn.Parameter(torch.empty((2 * inner, hidden), dtype=dtype, device=device))
        self.down = nn.Parameter(torch.empty((hidden, inner), dtype=dtype, device=device))
        nn.init.normal_(self.gate_up, std=hidden ** -0.5)
        nn.init.normal_(self.down, std=inner ** -0.5)

    def _products(self, y, seed, site):
        h = streamk.gated(y, self.gate_up, self.activation)
        if not (self.training and self.dropout):
            return streamk.linear(h, self.down)
        h = dropout(h, self.dropout, seed, site=2 * site)
        return streamk.linear(h, self.down, dropout=self.dropout, seed=seed, site=2 * site + 1)

    @torch.no_grad()
    def quantize(self, groupsize=128):
        """This block with 4-bit weights (`marlin.quantize`) and halves for everything else, on the
        device of its weights; hidden a multiple of 256, inner of 128."""
        post, gate = self.post_weight is not None, self.gate is not None
        block = QuantizedFeedForward(self.hidden, self.inner, self.activation, groupsize, post_norm=post, gate=gate,
                                     scale=self.scale, eps=self.eps, device=self.down.device)
        parts = []
        for weight in (self.gate_up[:self.inner], self.gate_up[self.inner:], self.down):
            fake, _, s = marlin.quantize(weight.half().t().contiguous(), groupsize)
            parts.append((marlin._Weight(fake.t()), s.t()))
        block.gate_up.pack(parts[0][0], parts[1][0], parts[0][1], parts[1][1])
        block.down.pack(*parts[2])
        for name in ("pre_weight", "post_weight", "gate"):
            if getattr(self, name) is not None:
                getattr(block, name).copy_(getattr(self, name))
        return block


class QuantizedFeedForward(_Half):
    """`FeedForward` with 4-bit weights, torch.half, for inference: `gate_up` a marlin.GatedLayer,
    `down` a marlin.Layer.  The products have no gradients: a backward pass that would need them
    raises RuntimeError, as does compiling for one."""

    def __init__(self, hidden, inner, activation="silu", groupsize=128, *, post_norm=True, gate=False, scale=1.0,
                 eps=1e-6, device=None):
        super().__init__(hidden, activation, post_norm, gate, scale, eps, torch.half, device)
        self.inner = inner
        self.gate_up = marlin.GatedLayer(hidden, inner, groupsize, activation).to(device)
        self.down = marlin.Layer(inner, hidden, groupsize).to(device)
        self.requires_grad_(False)

    def _products(self, y, seed, site):
        out = self.down(self.gate_up(y))
        if y.requires_grad and torch.is_grad_enabled():
            return _torch_binding.without_gradients(out, y)
        return out


class Mlp(nn.Module):
    """The feed-forward half of a block without a gate, torch.half or torch.bfloat16, with gradients
    of everything: pre-norm, up projection with bias and activation, down projection with bias, residual.
    hidden and inner are multiples of 8; `up` is (inner, hidden), `down` (hidden, inner).  With
    `dropout`, a probability, calls in training mode need a seed: the activations are dropped from,
    and what is added to the residual."""

    def __init__(self, hidden, inner, activation="gelu", *, bias=True, dropout=0.0, eps=1e-6, dtype=torch.bfloat16,
                 device=None):
        _check_widths(hidden, inner, dropout)
        super().__init__()
        streamk._activation(activation)
        self.hidden, self.inner, self.activation = hidden, inner, activation
        self.dropout, self.eps = float(dropout), float(eps)
        like = dict(dtype=dtype, device=device)
        self.pre_weight = nn.Parameter(torch.ones(hidden, **like))
        self.up = nn.Parameter(torch.empty((inner, hidden), **like))
        self.down = nn.Parameter(torch.empty((hidden, inner), **like))
        self.up_bias = nn.Parameter(torch.zeros(inner, **like)) if bias else None
        self.down_bias = nn.Parameter(torch.zeros(hidden, **like)) if bias else None
        nn.init.normal_(self.up, std=hidden ** -0.5)
        nn.init.normal_(self.down, std=inner ** -0.5)

    def forward(self, residual, next_weight=None, *, seed=None, site=0):
        """residual (..., hidden) -> (y, residual'): residual' = residual + drop(down(drop(act(up(
        pre_norm(residual)))))), y its norm by `next_weight`, the pre_weight of what follows, or None
        without one.  `seed` and `site`: as `FeedForward`'s."""
        y, _ = residual_norm(residual, pre_weight=self.pre_weight, eps=self.eps)
        return self.after_norm(y, residual, next_weight, seed=seed, site=site)

    def after_norm(self, y, residual, next_weight=None, *, seed=None, site=0):
        """`forward` from y, the residual's norm by pre_weight."""
        p = self.dropout if self.training else 0.0
        h = streamk.linear(y, self.up, self.up_bias, self.activation, dropout=p, seed=seed, site=2 * site)
        r = streamk.linear(h, self.down, self.down_bias, residual=residual, dropout=p, seed=seed, site=2 * site + 1)
        return (None if next_weight is None else residual_norm(r, pre_weight=next_weight, eps=self.eps)[0]), r
