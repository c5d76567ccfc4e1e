"""The feed-forward half of a decoder block: the norms around it, and the block as a module, dense
and trained (`FeedForward`) or with 4-bit weights (`QuantizedFeedForward`).  The norms' kernels are
in the HIP library (include/feedforward_amd.h), the products those of `streamk` and `marlin`; no
reference counterpart."""
import torch
import torch.nn as nn

import marlin
import streamk
from native import torch_binding as _torch_binding


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

    def _products(self, y):
        raise NotImplementedError

    def forward(self, residual, gate=None, next_weight=None):
        """residual (..., hidden) -> (y, residual'): residual' = scale * residual + gate *
        post_norm(down(gated(pre_norm(residual)))), y its norm by `next_weight`, the pre_weight of
        what follows, or None without one.  `gate`, if given, takes the place of the module's own,
        one for each sequence, say."""
        y, _ = residual_norm(residual, pre_weight=self.pre_weight, eps=self.eps)
        return self.after_norm(y, residual, gate, next_weight)

    def after_norm(self, y, residual, gate=None, next_weight=None):
        """`forward` from y, the residual's norm by pre_weight, which the block before has written
        already where it was given this module's as its `next_weight`."""
        return residual_norm(residual, self._products(y), post_weight=self.post_weight,
                             gate=self.gate if gate is None else gate, scale=self.scale, pre_weight=next_weight,
                             eps=self.eps)


class FeedForward(_Half):
    """The feed-forward half of a decoder block, dense, torch.half or torch.bfloat16, with gradients
    of everything: pre-norm, gated projections, down projection, post-norm, gate and residual.
    hidden and inner are multiples of 8.  `gate_up` (2 inner, hidden) holds the rows of the gate
    projection and behind them those of the up projection; `down` is (hidden, inner)."""

    def __init__(self, hidden, inner, activation="silu", *, post_norm=True, gate=False, scale=1.0, eps=1e-6,
                 dtype=torch.bfloat16, device=None):
        if hidden % 8 or inner % 8:
            raise ValueError("hidden and inner must be multiples of 8")
        super().__init__(hidden, activation, post_norm, gate, scale, eps, dtype, device)
        self.inner = inner
        self.gate_up = nn.Parameter(torch.empty((2 * inner, hidden), dtype=dtype, device=device))
        self.down = nn.Parameter(torch.empty((hidden, inner), dtype=dtype, device=device))
        nn.init.normal_(self.gate_up, std=hidden ** -0.5)
        nn.init.normal_(self.down, std=inner ** -0.5)

    def _products(self, y):
        return streamk.linear(streamk.gated(y, self.gate_up, self.activation), self.down)

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

    def _products(self, y):
        out = self.down(self.gate_up(y))
        if y.requires_grad and torch.is_grad_enabled():
            return _torch_binding.without_gradients(out, y)
        return out
