"""Dense fp16 GEMM with a stream-K tail (the reference's gemm/streamk_gemm) over
the C ABI of libmarlin_amd.so: C = A @ B.T with A (m, k) and B (n, k) in fp16,
fp32 accumulation.  The GEMM always runs in the HIP library; a missing library
is an import-time error.

Beside it the dense products of a feed-forward block that is trained, in fp16 or
bfloat16, with their gradients: `gated` and `linear` (include/feedforward_amd.h;
no reference counterpart)."""
import ctypes

import torch

from native import ACTIVATIONS, activation as _activation, lib as _lib, seed_parts as _seed_parts, torch_binding as _torch_binding  # noqa: F401,E501

_P, _I = ctypes.c_void_p, ctypes.c_int
_lib.streamk_amd_check.restype = _I
_lib.streamk_amd_check.argtypes = [_I, _I, _I]
_lib.streamk_amd_plan.restype = _I
_lib.streamk_amd_plan.argtypes = [_I, _I, _I, _I, _P]
_lib.streamk_amd_launches.restype = _I
_lib.streamk_amd_launches.argtypes = [_I, _I, _I, _I, _I, _P]
_lib.streamk_amd_tile.restype = _I
_lib.streamk_amd_tile.argtypes = [_I, _I, _I, _I, _P]
_lib.streamk_amd_force_tile.restype = None
_lib.streamk_amd_force_tile.argtypes = [_I, _I, _I]
_lib.streamk_amd_tile_coord.restype = None
_lib.streamk_amd_tile_coord.argtypes = [_I, _I, _I, _P]
_lib.streamk_amd_slice_coord.restype = None
_lib.streamk_amd_slice_coord.argtypes = [_I, _I, _I, _P]
_lib.streamk_amd_force_finish_polls.restype = None
_lib.streamk_amd_force_finish_polls.argtypes = [_I]
_lib.streamk_amd_last_error.restype = ctypes.c_char_p


def check(m, n, k):
    """Return code streamk_gemm_tn would give for these sizes (no GPU touched)."""
    return _lib.streamk_amd_check(m, n, k)


def plan(m, n, k, cus=256):
    """The split of the output tiles (tile_rows x tile_cols) into data-parallel and stream-K tiles."""
    out = (ctypes.c_int * 8)()
    rc = _lib.streamk_amd_plan(m, n, k, cus, out)
    keys = ("tiles_m", "tiles_n", "dp_tiles", "sk_tiles", "k_slices", "grid", "tile_rows", "tile_cols")
    return rc, dict(zip(keys, out))


def tile(m, n, k, cus=256):
    """(rows, cols, slices) of the tiles that compute the problem in one launch, in place of the
    plan's, or None."""
    out = (ctypes.c_int * 3)()
    _lib.streamk_amd_tile(m, n, k, cus, out)
    return tuple(out) if out[0] > 0 else None


def force_tile(rows, cols=0, slices=1):
    """Tiles that compute every problem, in place of the plan's (0 = by cost, -1 = never; calling
    thread only)."""
    _lib.streamk_amd_force_tile(int(rows), int(cols), int(slices))


def launches(m, n, k, cus=256, scratch=True):
    """The launches that compute the plan's tiles, unless tile() names others;
    `scratch`: whether there is room for partial sums."""
    out = (ctypes.c_int * 10)()
    count = _lib.streamk_amd_launches(m, n, k, cus, int(scratch), out)
    keys = ("rows", "cols", "waves", "tiles", "slices")
    return [dict(zip(keys, out[5 * i:5 * i + 5])) for i in range(count)]


def tile_coord(tile, tiles_m, tiles_n):
    """(row tile, column tile) of a tile number."""
    out = (ctypes.c_int * 2)()
    _lib.streamk_amd_tile_coord(tile, tiles_m, tiles_n, out)
    return out[0], out[1]


def slice_coord(block, tiles, slices):
    """(tile, slice) of a workgroup of a launch of slices."""
    out = (ctypes.c_int * 2)()
    _lib.streamk_amd_slice_coord(block, tiles, slices, out)
    return out[0], out[1]


def force_finish_polls(polls):
    """How often a workgroup looks for the other slices of its tile before it leaves them its
    share of the sums; -1 = the default (calling thread only)."""
    _lib.streamk_amd_force_finish_polls(int(polls))


def gemm(A, B, C=None):
    """C (m, n) = A (m, k) @ B (n, k).T on the current stream; returns C."""
    out = _torch_binding.dense(A, B, C)
    if out is not NotImplemented:
        return out
    # something records torch's operators, and sees this one (marlin.mul says more)
    if C is None:
        C = A.new_empty((A.shape[0], B.shape[0]))
    torch.ops.marlin_amd.gemm(A, B, C)
    return C


@torch.library.custom_op("marlin_amd::gemm", mutates_args=("C",))
def _gemm_op(A: torch.Tensor, B: torch.Tensor, C: torch.Tensor) -> None:
    _torch_binding.dense(A, B, C, True)


@_gemm_op.register_fake
def _gemm_fake(A, B, C):
    return None


# ---------------------------------------------------------------------------
# Products with gradients.  Under a compiler, or where something records the dispatcher's operators
# (the binding says NotImplemented), each is one operator of torch's dispatcher, which
# costs more host time than a product of a few rows takes; else the binding's, which is an autograd
# function where gradients are wanted.  (An argument more: the call is an operator's own.)

_lib.feedforward_plan.restype = _I
_lib.feedforward_plan.argtypes = [_I, _I, _I, _I, _I, _I, _P]
_lib.feedforward_force_tile.restype = None
_lib.feedforward_force_tile.argtypes = [_I, _I, _I]
_lib.feedforward_last_error.restype = ctypes.c_char_p


def gated(x, weight, activation="silu"):
    """Both projections of a gated feed-forward block, the activation and the product of the two in
    one launch: act(x @ G.T) * (x @ U.T), rounded once, for x (..., k) and weight (2n, k), the rows
    of G and behind them those of U; returns (..., n).

    torch.half or torch.bfloat16, n and k multiples of 8, weight at most 2 GiB; activation "silu"
    or "gelu" (its tanh form).  Where gradients are wanted the two sums are kept in fp32, 8n bytes a
    row.  Rows that do not start on 16 bytes are copied.  Differentiable once, on
    the current stream of x's device."""
    act = _activation(activation)
    if not torch.compiler.is_compiling():
        h = _torch_binding.gated_dense(x, weight, act)
        if h is not NotImplemented:
            return h
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return torch.ops.marlin_amd.gated_dense(x, weight, act)[0]
    return torch.ops.marlin_amd.gated_alone(x, weight, act)


def linear(x, weight, bias=None, activation=None, residual=None, *, dropout=0.0, seed=None, site=0):
    """x @ weight.T for x (..., k) and weight (n, k), torch.half or torch.bfloat16, n and k multiples
    of 8; returns (..., n).  With what else is given, in the product's epilogue and rounded once,

        residual + drop(activation(x @ weight.T + bias))

    bias: (n,).  activation: "silu" or "gelu" (its tanh form).  residual: the result's shape.
    dropout: the probability with which an element is dropped; `seed`, an int or one torch.int64 on x's
    device, and `site`, 0 to 2^32 - 1, which distinguishes masks of one seed, make the mask, that of
    `feedforward.dropout`, which is not stored: the backward pass makes it again, and a seed that is
    a tensor must not have been written until then.

    Where gradients are wanted, those of the bias and of the residual are there too, and with an
    activation its slopes are kept, 2n bytes a row: in bfloat16 good to 2^-8 of a slope down to 2^-102, in fp16 to
    2^-11 of it or 2^-27, whichever is more.  Differentiable once; streams and alignment as
    `gated`."""
    if bias is None and activation is None and residual is None and not dropout:
        if not torch.compiler.is_compiling():
            y = _torch_binding.linear_dense(x, weight)
            if y is not NotImplemented:
                return y
        return torch.ops.marlin_amd.linear_dense(x, weight)
    act = 0 if activation is None else _activation(activation)
    if not torch.compiler.is_compiling():
        y = _torch_binding.linear_full(x, weight, bias, residual, act, dropout, seed, site)
        if y is not NotImplemented:
            return y
    number, tensor = _seed_parts(dropout, seed)
    args = (x, weight, bias, residual, act, float(dropout), number, tensor, site)
    wants = [torch.is_grad_enabled() and t is not None and t.requires_grad for t in args[:4]]
    if any(wants):
        return torch.ops.marlin_amd.linear_full(*args, any(wants[:3]))[0]
    return torch.ops.marlin_amd.linear_alone(*args)


@torch.library.custom_op("marlin_amd::gated_dense", mutates_args=())
def _gated_op(x: torch.Tensor, weight: torch.Tensor, act: int) -> tuple[torch.Tensor, torch.Tensor]:
    return _torch_binding.gated_sums(x, weight, act)


@_gated_op.register_fake
def _gated_fake(x, weight, act):
    n = weight.shape[0] // 2
    return (x.new_empty(x.shape[:-1] + (n,)),
            x.new_empty((x.numel() // x.shape[-1], -(-n // 16) * 32), dtype=torch.float32))


# ... without gradients, and so without the sums
@torch.library.custom_op("marlin_amd::gated_alone", mutates_args=())
def _gated_alone_op(x: torch.Tensor, weight: torch.Tensor, act: int) -> torch.Tensor:
    return _torch_binding.gated_dense(x, weight, act, True)


@_gated_alone_op.register_fake
def _gated_alone_fake(x, weight, act):
    return x.new_empty(x.shape[:-1] + (weight.shape[0] // 2,))


# (of gradients that are not wanted an operator, which has to return tensors, returns empty ones)
def _wanted(x, dx, dw):
    return tuple(x.new_empty(0) if g is None else g for g in (dx, dw))


def _grads_fake(x, weight, want_x, want_weight):
    return x.new_empty(x.shape if want_x else 0), weight.new_empty(weight.shape if want_weight else 0)


@torch.library.custom_op("marlin_amd::gated_grads", mutates_args=())
def _gated_grads_op(dh: torch.Tensor, sums: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, act: int,
                    want_x: bool, want_weight: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _wanted(x, *_torch_binding.gated_grads(dh, sums, x, weight, act, want_x, want_weight))


@_gated_grads_op.register_fake
def _gated_grads_fake(dh, sums, x, weight, act, want_x, want_weight):
    return _grads_fake(x, weight, want_x, want_weight)


@torch.library.custom_op("marlin_amd::linear_dense", mutates_args=())
def _linear_op(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return _torch_binding.linear_dense(x, weight, True)


@_linear_op.register_fake
def _linear_fake(x, weight):
    return x.new_empty(x.shape[:-1] + (weight.shape[0],))


@torch.library.custom_op("marlin_amd::linear_grads", mutates_args=())
def _linear_grads_op(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, want_x: bool,
                     want_weight: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _wanted(x, *_torch_binding.linear_grads(dy, x, weight, want_x, want_weight))


@_linear_grads_op.register_fake
def _linear_grads_fake(dy, x, weight, want_x, want_weight):
    return _grads_fake(x, weight, want_x, want_weight)


_Maybe = torch.Tensor | None


# (a seed is a number, or a tensor that takes its place; keep: the slopes, which the residual's gradient alone does
# not take)
@torch.library.custom_op("marlin_amd::linear_full", mutates_args=())
def _full_op(x: torch.Tensor, weight: torch.Tensor, bias: _Maybe, residual: _Maybe, act: int, p: float, seed: int,
             seed_at: _Maybe, site: int, keep: bool) -> tuple[torch.Tensor, torch.Tensor]:
    args = (x, weight, bias, residual, act, p, seed if seed_at is None else seed_at, site)
    y, slopes = _torch_binding.linear_full_kept(*args) if keep else (_torch_binding.linear_full(*args, True), None)
    return y, x.new_empty(0, dtype=torch.int16) if slopes is None else slopes


@_full_op.register_fake
def _full_fake(x, weight, bias, residual, act, p, seed, seed_at, site, keep):
    n = weight.shape[0]
    return (x.new_empty(x.shape[:-1] + (n,)),
            x.new_empty((x.numel() // x.shape[-1], n) if act and keep else 0, dtype=torch.int16))


# ... without gradients, and so without the slopes
@torch.library.custom_op("marlin_amd::linear_alone", mutates_args=())
def _alone_op(x: torch.Tensor, weight: torch.Tensor, bias: _Maybe, residual: _Maybe, act: int, p: float, seed: int,
              seed_at: _Maybe, site: int) -> torch.Tensor:
    return _torch_binding.linear_full(x, weight, bias, residual, act, p, seed if seed_at is None else seed_at, site,
                                      True)


@_alone_op.register_fake
def _alone_fake(x, weight, bias, residual, act, p, seed, seed_at, site):
    return x.new_empty(x.shape[:-1] + (weight.shape[0],))


@torch.library.custom_op("marlin_amd::linear_full_grads", mutates_args=())
def _full_grads_op(dy: torch.Tensor, slopes: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, act: int, p: float,
                   seed: int, seed_at: _Maybe, site: int, want: list[bool],
                   leaves: list[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = _torch_binding.linear_full_grads(dy, slopes if act else None, x, weight, act, p,
                                           seed if seed_at is None else seed_at, site, *want, *leaves)
    return tuple(x.new_empty(0) if g is None else g for g in out)


@_full_grads_op.register_fake
def _full_grads_fake(dy, slopes, x, weight, act, p, seed, seed_at, site, want, leaves):
    return (*_grads_fake(x, weight, want[0], want[1]), x.new_empty(weight.shape[0] if want[2] else 0))


def _keep_full(ctx, inputs, output):
    x, weight, bias, residual, ctx.act, ctx.p, ctx.seed, seed_at, ctx.site, _ = inputs
    # (both operands, whichever is needed: they are also among the leaves that a captured backward pass looks at)
    ctx.save_for_backward(x, weight, output[1], seed_at, *_leaves(bias, residual))


def _leaves(*tensors):
    """Those that gradients are accumulated to."""
    return [t for t in tensors if t is not None and t.requires_grad and t.is_leaf]


def _full_backward(ctx, dy, _):
    x, weight, slopes, seed_at, *leaves = ctx.saved_tensors
    want = list(ctx.needs_input_grad[:4])  # (False of what is None)
    grads = (None,) * 3
    if any(want[:3]):
        grads = torch.ops.marlin_amd.linear_full_grads(dy, slopes, x, weight, ctx.act, ctx.p, ctx.seed, seed_at, ctx.site,
                                                       want[:3], leaves)
    return (*(g if w else None for g, w in zip(grads, want)), dy if want[3] else None, *(None,) * 6)


_full_op.register_autograd(_full_backward, setup_context=_keep_full)


def _keep_gated(ctx, inputs, output):
    ctx.save_for_backward(inputs[0], inputs[1], output[1])
    ctx.act = inputs[2]


def _gated_backward(ctx, dh, _):
    x, weight, sums = ctx.saved_tensors
    want = ctx.needs_input_grad
    dx, dw = torch.ops.marlin_amd.gated_grads(dh, sums, x, weight, ctx.act, want[0], want[1])
    return dx if want[0] else None, dw if want[1] else None, None


def _keep_linear(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _linear_backward(ctx, dy):
    want = ctx.needs_input_grad
    dx, dw = torch.ops.marlin_amd.linear_grads(dy, *ctx.saved_tensors, want[0], want[1])
    return dx if want[0] else None, dw if want[1] else None


_gated_op.register_autograd(_gated_backward, setup_context=_keep_gated)
_linear_op.register_autograd(_linear_backward, setup_context=_keep_linear)


def product_plan(m, n, k, gated=False, turned=0, cus=256):
    """(rows, columns, slices of k) of the tiles that compute `linear` or `gated` -- gated = 2: `linear` with
    anything in its epilogue; turned = 1: the
    gradient of their inputs, m rows of n over k; 2: that of their weights --, or None for empty ones.
    16 or 32 columns: all of up to 64 rows by workgroups of whole columns."""
    out = (ctypes.c_int * 3)()
    if _lib.feedforward_plan(m, n, k, int(gated), turned, cus, out) != 0:
        raise ValueError(_lib.feedforward_last_error().decode())
    return tuple(out) if out[0] > 0 else None


def force_product_tile(rows, cols=0, slices=0):
    """Tiles and slices for every product of the calling thread that they can compute; 0 = by cost."""
    _lib.feedforward_force_tile(int(rows), int(cols), int(slices))
