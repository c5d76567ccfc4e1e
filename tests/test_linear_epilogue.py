"""Products with bias, activation, dropout and residual in their epilogue: streamk.linear, its gradients
and the C entries.

The oracle is the definition in 64 bits on the rounded inputs, and the mask tests/_masks.py's.  Bounds,
element by element, with e half a step of the type (2^-11 fp16, 2^-8 bf16):
  z = x w^T + b is a sum of k products and one addition in fp32, off by at most (k + 1) 2^-24 of the
  sum S of its terms' magnitudes;
  the activations' slopes stay below 1.13, their second derivatives below 1, and in fp32 values and
  slopes are off by less than 2^-18 of their size (an exponential whose argument is good to 2^-24 of
  itself), slopes near zero by 2^-18 altogether; for the backward pass slopes are kept in steps of 2^-15,
  half a step of which they are off by;
  the mask's factor and the residual's addition round three times more, 2^-22 of the terms together;
  a result is rounded once, e of it, and for the products of the backward pass so is dz.
"""
import ctypes
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import _masks  # noqa: E402
import feedforward  # noqa: E402
import streamk  # noqa: E402

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
FP32, FEW, ACT, SLOPE = 2.0 ** -24, 2.0 ** -22, 2.0 ** -18, 2.0 ** -16
TILES = [(64, 64), (64, 128), (96, 128), (128, 128), (96, 256), (128, 256), (160, 256), (192, 256), (224, 256),
         (256, 256)]


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):  # half the smallest step of all
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -134


def act64(z, name):
    """value and slope"""
    if name is None:
        return z, torch.ones_like(z)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    t = torch.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3))
    return z / 2 * (1 + t), (1 + t) / 2 + z / 2 * (1 - t * t) * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * z * z)


def within(got, want, bound, type, parts):
    bound = bound * (1 + 2.0 ** -6) + least(type)  # (roundings of what is off already)
    err = (got.double() - want).abs()
    assert got.dtype == type and got.shape == want.shape and torch.isfinite(got).all()
    assert (err <= bound).all(), float((err / bound).max())
    # roundings are independent of each other: together they stay near one of them
    assert err.norm() <= parts * half_step(type) * want.norm() + least(type) * want.numel() ** 0.5


class Full64:
    """All there is, of m rows."""

    def __init__(self, x, w, bias, act, residual, p=0.0, seed=0, site=0):
        self.type = x.dtype
        self.x, self.w = x.double().reshape(-1, x.shape[-1]), w.double()
        m, n, k = len(self.x), len(w), w.shape[1]
        z, size = self.x @ self.w.t(), self.x.abs() @ self.w.abs().t()
        if bias is not None:
            z, size = z + bias.double(), size + bias.double().abs()
        self.off_z = (k + 1) * FP32 * size
        self.act = act
        self.value, self.slope = act64(z, act)
        self.off = 1.13 * self.off_z + ACT * self.value.abs() if act else self.off_z
        self.factor = torch.ones((m, n), dtype=torch.double, device=x.device)
        if p:
            keep, factor = _masks.mask((m, n), p, seed, site)
            self.factor = torch.from_numpy(keep).to(x.device).double() * factor
        self.residual = None if residual is None else residual.double().reshape(m, n)

    def check_forward(self, y):
        v = self.factor * self.value
        r = torch.zeros_like(v) if self.residual is None else self.residual
        want = v + r
        bound = self.factor * self.off + FEW * (v.abs() + r.abs()) + half_step(self.type) * want.abs()
        within(y.reshape(want.shape), want, bound, self.type, 1.01)
        dropped = self.factor == 0
        assert torch.equal(y.reshape(want.shape)[dropped].double(), r[dropped])

    def check_slopes(self, codes):
        """Steps of 2^-15 from -1/4 on, a number of 16 bits each."""
        got = ((codes.long() & 0xffff) - 8192).double() / 32768
        assert codes.dtype == torch.int16 and ((got - self.slope).abs() <= self.off_z + ACT + SLOPE).all()

    def check_grads(self, dy, dx=None, dw=None, dbias=None, dresidual=None):
        d, e, type = dy.double().reshape(self.factor.shape) * self.factor, half_step(self.type), self.type
        m, n = d.shape
        dz = d * self.slope
        off = FEW * dz.abs() + (d.abs() * (self.off_z + ACT + SLOPE) if self.act else 0)
        if dbias is not None:
            want = dz.sum(0)
            within(dbias, want, off.sum(0) + m * FP32 * dz.abs().sum(0) + e * want.abs(), type, 1.5)
        rounds = self.act is not None or (self.factor != 1).any()
        if rounds:
            off = off + e * dz.abs() + least(type)
        if dx is not None:
            want = dz @ self.w
            bound = off @ self.w.abs() + n * FP32 * (dz.abs() @ self.w.abs()) + e * want.abs()
            within(dx.reshape(want.shape), want, bound, type, 1.5)
        if dw is not None:
            want = dz.t() @ self.x
            bound = off.t() @ self.x.abs() + m * FP32 * (dz.abs().t() @ self.x.abs()) + e * want.abs()
            within(dw, want, bound, type, 1.5)
        if dresidual is not None:
            assert torch.equal(dresidual, dy)


def make(m, n, k, type, seed, dev="cuda"):
    """x, weight, bias, residual, dy"""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device=dev, generator=gen) * std).to(type)

    return randn(m, k), randn(n, k, std=k ** -0.5), randn(n), randn(m, n), randn(m, n)


# bias, activation, residual, probability
FORMS = [(True, None, False, 0), (False, "gelu", False, 0), (False, None, True, 0), (False, None, False, 0.25),
         (True, "silu", True, 0.1), (True, "gelu", False, 0.5), (True, None, True, 0.1), (False, "silu", True, 0)]


def call(x, w, bias, residual, form, seed=0, site=0):
    has_bias, act, has_residual, p = form
    return streamk.linear(x, w, bias if has_bias else None, act, residual if has_residual else None, dropout=p,
                          seed=seed, site=site)


def oracle(x, w, bias, residual, form, seed=0, site=0):
    has_bias, act, has_residual, p = form
    return Full64(x, w, bias if has_bias else None, act, residual if has_residual else None, p, seed, site)


# --- without a GPU -------------------------------------------------------------------------

def test_refusals():
    x, w, bias, residual, _ = make(2, 16, 16, torch.float16, 0, "cpu")
    for kwargs, error, text in (
            (dict(bias=bias), ValueError, "on the GPU"), (dict(activation="relu"), ValueError, "activation"),
            (dict(activation=1), ValueError, "activation"), (dict(bias=3), TypeError, "Tensor"),
            (dict(residual="r"), TypeError, "Tensor"), (dict(dropout=0.1), ValueError, "needs a seed"),
            (dict(dropout=0.1, seed=2 ** 64), ValueError, "64 bits"), (dict(dropout="p", seed=1), TypeError, "real number|float"),
            (dict(bias=bias, site=2 ** 70), ValueError, "64 bits"), (dict(dropout=0.1, seed=0.5), TypeError, "int")):
        with pytest.raises(error, match=text):
            streamk.linear(x, w, **kwargs)


def test_refuses_forward_mode():
    import torch.autograd.forward_ad as forward_ad
    x, w, bias, residual, _ = make(2, 16, 16, torch.float16, 0, "cpu")
    with forward_ad.dual_level():
        for i in range(4):
            args = [forward_ad.make_dual(t, t) if j == i else t for j, t in enumerate((x, w, bias, residual))]
            with pytest.raises(RuntimeError, match="forward-mode"):
                streamk.linear(args[0], args[1], args[2], "silu", args[3])


class DropArgs(ctypes.Structure):
    _fields_ = [("p", ctypes.c_double), ("seed", ctypes.c_longlong), ("seed_at", ctypes.c_void_p),
                ("site", ctypes.c_uint)]


def test_codes_of_the_entries():
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p

    def linear(m=0, n=8, k=8, x=16, w=16, y=16, bias=None, residual=None, slopes=None, ldx=8, ldw=8, ldy=8, ldr=8, lds=8,
               type=0, act=0, p=None, room=None):
        drop = None if p is None else ctypes.byref(DropArgs(p, 0, None, 0))
        return lib.feedforward_linear(P(x), P(w), P(y), P(bias), P(residual), P(slopes), m, n, k, L(ldx), L(ldw), L(ldy),
                                      L(ldr), L(lds), type, act, drop, P(room), L(0), 0, None)

    assert linear() == 0 and linear(x=None, w=None, y=None) == 0
    assert linear(bias=16, residual=16, slopes=16, act=2, p=0.5) == 0
    for bad in (dict(m=-1), dict(n=12), dict(k=12, ldx=16, ldw=16), dict(ldx=4), dict(ldw=0), dict(ldy=12), dict(type=2),
                dict(act=3), dict(act=-1), dict(x=8), dict(bias=8), dict(residual=8), dict(slopes=8, act=1), dict(residual=16, ldr=0),
                dict(slopes=16, act=1, lds=4), dict(slopes=16), dict(p=2.0), dict(p=float("nan")), dict(residual=16, ldr=1 << 22),
                dict(m=4, k=0, ldx=0, ldw=0), dict(m=4, x=None), dict(m=4, w=None), dict(m=4, y=None),
                dict(m=4, room=8), dict(m=0x7fffffff)):
        assert linear(**bad) == 1, bad
        assert lib.feedforward_last_error()

    lib.feedforward_linear_grad_bytes.restype = L
    many = lib.feedforward_linear_grad_bytes

    def grad(m=4, n=8, dy=16, slopes=None, dz=16, dbias=None, lddy=8, lds=8, lddz=8, type=0, p=None, partials=None,
             count=0):
        drop = None if p is None else ctypes.byref(DropArgs(p, 0, None, 0))
        return lib.feedforward_linear_grad(P(dy), P(slopes), P(dz), P(dbias), m, n, L(lddy), L(lds), L(lddz), type,
                                           drop, P(partials), L(count), 0, None)

    assert grad(m=0) == 0 and grad(n=0) == 0 and grad(m=0, dy=None, dz=None) == 0
    for bad in (dict(m=-1), dict(n=12), dict(lddy=4), dict(dz=8), dict(lddz=0), dict(slopes=8),
                dict(slopes=16, lds=4), dict(type=2), dict(p=-1.0),
                dict(dy=None), dict(dz=None), dict(m=4096, dbias=16),
                dict(m=4096, dbias=16, partials=16, count=many(4096, 8) - 1),
                dict(m=4096, dbias=16, partials=18, count=many(4096, 8))):
        assert grad(**bad) == 1, bad
    assert many(-1, 8) == -1 and many(4, 12) == -1 and many(0, 8) == 0 and many(4, 0) == 0
    assert many(1, 8) == 0 and many(7, 1 << 21) == 0
    for m, n in ((1 << 20, 8), (2048, 10752), (300, 1 << 14), (0x7fffffff, 8)):
        assert 4 * n < many(m, n) <= 4 * n * 4096


def test_fake_tensors_record_the_operators():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, w, b, r):
        y = streamk.linear(x, w, b, "gelu", r, dropout=0.1, seed=3)
        return torch.autograd.grad(y, (x, w, b, r), y)

    inputs = [t.requires_grad_() for t in make(6, 24, 16, torch.float16, 0, "cpu")[:4]]
    graph = make_fx(step, tracing_mode="fake")(*inputs)

    def names(graph):
        return [str(n.target).split(".")[1] for n in graph.graph.nodes if "marlin_amd" in str(n.target)]

    assert names(graph) == ["linear_full", "linear_full_grads"]
    with torch.no_grad():
        graph = make_fx(lambda x, w, b: streamk.linear(x, w, b), tracing_mode="fake")(*inputs[:3])
    assert names(graph) == ["linear_alone"]
    # a product alone is the one that it was
    with torch.no_grad():
        graph = make_fx(lambda x, w: streamk.linear(x, w, site=3), tracing_mode="fake")(*inputs[:2])
    assert names(graph) == ["linear_dense"]


# --- on the GPU ----------------------------------------------------------------------------

FORWARD = [(1, 8, 8), (1, 10752, 4096), (2, 40, 72), (16, 5208, 4160), (17, 2744, 1032), (33, 24, 8), (45, 5120, 13568),
           (64, 4104, 968), (65, 8, 8), (65, 72, 136), (300, 520, 4160), (777, 5208, 4160), (1025, 264, 64),
           (2100, 1544, 192)]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("m,n,k", FORWARD)
def test_forward(m, n, k, type):
    x, w, bias, residual, _ = make(m, n, k, type, m + n + k)
    for i, form in enumerate(FORMS):
        oracle(x, w, bias, residual, form, m, i).check_forward(call(x, w, bias, residual, form, m, i))


SMALL = [(32, 32), (32, 64)]  # with an epilogue alone


def test_plans_with_an_epilogue():
    """The small tiles are reached, and are no other products'; where they are not taken the plan is the
    product's without an epilogue."""
    seen, rng = set(), np.random.default_rng(0)
    for _ in range(4000):
        m, n, k = (int(2 ** rng.uniform(*r)) for r in ((0, 13), (3, 13), (3, 13)))
        n, k = 8 * max(1, n // 8), 8 * max(1, k // 8)
        rows, cols, slices = plan = streamk.product_plan(m, n, k, 2)
        bare = streamk.product_plan(m, n, k)
        if cols <= 32 and m <= 64:
            assert plan == bare and slices == 1 and rows == -(-m // 16) * 16
        elif (rows, cols) in SMALL:
            assert cols == 64 or m > 64
            assert 1 <= slices <= min(8, -(-k // 64))
            seen.add((rows, cols))
        else:
            assert plan == bare and (rows, cols) in TILES
        assert bare[:2] not in SMALL or m <= 64
    assert seen == set(SMALL)
    try:
        streamk.force_product_tile(32, 64, 2)
        assert streamk.product_plan(300, 520, 192, 2) == (32, 64, 2)
        assert streamk.product_plan(300, 520, 192) != (32, 64, 2) and streamk.product_plan(20, 520, 192, 2) == (32, 64, 2)
        streamk.force_product_tile(32, 32)
        assert streamk.product_plan(300, 520, 192, 2)[:2] == (32, 32)
        assert streamk.product_plan(300, 520, 192)[:2] != (32, 32)
        assert streamk.product_plan(20, 520, 192, 2) == streamk.product_plan(20, 520, 192) == (32, 32, 1)
        streamk.force_product_tile(16, 16)
        assert streamk.product_plan(300, 520, 192, 2)[1] != 16
    finally:
        streamk.force_product_tile(0)


@gpu
@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("tile", SMALL + TILES)
@pytest.mark.parametrize("m,n,k", [(1, 8, 64), (300, 520, 192), (257, 136, 1096), (333, 304, 640), (65, 40, 72)])
def test_every_tile(tile, m, n, k, slices):
    try:
        streamk.force_product_tile(*tile, slices)
        for type in TYPES:
            x, w, bias, residual, _ = make(m, n, k, type, 5)
            for i, form in enumerate(FORMS):
                oracle(x, w, bias, residual, form, 9, i).check_forward(call(x, w, bias, residual, form, 9, i))
            # what the backward pass takes
            slopes = streamk._torch_binding.linear_full_slopes(x, w, bias, None, 1, 0.0, None, 0)[1]
            Full64(x, w, bias, "silu", None).check_slopes(slopes)
    finally:
        streamk.force_product_tile(0)


@gpu
@pytest.mark.parametrize("cols", [16, 32])
@pytest.mark.parametrize("m,n,k", FORWARD[:8])
def test_whole_columns_of_few_rows(m, n, k, cols):
    try:
        streamk.force_product_tile(16, cols)
        for type in TYPES:
            x, w, bias, residual, _ = make(m, n, k, type, m + n)
            for i, form in enumerate(FORMS):
                oracle(x, w, bias, residual, form, 1, i).check_forward(call(x, w, bias, residual, form, 1, i))
            slopes = streamk._torch_binding.linear_full_slopes(x, w, bias, None, 1, 0.0, None, 0)[1]
            Full64(x, w, bias, "silu", None).check_slopes(slopes)
    finally:
        streamk.force_product_tile(0)


@gpu
@pytest.mark.parametrize("slices", [1, 2])
@pytest.mark.parametrize("tile", [(16, 16), (16, 32)] + SMALL + TILES)
def test_inside_rows_that_hold_nan(tile, slices):
    """Matrices inside larger ones: what lies beside them, and behind their last row, is NaN, and stays."""
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
    for type in TYPES:
        for m, n, k in ((40, 200, 136), (328, 264, 320), (264, 520, 456)):
            x, w, bias, residual, _ = make(m, n, k, type, m)

            def inside(t, dtype=None):
                rows, cols = t.shape
                room = torch.full((rows + 80, cols + 96), -7 if dtype else float("nan"), dtype=dtype or type, device="cuda")
                room[8:8 + rows, 16:16 + cols] = t
                return room, room[8:8 + rows, 16:16 + cols]

            (_, vx), (_, vw), (_, vr) = inside(x), inside(w), inside(residual)
            (ry, vy), (rs, vs) = inside(torch.zeros_like(residual)), inside(torch.zeros_like(residual), torch.int16)
            vb = inside(bias[None])[1]
            before, before_slopes = ry.clone(), rs.clone()
            room = torch.empty(3 * m * n, device="cuda")
            drop = DropArgs(0.3, 77, None, 2)
            try:
                streamk.force_product_tile(*tile, slices)
                code = lib.feedforward_linear(
                    P(vx.data_ptr()), P(vw.data_ptr()), P(vy.data_ptr()), P(vb.data_ptr()), P(vr.data_ptr()),
                    P(vs.data_ptr()), m, n, k, L(vx.stride(0)), L(vw.stride(0)), L(vy.stride(0)), L(vr.stride(0)),
                    L(vs.stride(0)), int(type == torch.bfloat16), 2, ctypes.byref(drop), P(room.data_ptr()),
                    L(4 * room.numel()), 0, P(torch.cuda.current_stream().cuda_stream))
            finally:
                streamk.force_product_tile(0)
            assert code == 0
            Full64(x, w, bias, "gelu", residual, 0.3, 77, 2).check_forward(vy)
            Full64(x, w, bias, "gelu", None).check_slopes(vs)
            vy.copy_(before[8:8 + m, 16:16 + n])
            vs.copy_(before_slopes[8:8 + m, 16:16 + n])
            assert torch.equal(ry.isnan(), before.isnan()) and not ry.nan_to_num().any()
            assert torch.equal(rs, before_slopes)


GRADS = [(1, 8, 8), (3, 40, 72), (65, 64, 64), (64, 520, 136), (200, 1032, 264), (777, 200, 1000), (1237, 2744, 1032),
         (2048, 512, 512), (5000, 8, 16)]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("m,n,k", GRADS)
def test_gradients(m, n, k, type):
    x, w, bias, residual, dy = make(m, n, k, type, m + n)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    for i, form in enumerate(FORMS):
        there = [True, True, form[0], form[2]]
        ref = oracle(*(t.detach() for t in leaves), form, 3, i)
        y = call(*leaves, form, 3, i)
        ref.check_forward(y.detach())
        grads = iter(torch.autograd.grad(y, [t for t, is_there in zip(leaves, there) if is_there], dy))
        ref.check_grads(dy, *(next(grads) if is_there else None for is_there in there))


@gpu
def test_gradients_against_differences():
    """In the inputs' own steps, d and what is left of it after rounding to fp16 weighed exactly: the
    difference of the sums of dy y over a symmetric step, against the gradients' products with the step."""
    m, n, k = 24, 40, 32
    x, w, bias, residual, dy = make(m, n, k, torch.float16, 4)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    args = dict(dropout=0.25, seed=6)
    for act in ("silu", "gelu"):
        grads = torch.autograd.grad(streamk.linear(x, w, bias, act, residual, **args), leaves, dy)
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            d = make(m, n, k, torch.float16, 50 + i)[i] * 2.0 ** -5
            up, down = (leaf.detach() + d), (leaf.detach() - d)
            values = []
            for moved in (up, down):
                inputs = [moved if t is leaf else t.detach() for t in leaves]
                values.append((streamk.linear(inputs[0], inputs[1], inputs[2], act, inputs[3], **args).double() * dy.double()).sum())
            step = up.double() - down.double()
            # The function's third derivative over the step: of both activations below 1.3 in size, so a
            # sixth of |dz'|^3, dz' the half step's change of z, for each output; a rounding of half a
            # step for each output twice, independent (six deviations), and of each gradient.
            first, second, half = leaves[0].detach().double(), leaves[1].detach().double(), step / 2
            dz = {0: lambda: half @ second.t(), 1: lambda: first @ half.t(), 2: lambda: half.expand(m, n),
                  3: lambda: torch.zeros(m, n, device="cuda", dtype=torch.double)}[i]()
            y = streamk.linear(*(t.detach() for t in leaves[:3]), act, leaves[3].detach(), **args).double()
            bend = (1.3 / 3 * dz.abs() ** 3 * dy.double().abs() / 0.75).sum()
            rounds = 6 * 2.0 ** -11 * (2 * (y * dy.double()).norm() ** 2 + (grad.double() * step).norm() ** 2) ** 0.5
            # (dz of the backward pass, rounded as well, reaches the gradient's product with the step)
            rounds += 6 * 2.0 ** -11 * 1.13 / 0.75 * (2 * dz * dy.double()).norm()
            assert abs(values[0] - values[1] - (grad.double() * step).sum()) <= bend + rounds


@gpu
def test_only_the_gradients_that_are_wanted():
    names = ("x", "w", "bias", "residual")
    for wanted in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (2, 3), (0, 1, 2, 3)):
        tensors = make(70, 72, 136, torch.bfloat16, 1)
        *inputs, dy = tensors
        for i in wanted:
            inputs[i].requires_grad_()
        for p in (0, 0.5):
            for act in (None, "gelu"):
                y = streamk.linear(*inputs[:3], act, inputs[3], dropout=p, seed=2)
                ref = Full64(*(t.detach() for t in inputs[:3]), act, inputs[3].detach(), p, 2)
                grads = torch.autograd.grad(y, [inputs[i] for i in wanted], dy)
                ref.check_grads(dy, **{"d" + names[i]: g for i, g in zip(wanted, grads)})


@gpu
@pytest.mark.parametrize("m", [5, 200])
def test_strides_alignment_and_shapes(m):
    type = torch.float16
    x, w, bias, residual, dy = make(m, 40, 72, type, 1)
    form = (True, "silu", True, 0.3)
    ref = oracle(x, w, bias, residual, form)
    wide = torch.zeros(m, 200, dtype=type, device="cuda")

    def placed(t, start, stride=200):
        room = torch.zeros(t.shape[0] * stride + 64, dtype=type, device="cuda")
        view = room.as_strided(t.shape, (stride, 1), start)
        return view.copy_(t)

    for start, stride in ((0, 200), (8, 200), (1, 200), (8, 201), (3, 75)):
        for which in range(4):
            inputs = [x, w, bias, residual]
            if which == 2:
                room = torch.zeros(100, dtype=type, device="cuda")
                inputs[2] = room[start:start + 40].copy_(bias)
            else:
                inputs[which] = placed(inputs[which], start, stride)
            leaves = [t.detach().requires_grad_() for t in inputs]
            y = call(*leaves, form)
            ref.check_forward(y.detach())
            ref.check_grads(dy, *torch.autograd.grad(y, leaves, dy))
    strided = torch.stack([bias, bias], dim=1)[:, 0]
    ref.check_forward(call(x, w, strided, residual, form))
    turned = [t.t().contiguous().t() for t in (x, w)] + [bias, residual.t().contiguous().t()]
    ref.check_forward(call(*turned, form))
    y = call(x.requires_grad_(), w, bias, residual, form)
    placed_dy = placed(dy, 1, 75)
    ref.check_grads(placed_dy, *torch.autograd.grad(y, (x,), placed_dy))
    # a residual that is one row for all, and shapes of one and of three dimensions
    one = residual[:1].expand(m, 40)
    oracle(x.detach(), w, bias, one, form).check_forward(call(x.detach(), w, bias, one, form))
    x3, r3 = x.detach().view(1, m, 72), residual.view(1, m, 40)
    y = call(x3, w, bias, r3, form)
    assert y.shape == (1, m, 40)
    ref.check_forward(y)
    y = call(x.detach()[0], w, bias, residual[0], form)
    assert y.shape == (40,)
    oracle(x.detach()[:1], w, bias, residual[:1], form).check_forward(y)
    del wide


@gpu
def test_a_broadcast_residuals_gradient():
    x, w, bias, residual, dy = make(60, 40, 72, torch.float16, 1)
    row = residual[0].clone().requires_grad_()
    y = streamk.linear(x, w, bias, None, row.expand(60, 40))
    got, = torch.autograd.grad(y, row, dy)
    want = dy.double().sum(0)
    # (torch's own sum of the expanded gradient, rounded once)
    assert ((got.double() - want).abs() <= 60 * FP32 * dy.double().abs().sum(0) + half_step(torch.float16) * want.abs()).all()


@gpu
def test_empty():
    w, bias = torch.ones(16, 8, device="cuda").half(), torch.ones(16, device="cuda").half()
    x, r = torch.ones(0, 8, device="cuda").half(), torch.ones(0, 16, device="cuda").half()
    leaves = [t.requires_grad_() for t in (x, w, bias, r)]
    y = streamk.linear(x, w, bias, "silu", r, dropout=0.5, seed=1)
    assert y.shape == (0, 16)
    dx, dw, db, dr = torch.autograd.grad(y.sum(), leaves)
    assert dx.shape == (0, 8) and dr.shape == (0, 16) and not dw.any() and not db.any()
    x, w, bias = torch.ones(3, 8, device="cuda").half(), torch.ones(0, 8, device="cuda").half(), torch.ones(0, device="cuda").half()
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    y = streamk.linear(x, w, bias, "gelu")
    assert y.shape == (3, 0)
    dx, dw, db = torch.autograd.grad(y.sum(), leaves)
    assert not dx.any() and dw.shape == (0, 8) and db.shape == (0,)


@gpu
def test_refusals_on_the_gpu():
    x, w, bias, residual, _ = make(6, 24, 16, torch.float16, 0)
    seed = torch.ones(1, dtype=torch.int64, device="cuda")
    for kwargs, text in (
            (dict(bias=bias[:8]), "bias"), (dict(bias=bias[None]), "bias"), (dict(bias=bias.bfloat16()), "bias"),
            (dict(bias=bias.cpu()), "bias"), (dict(bias=torch._neg_view(bias)), "bias"),
            (dict(residual=residual[:5]), "residual"), (dict(residual=residual[None]), "residual"),
            (dict(residual=residual.float()), "residual"), (dict(residual=residual.cpu()), "residual"),
            (dict(residual=residual[:, :16]), "residual"), (dict(residual=residual.view(12, 12)), "residual"),
            (dict(dropout=1.5, seed=1), "probability"), (dict(dropout=float("nan"), seed=1), "probability"),
            (dict(dropout=-0.5, seed=1), "probability"), (dict(dropout=0.5, seed=seed.cpu()), "seed"),
            (dict(dropout=0.5, seed=seed.int()), "seed"), (dict(dropout=0.5, seed=seed.expand(2)), "seed"),
            (dict(bias=bias, site=-1), "site"), (dict(bias=bias, site=2 ** 32), "site")):
        with pytest.raises(ValueError, match=text):
            streamk.linear(x, w, **kwargs)
    with pytest.raises(ValueError, match="multiples of 8"):
        streamk.linear(x, w[:12], bias[:12])
    with pytest.raises(ValueError, match="one type"):
        streamk.linear(x.bfloat16(), w, bias)


@gpu
@pytest.mark.parametrize("m", [4, 300])
def test_infinities_and_nan(m):
    x, w, bias, residual, dy = make(m, 72, 64, torch.float16, 1)
    form = (True, "gelu", True, 0.5)
    clean = call(x, w, bias, residual, form)
    keep = torch.from_numpy(_masks.mask((m, 72), 0.5, 0)[0]).cuda()
    for bad in (float("inf"), float("nan")):
        dirty = x.clone()
        dirty[m // 2, 5] = bad
        y = call(dirty, w, bias, residual, form)
        rows = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(y[rows], clean[rows])
        # in the row itself what is dropped is the residual
        assert torch.equal(y[m // 2][~keep[m // 2]], residual[m // 2][~keep[m // 2]])
        # a column of the bias stays in its column
        b = bias.clone()
        b[7] = bad
        y = call(x, w, b, residual, form)
        cols = torch.arange(72, device="cuda") != 7
        assert torch.equal(y[:, cols], clean[:, cols])
        # what is dropped has no gradient, whatever it is and whatever comes back for it
        leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
        ndy = torch.where(keep, dy, torch.full_like(dy, bad))
        got = torch.autograd.grad(call(*leaves, residual, form), leaves, ndy)
        want = torch.autograd.grad(call(*leaves, residual, form), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # NaN in a row of x is in that row's gradients, where they are kept, and in no other's
    for act in ("silu", "gelu"):
        dirty = x.clone()
        dirty[m // 2, 5] = float("nan")
        dirty.requires_grad_()
        g, = torch.autograd.grad(streamk.linear(dirty, w, bias, act), dirty, dy)
        rows = torch.arange(m, device="cuda") != m // 2
        assert torch.isfinite(g[rows]).all() and g[m // 2].isnan().all()
    # far out the activations are their arguments and zero, their slopes one and zero
    far = torch.full((1, 8), 200.0, device="cuda").half().requires_grad_()
    eye = torch.eye(8, device="cuda").half()
    for act in ("silu", "gelu"):
        for sign in (1.0, -1.0):
            y = streamk.linear(far, sign * eye, None, act)
            g, = torch.autograd.grad(y.sum(), far)
            assert (y == (200.0 if sign > 0 else 0.0)).all() and (g == (1.0 if sign > 0 else 0.0)).all()


@gpu
def test_what_may_be_written_between_the_passes():
    x, w, bias, residual, dy = make(20, 24, 16, torch.float16, 1)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    want = torch.autograd.grad(streamk.linear(*leaves[:3], "silu", residual, dropout=0.5, seed=1), leaves, dy)
    b, r = bias * 1, residual * 1
    y = streamk.linear(x, w, b, "silu", r, dropout=0.5, seed=1)
    b.detach().zero_()
    r.detach().zero_()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, dy), want))
    seed = torch.ones(1, dtype=torch.int64, device="cuda")
    y = streamk.linear(x, w, dropout=0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)


@gpu
def test_second_derivatives_raise():
    x, w, bias, residual, _ = make(20, 24, 16, torch.float16, 0)
    y = streamk.linear(x, w, bias, "silu", residual)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual, y.clone())]
    for i in range(4):
        y = streamk.linear(*leaves[:3], "silu", residual, dropout=0.5, seed=1)
        g, = torch.autograd.grad(y, leaves[i], leaves[4], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.float().sum() + leaves[4].float().sum(), leaves[4])


@gpu
def test_streams_and_two_at_once():
    cases = [make(m, n, k, torch.bfloat16, m) for m, n, k in ((300, 520, 1096), (64, 2048, 4096), (2048, 512, 512))]
    form = (True, "gelu", True, 0.1)
    want = [call(*c[:4], form) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for c, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(call(*c[:4], form))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("m", [1, 64, 200])
def test_captured_and_replayed(m):
    x, w, bias, residual, dy = make(m, 264, 4160, torch.bfloat16, 6)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    seed = torch.full((1,), 40, dtype=torch.int64, device="cuda")

    def step(seed):
        y = streamk.linear(x, w, bias, "gelu", residual, dropout=0.2, seed=seed, site=5)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(seed)
    side.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(seed))
            seed.add_(1)
    for turn in range(3):
        for i in range(2):
            graphs[i].replay()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                eager = step(40 + 2 * turn + i)
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], eager))
            del eager


@gpu
def test_a_captured_backward_pass_beside_an_eager_graph_of_its_leaves():
    x, w, bias, residual, dy = make(70, 72, 136, torch.float16, 6)
    side = torch.cuda.Stream()
    for i in range(4):
        inputs = [x, w, bias, residual]
        inputs[i] = inputs[i].clone().requires_grad_()

        def forward():
            return streamk.linear(*inputs[:3], "silu", inputs[3], dropout=0.5, seed=1)

        alive = forward()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                torch.autograd.grad(forward(), inputs[i], dy)
        torch.cuda.synchronize()
        assert torch.isfinite(torch.autograd.grad(alive, inputs[i], dy)[0]).all()
        del alive
    leaf = x.clone().requires_grad_()
    alive = feedforward.dropout(leaf, 0.5, 1)
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            torch.autograd.grad(feedforward.dropout(leaf, 0.5, 1), leaf, x)
    torch.cuda.synchronize()
    del alive


@gpu
def test_recorded_and_compiled():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, bias, residual, dy = make(70, 72, 136, torch.bfloat16, 1)
    seed = torch.full((1,), 11, dtype=torch.int64, device="cuda")
    calls = {
        "bias": lambda x, w, b, r: streamk.linear(x, w, b),
        "all": lambda x, w, b, r: streamk.linear(x, w, b, "gelu", r, dropout=0.25, seed=11, site=4),
        "seed": lambda x, w, b, r: streamk.linear(x, w, b, "gelu", r, dropout=0.25, seed=seed, site=4),
    }
    other = make(70, 72, 136, torch.bfloat16, 2)[:4]
    for name, f in calls.items():
        inputs = [x, w, bias, residual]
        want = f(*inputs)
        graph = make_fx(f)(*other)
        assert torch.equal(graph(*inputs), want)
        assert torch.equal(torch.jit.trace(f, tuple(other), check_trace=False)(*inputs), want)
        torch._dynamo.reset()
        compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
        assert torch.equal(compiled(*inputs), want)
        leaves = [t.clone().requires_grad_() for t in inputs[:(3 if name == "bias" else 4)]] + inputs[(3 if name == "bias" else 4):]
        asked = [t for t in leaves if t.requires_grad]
        got = torch.autograd.grad(compiled(*leaves), asked, dy)
        ref = torch.autograd.grad(f(*leaves), asked, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
        # some of them alone
        leaves = [x, w, bias.clone().requires_grad_(), residual]
        got, = torch.autograd.grad(compiled(*leaves), leaves[2:3], dy)
        assert torch.equal(got, torch.autograd.grad(f(*leaves), leaves[2:3], dy)[0])


@gpu
def test_the_mask_is_that_of_dropout():
    x, w, bias, residual, _ = make(77, 264, 64, torch.bfloat16, 3)
    seed = torch.full((), -3, dtype=torch.int64, device="cuda")
    for m in (3, 77):
        y = streamk.linear(x[:m], w, dropout=0.4, seed=seed, site=9)
        ones = feedforward.dropout(torch.ones(m, 264, device="cuda"), 0.4, -3, site=9)
        assert torch.equal(y == 0, ones == 0)


@gpu
def test_the_operators_as_they_are_used_together():
    """Two blocks of a model trained for three steps, each step captured once and replayed, with masks
    of its own: the same as eager steps."""
    def model():
        torch.manual_seed(3)
        return [feedforward.Mlp(64, 256, dropout=0.1, device="cuda"),
                feedforward.FeedForward(64, 136, dropout=0.1, device="cuda")]

    def gradients(blocks, x, dy, seed):
        x = feedforward.dropout(x, 0.1, seed, site=100)
        y, r = blocks[0](x, next_weight=blocks[1].pre_weight, seed=seed, site=0)
        _, r = blocks[1].after_norm(y, r, seed=seed, site=1)
        params = [p for b in blocks for p in b.parameters()]
        return r.detach(), torch.autograd.grad(r, params, dy)

    gen = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn((2, 50, 64), device="cuda", generator=gen).bfloat16() for _ in range(2))
    eager = model()
    want = []
    for step in range(3):
        want.append(gradients(eager, x, dy, 7 + step))
        with torch.no_grad():
            for p, g in zip([p for b in eager for p in b.parameters()], want[-1][1]):
                p -= 0.01 * g
    blocks = model()
    seed = torch.full((1,), 7, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        gradients(blocks, x, dy, seed)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, grads = gradients(blocks, x, dy, seed)
        with torch.no_grad():
            for p, g in zip([p for b in blocks for p in b.parameters()], grads):
                p -= 0.01 * g
        seed.add_(1)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[step][0])
        assert all(torch.equal(a, b) for a, b in zip(grads, want[step][1]))


# --- two slices of a big tile, which finish it together -------------------------------------

@pytest.fixture
def polls():
    lib = streamk._lib
    lib.feedforward_force_polls.argtypes = [ctypes.c_int]
    lib.feedforward_force_polls.restype = None
    yield lib.feedforward_force_polls
    lib.feedforward_force_polls(-1)


def product(a, b, m, n, k, turned, room, garbage=0):
    """The C entry, with that many bytes of room, filled with the byte `garbage`."""
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
    c = torch.full((m, n), float("nan"), dtype=a.dtype, device="cuda")
    at = torch.full((max(room, 16),), garbage, dtype=torch.uint8, device="cuda")
    assert lib.feedforward_product(P(a.data_ptr()), P(b.data_ptr()), P(c.data_ptr()), m, n, k, L(a.stride(0)),
                                   L(b.stride(0)), L(n), turned, int(a.dtype == torch.bfloat16), P(at.data_ptr()),
                                   L(room), 0, P(torch.cuda.current_stream().cuda_stream)) == 0
    return c, at


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tile", TILES[6:])
@pytest.mark.parametrize("m,n,k", [(328, 264, 320), (8, 8, 72), (1000, 1544, 200)])
def test_slices_that_meet_are_their_sum(m, n, k, tile, type, polls):
    """To the bit, whether they wait for each other or not, whatever was in the room, and with room that
    does for the sums alone, which a launch of its own adds up."""
    lib = streamk._lib
    lib.feedforward_product_bytes.restype = ctypes.c_longlong
    gen = torch.Generator(device="cuda").manual_seed(m)
    a, b = (torch.randn(r, k, device="cuda", generator=gen).to(type) for r in (m, n))
    for turned in (0, 1, 2):
        va, vb = a.t().contiguous() if turned == 2 else a, b.t().contiguous() if turned else b
        try:
            streamk.force_product_tile(*tile, 2)
            assert streamk.product_plan(m, n, k, False, turned) == (*tile, 2)
            room = lib.feedforward_product_bytes(m, n, k, 0, turned, 0)
            assert room > 8 * m * n
            want, _ = product(va, vb, m, n, k, turned, 8 * m * n)
            for count in (-1, 0, 1, 64):
                polls(count)
                for garbage in (0, 255, 37):
                    got, at = product(va, vb, m, n, k, turned, room, garbage)
                    assert torch.equal(got, want)
                # once more in what the last call left there
                lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
                again = torch.full_like(got, float("nan"))
                assert lib.feedforward_product(
                    P(va.data_ptr()), P(vb.data_ptr()), P(again.data_ptr()), m, n, k, L(va.stride(0)), L(vb.stride(0)),
                    L(n), turned, int(type == torch.bfloat16), P(at.data_ptr()), L(room), 0,
                    P(torch.cuda.current_stream().cuda_stream)) == 0
                assert torch.equal(again, want)
        finally:
            streamk.force_product_tile(0)
        exact = a.double() @ b.double().t()
        bound = k * FP32 * (a.double().abs() @ b.double().abs().t()) + half_step(type) * exact.abs()
        within(want, exact, bound, type, 1.01)


@gpu
@pytest.mark.parametrize("tile", TILES[6:])
def test_epilogues_of_slices_that_meet(tile, polls):
    for type in TYPES:
        for m, n, k in ((333, 528, 640), (100, 144, 1096)):
            x, w, bias, residual, _ = make(m, n, k, type, 5)
            for count in (-1, 0):
                polls(count)
                try:
                    streamk.force_product_tile(*tile, 2)
                    for i, form in enumerate(FORMS):
                        oracle(x, w, bias, residual, form, 9, i).check_forward(call(x, w, bias, residual, form, 9, i))
                    slopes = streamk._torch_binding.linear_full_slopes(x, w, bias, None, 2, 0.0, None, 0)[1]
                    Full64(x, w, bias, "gelu", None).check_slopes(slopes)
                    # the gated epilogue, and what it keeps, against its form in one slice
                    h, sums = streamk._torch_binding.gated_sums(x, w, 1)
                    streamk.force_product_tile(*tile, 1)
                    h1, sums1 = streamk._torch_binding.gated_sums(x, w, 1)
                finally:
                    streamk.force_product_tile(0)
                size = x.double().abs() @ w.double().abs().t()
                off = 2 * k * FP32 * size.max() + 2.0 ** -22
                half = n // 2
                for c in range(0, half, 16):
                    wide = min(16, half - c)
                    for at in (2 * c, 2 * c + 16):
                        assert ((sums[:, at:at + wide] - sums1[:, at:at + wide]).abs() <= off).all()
                assert ((h.double() - h1.double()).abs() <= 4 * half_step(type) * h1.double().abs() + 8 * off * (1 + size.max())).all()


@gpu
def test_slices_that_meet_captured_and_on_two_streams():
    a, b = (torch.randn(r, 4096, device="cuda").bfloat16() for r in (512, 1024))
    try:
        streamk.force_product_tile(256, 256, 2)
        want = streamk.linear(a, b)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        graphs, outs = [], []
        for stream in streams:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append([streamk.linear(a, b) for _ in range(3)])
            graphs.append(graph)
        for _ in range(4):
            for out in outs:
                for o in out:
                    o.zero_()
            torch.cuda.synchronize()
            eager = []
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
                    eager.append(streamk.linear(a, b))
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for out in outs for o in out)
            assert all(torch.equal(o, want) for o in eager)
    finally:
        streamk.force_product_tile(0)


# --- sizes and ways of calling at the ends ---------------------------------------------------

@gpu
def test_results_of_more_than_32_bits():
    """2^31 elements and more, 4 GiB each of result, residual and gradient: the last rows, their mask and their
    gradients."""
    m, n, k = (1 << 16) + 40, (1 << 15) + 8, 64
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, w, bias = (torch.randn(s, device="cuda", generator=gen).bfloat16() for s in ((m, k), (n, k), (n,)))
    residual = torch.empty((m, n), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    for t in (x, w, bias):
        t.requires_grad_()
    y = streamk.linear(x, w, bias, "silu", residual, dropout=0.5, seed=77, site=3)
    grads = torch.autograd.grad(y, (x, w, bias), residual)
    y = y.detach()
    last = slice(m - 16, m)
    with torch.no_grad():
        ref = Full64(x[last], w, bias, "silu", residual[last])
        # the mask of these rows, element by element of the generator
        first = (m - 16) * n
        assert first % 8 == 0
        group = np.arange(first // 8, m * n // 8, dtype=np.uint64)
        c = [group & _masks.LOW, group >> np.uint64(32), np.full_like(group, 3), np.zeros_like(group)]
        for r in range(7):
            k0, k1 = np.uint64((77 + r * _masks.W0) % 2 ** 32), np.uint64(r * _masks.W1 % 2 ** 32)
            a, b = c[0] * np.uint64(_masks.M0), c[2] * np.uint64(_masks.M1)
            c = [b >> np.uint64(32) ^ c[1] ^ k0, b & _masks.LOW, a >> np.uint64(32) ^ c[3] ^ k1, a & _masks.LOW]
        words = np.stack(c, axis=1)
        bits = np.stack([words & np.uint64(0xffff), words >> np.uint64(16)], axis=2).reshape(16, n)
        ref.factor = torch.from_numpy((bits >= 32768).astype(np.float64) * 2).cuda()
        ref.check_forward(y[last])
        ref.check_grads(residual[last], dx=grads[0][last])
    assert all(torch.isfinite(g).all() for g in grads)


@gpu
def test_only_the_residual_wants_a_gradient():
    x, w, bias, residual, dy = make(20, 24, 16, torch.float16, 1)
    residual.requires_grad_()
    y = streamk.linear(x, w, bias, "silu", residual, dropout=0.5, seed=1)
    assert torch.equal(torch.autograd.grad(y, residual, dy)[0], dy)
    y = feedforward.dropout(dy, 0.5, 1, residual=residual)
    assert torch.equal(torch.autograd.grad(y, residual, dy)[0], dy)


@gpu
def test_backward_twice_and_accumulated():
    x, w, bias, residual, dy = make(70, 72, 136, torch.bfloat16, 1)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    y = streamk.linear(x, w, bias, "gelu", residual, dropout=0.25, seed=3)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    y.backward(dy, retain_graph=True)
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))
    kept = dy.clone()
    y.backward(dy)
    assert all(torch.equal(t.grad, g + g) for t, g in zip(leaves, want))
    assert torch.equal(dy, kept)  # the residual's gradient is dy, and accumulating does not write to it


@gpu
def test_threads_at_once():
    import threading
    cases = [make(m, 264, 4160, torch.bfloat16, m) for m in (1, 70, 300, 600)]
    form = (True, "gelu", True, 0.25)

    def step(c):
        leaves = [t.detach().requires_grad_() for t in c[:4]]
        y = call(*leaves, form)
        return (y.detach(), *torch.autograd.grad(y, leaves, c[4]))

    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    got = [None] * len(cases)

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = step(cases[i])
        torch.cuda.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@gpu
def test_a_compiled_block_and_a_checkpointed_one():
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(0)
    mlp = feedforward.Mlp(64, 136, dropout=0.2, device="cuda")
    x = torch.randn((3, 37, 64), device="cuda").bfloat16().requires_grad_()
    params = [x, *mlp.parameters()]

    def loss(f):
        return torch.autograd.grad(f(x)[1].float().square().sum(), params)

    want = loss(lambda t: mlp(t, seed=5))
    torch._dynamo.reset()
    compiled = torch.compile(lambda t: mlp(t, seed=5), backend="aot_eager", fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(loss(compiled), want))
    again = loss(lambda t: checkpoint(lambda u: mlp(u, seed=5), t, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(again, want))
