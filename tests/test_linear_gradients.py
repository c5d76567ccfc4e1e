"""Gradients of products with dropout and without an activation: the masked gradient enters the products as it is, and
the factor of what is kept is theirs.

dx = f (mask dy) W and dW = f (mask dy)^T x are sums of exact products in fp32, each off by at most one 2^-24 a term of
the sum of the terms' magnitudes, then multiplied by a factor that is rounded to 2^-24 itself and rounds the product once more
(2^-22 of the result covers both), and rounded once to the type: e, half a step, of it.
"""
import ctypes
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import _masks  # noqa: E402
import feedforward  # noqa: E402,F401  (its operators)
import streamk  # noqa: E402

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
FP32, FEW = 2.0 ** -24, 2.0 ** -22
FEW_ROWS = [(16, 16), (16, 32)]
TILES = [(64, 64), (64, 128), (96, 128), (128, 128), (96, 256), (128, 256), (160, 256), (192, 256), (224, 256),
         (256, 256)]
P, L = ctypes.c_void_p, ctypes.c_longlong


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):  # half the smallest step of all
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -134


def make(m, n, k, type, seed, dev="cuda"):
    """x, weight, bias, residual, dy"""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device=dev, generator=gen) * std).to(type)

    return randn(m, k), randn(n, k, std=k ** -0.5), randn(n), randn(m, n), randn(m, n)


def within(got, want, size, terms):
    e = half_step(got.dtype)
    bound = (terms * FP32 * size + (FEW + e) * want.abs()) * (1 + 2.0 ** -6) + least(got.dtype)
    err = (got.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("p", [0.1, 0.3, 0.9])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (3, 40, 72), (65, 64, 64), (200, 1032, 264), (777, 200, 1000), (2048, 512, 512)])
def test_masked_gradients_are_not_rounded(m, n, k, p, type):
    x, w, bias, residual, dy = make(m, n, k, type, m + n)
    leaves = [t.requires_grad_() for t in (x, w, bias, residual)]
    y = streamk.linear(x, w, bias, None, residual, dropout=p, seed=5, site=2)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    keep, factor = _masks.mask((m, n), p, 5, 2)
    dz = dy.double() * torch.from_numpy(keep).cuda() * factor
    x, w = x.detach().double(), w.detach().double()
    within(dx, dz @ w, dz.abs() @ w.abs(), n)
    within(dw, dz.t() @ x, dz.abs().t() @ x.abs(), m)
    within(db, dz.sum(0), dz.abs().sum(0), m)
    assert torch.equal(dr, dy)


@gpu
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("m", [4, 300])
def test_a_factor_past_the_range_of_fp16(m, act):
    """p = 1 - 2^-16: what is kept is multiplied by 65536, which dz in 16 bits would not hold.  (Activations of arguments
    above 30, whose slopes are one.)"""
    n, k, p = 4096, 64, 1 - 2.0 ** -16
    x = torch.ones((m, k), dtype=torch.float16, device="cuda")
    w = torch.full((n, k), 2.0 ** -12, dtype=torch.float16, device="cuda")
    bias = torch.full((n,), 32.0, dtype=torch.float16, device="cuda")
    dy = torch.full((m, n), 4.0, dtype=torch.float16, device="cuda")
    dy[:, 1::2] = -2.0
    for seed in range(64):  # (one in 65536 is kept)
        keep = torch.from_numpy(_masks.mask((m, n), p, seed)[0]).cuda()
        if keep.any():
            break
    assert keep.any()
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    dx, dw, db = torch.autograd.grad(streamk.linear(x, w, bias, act, dropout=p, seed=seed), leaves, dy)
    dz = dy.double() * keep * 65536
    # exact: powers of two, and few of them
    assert torch.equal(dx.double(), dz @ w.detach().double())
    for got, want in ((dw, dz.t() @ x.detach().double()), (db, dz.sum(0))):
        assert torch.equal(got.isinf(), want.abs() > 65504) and not got.isnan().any()


def product(a, b, m, n, k, turned, scale, room):
    """The C entry: feedforward_product where scale is None."""
    lib = streamk._lib
    c = torch.full((m, n), float("nan"), dtype=a.dtype, device="cuda")
    at = torch.empty(max(room, 16), dtype=torch.uint8, device="cuda")
    entry, scales = (lib.feedforward_product, []) if scale is None else (lib.feedforward_product_scaled, [ctypes.c_float(scale)])
    assert entry(P(a.data_ptr()), P(b.data_ptr()), P(c.data_ptr()), m, n, k, L(a.stride(0)), L(b.stride(0)), L(n), turned,
                 int(a.dtype == torch.bfloat16), *scales, P(at.data_ptr()), L(room), 0,
                 P(torch.cuda.current_stream().cuda_stream)) == 0
    return c


@gpu
@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("tile", FEW_ROWS + TILES)
@pytest.mark.parametrize("m,n,k", [(40, 200, 136), (328, 264, 320)])
def test_scaled_products_by_every_tile(m, n, k, tile, slices):
    lib = streamk._lib
    lib.feedforward_product_bytes.restype = L
    for type in TYPES:
        a, b = make(m, n, k, type, 3)[:2]
        a, b = a.contiguous(), b.contiguous()
        for turned in (0, 1, 2):
            va, vb = a.t().contiguous() if turned == 2 else a, b.t().contiguous() if turned else b
            try:
                streamk.force_product_tile(*tile, slices)
                # (room for slices that meet, and for those whose sums a launch adds)
                for room in (lib.feedforward_product_bytes(m, n, k, 0, turned, 0), 4 * slices * m * n):
                    plain = product(va, vb, m, n, k, turned, None, room)
                    assert torch.equal(product(va, vb, m, n, k, turned, 1.0, room), plain)
                    # (exact: these values keep far from the ends of fp16's range, but where they are near zero)
                    eight = product(va, vb, m, n, k, turned, 8.0, room)
                    normal = plain.abs() >= 2.0 ** -13
                    assert torch.equal(eight[normal], 8 * plain[normal])
                    third = product(va, vb, m, n, k, turned, 0.3, room)
            finally:
                streamk.force_product_tile(0)
            want = 0.3 * (a.double() @ b.double().t())
            within(third, want, 0.3 * (a.double().abs() @ b.double().abs().t()), k)


def test_codes_of_the_entry():
    lib = streamk._lib

    def call(m=0, n=8, k=8, turned=0, type=0, a=16, lda=8):
        return lib.feedforward_product_scaled(P(a), P(16), P(16), m, n, k, L(lda), L(8), L(8), turned, type, ctypes.c_float(2.0),
                                              None, L(0), 0, None)

    assert call() == 0
    for bad in (dict(m=-1), dict(n=12), dict(k=12), dict(turned=3), dict(turned=2, m=4), dict(type=2), dict(a=8),
                dict(lda=4), dict(m=4, k=0), dict(m=4, a=None)):
        assert call(**bad) == 1, bad


def test_the_factor_of_the_entry():
    """Set on the host, with or without a GPU."""
    from test_linear_slopes import DropArgs
    lib, factor = streamk._lib, ctypes.c_float(7.0)

    def call(p, slopes):
        drop = ctypes.byref(DropArgs(p, 0, None, 0))
        return lib.feedforward_linear_backward(None, P(slopes), None, None, 0, 8, L(8), L(8), L(8), 0, drop, None, L(0),
                                               ctypes.byref(factor), 0, None)

    for slopes in (None, 16):
        factor.value = 7.0
        assert call(0.5, slopes) == 0 and factor.value == 1.0  # (of no rows)


# --- what is kept between the passes ---------------------------------------------------------

def kept_bytes(call):
    """(what lives after `call` beyond what it was given and what it returns, its result)"""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = call()
    return torch.cuda.memory_allocated() - before - y.numel() * y.element_size(), y


@gpu
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dropout", [0, 0.5])
def test_slopes_are_kept_for_the_gradients_that_take_them(act, dropout):
    m, n, k = 1024, 2048, 512
    for wanted in range(4):
        inputs = list(make(m, n, k, torch.bfloat16, 1))
        dy = inputs.pop()
        inputs[wanted].requires_grad_()
        bytes, y = kept_bytes(lambda: streamk.linear(*inputs[:3], act, inputs[3], dropout=dropout, seed=3))
        assert bytes == (2 * m * n if act and wanted < 3 else 0)
        g, = torch.autograd.grad(y, inputs[wanted], dy)
        assert g.shape == inputs[wanted].shape and torch.isfinite(g).all() and g.any()
        if wanted == 3:
            assert torch.equal(g, dy)


@gpu
@pytest.mark.parametrize("act", [None, "silu"])
def test_operands_are_kept_for_each_others_gradients(act):
    """A frozen layer's input, and a weight whose input wants nothing, need not live until the backward pass, and
    what is written to them then does not matter."""
    m, n, k = 1024, 2048, 512
    x, w, bias, residual, dy = make(m, n, k, torch.bfloat16, 1)
    leaf = x.clone().requires_grad_()
    want, = torch.autograd.grad(streamk.linear(leaf, w, bias, act, residual), leaf, dy)
    inner = leaf * 1
    bytes, y = kept_bytes(lambda: streamk.linear(inner, w, bias, act, residual))
    assert bytes == (2 * m * n if act else 0)
    before = torch.cuda.memory_allocated()
    del inner
    assert before - torch.cuda.memory_allocated() == 2 * m * k
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
    inner = leaf * 1
    y = streamk.linear(inner, w, bias, act, residual)
    inner.detach().zero_()
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
    # the weight alone, and the bias alone
    weight = w.clone().requires_grad_()
    want, = torch.autograd.grad(streamk.linear(x, weight, bias, act, residual), weight, dy)
    inner = weight * 1
    y = streamk.linear(x, inner, bias, act, residual)
    before = torch.cuda.memory_allocated()
    del inner
    assert before - torch.cuda.memory_allocated() == 2 * n * k
    assert torch.equal(torch.autograd.grad(y, weight, dy)[0], want)
    b = bias.clone().requires_grad_()
    want, = torch.autograd.grad(streamk.linear(x, w, b, act, residual), b, dy)
    copies = [x.clone(), w.clone()]
    y = streamk.linear(*copies, b, act, residual)
    before = torch.cuda.memory_allocated()
    del copies
    assert before - torch.cuda.memory_allocated() == 2 * (m + n) * k
    assert torch.equal(torch.autograd.grad(y, b, dy)[0], want)
    # what is needed is still looked at
    inner = x * 1
    y = streamk.linear(inner, weight, bias, act, residual)
    inner.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, weight, dy)


@gpu
@pytest.mark.parametrize("act", [None, "gelu"])
def test_compiled_passes_with_some_of_the_gradients(act):
    from torch.fx.experimental.proxy_tensor import make_fx
    m, n, k = 70, 72, 136
    for wanted in range(4):
        inputs = list(make(m, n, k, torch.bfloat16, 1))
        dy = inputs.pop()
        inputs[wanted].requires_grad_()

        def f(x, w, b, r):
            return streamk.linear(x, w, b, act, r, dropout=0.25, seed=7)

        want, = torch.autograd.grad(f(*inputs), inputs[wanted], dy)
        torch._dynamo.reset()
        compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
        assert torch.equal(torch.autograd.grad(compiled(*inputs), inputs[wanted], dy)[0], want)

        def step(x, w, b, r, dy):
            return torch.autograd.grad(f(x, w, b, r), (x, w, b, r)[wanted], dy)[0]

        assert torch.equal(make_fx(step)(*inputs, dy)(*inputs, dy), want)


@gpu
def test_refusals_of_the_gradients_by_themselves():
    x, w, bias, residual, dy = make(20, 24, 16, torch.float16, 1)
    grads = streamk._torch_binding.linear_full_grads
    slopes = torch.zeros(20, 24, dtype=torch.int16, device="cuda")
    want = (True, False, True)
    dx, dw, db = grads(dy, slopes, x, w, 1, 0.0, None, 0, *want)
    assert dx.shape == (20, 16) and dw is None and db.shape == (24,)
    for args in ((dy, None, x, w[:16], 0), (dy[:10], None, x, w, 0), (dy.bfloat16(), None, x, w, 0), (dy.cpu(), None, x, w, 0),
                 (dy, None, x, w[:, :8], 0), (dy, None, x, w, 1), (dy, slopes, x, w, 0), (dy, slopes[:10], x, w, 1)):
        with pytest.raises(ValueError):
            grads(*args, 0.0, None, 0, *want)
    with pytest.raises(ValueError):
        grads(dy, None, x, w, 0, 1.5, 1, 0, *want)


@gpu
def test_a_captured_pass_of_an_operator_beside_an_eager_graph_of_its_leaves():
    """The operators that compilers see look at all that gradients go to, as the eager functions do."""
    x, w, bias, residual, dy = make(70, 72, 136, torch.float16, 6)
    side = torch.cuda.Stream()
    full, dropout = torch.ops.marlin_amd.linear_full, torch.ops.marlin_amd.dropout

    def beside(leaf, forward, others):
        alive = forward()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                torch.autograd.grad(forward(), [leaf, *others], dy)
        torch.cuda.synchronize()
        assert torch.isfinite(torch.autograd.grad(alive, leaf, dy)[0]).all()

    for i in range(4):
        inputs = [x, w, bias, residual]
        inputs[i] = inputs[i].clone().requires_grad_()
        # (the residual's gradient alone takes no kernel: beside one that does, whose own graph is on the side stream)
        with torch.cuda.stream(side):
            other = bias.clone().requires_grad_()
        torch.cuda.synchronize()
        if i == 3:
            beside(inputs[3], lambda: full(x, w, other if torch.cuda.current_stream() == side else bias, inputs[3], 1, 0.0, 0,
                                           None, 0, True)[0], [other])
        else:
            beside(inputs[i], lambda: full(*inputs, 1, 0.0, 0, None, 0, True)[0], [])
    leaf = dy.clone().requires_grad_()
    beside(leaf, lambda: dropout(leaf, None, 0.5, 1, None, 0), [])


@gpu
@pytest.mark.parametrize("act", [None, "silu"])
def test_second_derivatives_raise_where_an_operand_is_not_kept(act):
    """Also where another path leads to the input that the backward pass has not kept."""
    m, n, k = 20, 24, 16
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        for leaf in (True, False):
            inputs = list(make(m, n, k, torch.float16, 1))
            dy = inputs.pop()
            roots = {i: inputs[i].requires_grad_() for i in wanted}
            if not leaf:
                for i in wanted:
                    inputs[i] = roots[i] * 1
            y = streamk.linear(*inputs[:3], act, inputs[3], dropout=0.25, seed=3)
            for i in wanted:
                g, = torch.autograd.grad(y, roots[i], dy, create_graph=True)
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(g.float().sum() + roots[i].float().sum(), roots[i], retain_graph=True)
