"""Dropout by a counter-based generator: feedforward.dropout, its C entry, and FeedForward's and Mlp's.

The mask's oracle is tests/_masks.py, and masks have to be equal.  What is kept is off by the fp32
factor's rounding, its product's and the addition's, each 2^-24 of a term, and one rounding to the type
(half a step e): bound e |want| + 2^-22 (|x| factor + |residual|).
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
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def least(t):  # half the smallest step of all
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[t]


def kept(shape, p, seed, site=0):
    keep, factor = _masks.mask(tuple(shape), p, seed, site)
    return torch.from_numpy(keep).cuda(), factor


def check(y, x, p, seed, site=0, residual=None):
    keep, factor = kept(x.shape, p, seed, site)
    v = torch.where(keep, x.double() * factor, torch.zeros((), dtype=torch.double, device="cuda"))
    r = 0 if residual is None else residual.double()
    want = v + r
    size = v.abs() + (0 if residual is None else r.abs())
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -6) + 2.0 ** -22 * size + least(x.dtype)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    assert ((y.double() - want).abs() <= bound).all()
    if residual is None:
        assert not y[~keep].any()
    else:
        assert torch.equal(y[~keep], residual.expand(x.shape)[~keep])


def make(shape, type, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=gen).to(type)


# --- without a GPU -------------------------------------------------------------------------

def test_the_oracle_gives_the_generators_known_answers():
    # of the generator's published test vectors: zeros, ones, digits of pi; seven and ten rounds
    ones, pi = 0xffffffff, (0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344)
    assert _masks.philox((0,) * 4, (0, 0), 7) == (0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48)
    assert _masks.philox((0,) * 4, (0, 0), 10) == (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)
    assert _masks.philox((ones,) * 4, (ones, ones), 10) == (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)
    assert _masks.philox(pi, (0xa4093822, 0x299f31d0), 10) == (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)


def test_the_oracle_by_elements_is_the_generator():
    for seed, site in ((0, 0), (-1, 2 ** 32 - 1), (0x123456789abcdef, 7)):
        got = _masks.bits(77, seed, site)
        key = (seed % 2 ** 32, seed % 2 ** 64 // 2 ** 32)
        for i in range(77):
            word = _masks.philox((i // 8, 0, site, 0), key, 7)[i % 8 // 2]
            assert int(got[i]) == word >> 16 * (i % 2) & 0xffff


def test_the_oracles_bits_are_even():
    draws = _masks.bits(1 << 20, 11, 3).astype(np.int64)
    # means and correlations of 2^20 numbers, six deviations wide
    assert abs((draws < 6554).mean() - 0.1) < 6 * (0.09 / 2 ** 20) ** 0.5
    unit = draws / 65536 - 0.5
    for lag in (1, 2, 7, 8, 64, 4096):
        assert abs((unit[lag:] * unit[:-lag]).mean() * 12) < 6 / 2 ** 10


def test_refusals():
    x = torch.zeros(4, 16)
    for args, kwargs, error, text in (
            ((x, 0.1, 1), {}, ValueError, "on the GPU"), ((x, 0.1, None), {}, ValueError, "needs a seed"),
            ((x, 0.1, 2 ** 63), {}, ValueError, "64 bits"), ((x, 0.1, "a"), {}, TypeError, "int"),
            ((None, 0.1, 1), {}, TypeError, "Tensor"), ((x, None, 1), {}, TypeError, "real number|float"),
            ((x, 0.1, 1), {"residual": 3}, TypeError, "Tensor"), ((x, 0.1, 1.5), {}, TypeError, "int")):
        with pytest.raises(error, match=text):
            feedforward.dropout(*args, **kwargs)
    with pytest.raises(ValueError, match="probability"):
        feedforward.Mlp(16, 16, dropout=1.5)
    with pytest.raises(ValueError, match="probability"):
        feedforward.FeedForward(16, 16, dropout=-0.1)
    with pytest.raises(ValueError, match="multiples of 8"):
        feedforward.Mlp(16, 12)
    with pytest.raises(ValueError, match="activation"):
        feedforward.Mlp(16, 16, "relu")


class DropArgs(ctypes.Structure):
    _fields_ = [("p", ctypes.c_double), ("seed", ctypes.c_longlong), ("seed_at", ctypes.c_void_p),
                ("site", ctypes.c_uint)]


def test_codes_of_the_entry():
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p

    def call(count, type=0, p=0.5, x=16, residual=None, y=16, seed_at=None):
        drop = DropArgs(p, 1, seed_at, 0)
        return lib.feedforward_dropout(P(x), P(residual), P(y), L(count), type, ctypes.byref(drop), 0, None)

    assert call(0) == 0 and call(0, x=None, y=None) == 0
    assert call(-1) == 1 and call(2 ** 34 + 1) == 1 and call(8, type=3) == 1
    for p in (-0.1, 1.1, float("nan"), float("inf")):
        assert call(0, p=p) == 1 and b"probability" in lib.feedforward_last_error()
    assert call(8, x=17) == 1 and call(8, residual=17) == 1 and call(8, y=18, type=2) == 1
    assert call(0, seed_at=12) == 1
    assert call(8, x=None) == 1 and call(8, y=None) == 1


def test_fake_tensors_record_the_operator():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, r):
        return torch.autograd.grad(feedforward.dropout(x, 0.1, 5, site=3, residual=r), (x, r), x)

    inputs = [torch.randn(4, 24).half().requires_grad_() for _ in range(2)]
    graph = make_fx(step, tracing_mode="fake")(*inputs)
    names = [str(n.target) for n in graph.graph.nodes if "marlin_amd" in str(n.target)]
    assert [n.split(".")[1] for n in names] == ["dropout", "dropout_grad"]


# --- on the GPU ----------------------------------------------------------------------------

SHAPES = [(1,), (7,), (8,), (9,), (2048,), (2049,), (3, 5, 7), (64, 1024), (777, 1033), (5, 8, 4096)]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, type):
    x, r = make(shape, type, 1), make(shape, type, 2)
    for p, seed, site in ((0.1, 0, 0), (0.5, -7, 3), (0.9, 2 ** 62 + 12345, 2 ** 32 - 1)):
        check(feedforward.dropout(x, p, seed, site=site), x, p, seed, site)
        check(feedforward.dropout(x, p, seed, site=site, residual=r), x, p, seed, site, r)


@gpu
@pytest.mark.parametrize("type", TYPES)
def test_probabilities_at_the_ends(type):
    x, r = make((33, 40), type, 1), make((33, 40), type, 2)
    for p in (0.0, 2.0 ** -18, 2.0 ** -16, 1 - 2.0 ** -16, 1.0):
        check(feedforward.dropout(x, p, 5), x, p, 5)
        check(feedforward.dropout(x, p, 5, residual=r), x, p, 5, residual=r)
    assert torch.equal(feedforward.dropout(x, 0, None), x)
    assert feedforward.dropout(x, 0, None) is not x
    assert not feedforward.dropout(x, 1, 5).any()


@gpu
def test_a_seed_on_the_gpu_is_that_number():
    x = make((100, 24), torch.bfloat16)
    for seed in (0, 1, -1, 2 ** 63 - 1, -2 ** 63, 0x123456789abcdef):
        want = feedforward.dropout(x, 0.3, seed, site=2)
        for shape in ((), (1,), (1, 1)):
            at = torch.full(shape, seed, dtype=torch.int64, device="cuda")
            assert torch.equal(feedforward.dropout(x, 0.3, at, site=2), want)
    many = torch.arange(10, device="cuda")
    assert torch.equal(feedforward.dropout(x, 0.3, many[3]), feedforward.dropout(x, 0.3, 3))


@gpu
def test_masks_of_other_seeds_and_sites_are_others():
    x = torch.ones(1 << 16, device="cuda")
    masks = [feedforward.dropout(x, 0.5, seed, site=site) != 0 for seed, site in ((0, 0), (1, 0), (2 ** 32, 0), (0, 1))]
    for i, a in enumerate(masks):
        for b in masks[:i]:
            assert abs((a == b).double().mean().item() - 0.5) < 6 * 0.5 / 2 ** 8


@gpu
@pytest.mark.parametrize("type", TYPES)
def test_what_is_dropped_may_be_anything(type):
    x = make((64, 40), type)
    keep, factor = kept(x.shape, 0.5, 9)
    clean = feedforward.dropout(x, 0.5, 9)
    for bad in (float("inf"), -float("inf"), float("nan")):
        dirty = torch.where(keep, x, torch.full_like(x, bad))
        assert torch.equal(feedforward.dropout(dirty, 0.5, 9), clean)
        leaf = x.clone().requires_grad_()
        dx, = torch.autograd.grad(feedforward.dropout(leaf, 0.5, 9), leaf, dirty)
        assert torch.equal(dx, clean)
        y = feedforward.dropout(torch.full_like(x, bad), 0.5, 9)
        assert not y[~keep].any() and not torch.isfinite(y[keep]).any()


@gpu
@pytest.mark.parametrize("type", TYPES)
def test_strides_and_alignment(type):
    base, more = make((40, 48), type), make((40, 48), type, 3)
    for pick in (lambda t: t[:, 8:32], lambda t: t.t(), lambda t: t[::2], lambda t: t.view(-1)[1:1001],
                 lambda t: t.view(-1)[3:], lambda t: t[0].expand(24, 48), lambda t: t.view(40, 6, 8).permute(1, 0, 2)):
        x, r = pick(base), pick(more)
        check(feedforward.dropout(x, 0.4, 6, residual=r), x, 0.4, 6, residual=r)
        check(feedforward.dropout(x, 0.4, 6), x, 0.4, 6)
        # (one of them off 16 bytes)
        check(feedforward.dropout(x, 0.4, 6, residual=r.clone()), x, 0.4, 6, residual=r)


@gpu
def test_nothing_beside_the_result_is_written():
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
    for count, start in ((1, 8), (7, 8), (8, 8), (2055, 8), (1000, 3)):
        for code, type in enumerate(TYPES):
            x = make((count,), type)
            room = torch.full((count + 64,), 7.0, dtype=type, device="cuda")
            y = room[start:start + count]
            drop = DropArgs(0.25, 3, None, 1)
            stream = P(torch.cuda.current_stream().cuda_stream)
            assert lib.feedforward_dropout(P(x.data_ptr()), None, P(y.data_ptr()), L(count), code, ctypes.byref(drop), 0,
                                           stream) == 0
            assert torch.equal(y, feedforward.dropout(x, 0.25, 3, site=1))
            assert (room[:start] == 7).all() and (room[start + count:] == 7).all()
            # in place, of x and of the residual
            for at in (x.clone(), None):
                into = at if at is not None else make((count,), type, 5)
                want = feedforward.dropout(x, 0.25, 3, site=1, residual=None if at is not None else into)
                assert lib.feedforward_dropout(P((at if at is not None else x).data_ptr()),
                                               P(None if at is not None else into.data_ptr()), P(into.data_ptr()), L(count),
                                               code, ctypes.byref(drop), 0, stream) == 0
                assert torch.equal(into, want)


@gpu
def test_more_elements_than_32_bits_of_bytes():
    x = torch.ones((1 << 31) + 8, dtype=torch.bfloat16, device="cuda")
    y = feedforward.dropout(x, 0.5, 21)
    del x
    # the groups of its last elements, by the generator itself
    for i in (0, 1 << 30, (1 << 31) - 8, 1 << 31):
        words = _masks.philox((i // 8, 0, 0, 0), (21, 0), 7)
        want = [2.0 if words[e // 2] >> 16 * (e % 2) & 0xffff >= 32768 else 0.0 for e in range(8)]
        assert y[i:i + 8].tolist() == want


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("shape", SHAPES[2:])
def test_gradients(shape, type):
    x, r, dy = (make(shape, type, s).requires_grad_(s != 3) for s in (1, 2, 3))
    for residual in (None, r):
        leaves = (x,) if residual is None else (x, r)
        y = feedforward.dropout(x, 0.3, 4, site=1, residual=residual)
        check(y.detach(), x.detach(), 0.3, 4, 1, None if residual is None else r.detach())
        grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        check(grads[0], dy, 0.3, 4, 1)
        if residual is not None:
            assert torch.equal(grads[1], dy)
            only, = torch.autograd.grad(y, r, dy)
            assert torch.equal(only, dy)
    # a gradient that is one value, and one to be read negated
    dx, = torch.autograd.grad(feedforward.dropout(x, 0.3, 4).sum(), x)
    check(dx, torch.ones_like(dx), 0.3, 4)
    dx, = torch.autograd.grad(feedforward.dropout(x, 0.3, 4), x, torch._neg_view(-dy))
    check(dx, dy, 0.3, 4)


@gpu
def test_gradients_against_differences():
    x, d = make((20, 24), torch.float32, 1).requires_grad_(), make((20, 24), torch.float32, 2)
    weight = make((20, 24), torch.float32, 3)

    def value(t):
        return (feedforward.dropout(t, 0.3, 8).double() * weight).sum()

    dx, = torch.autograd.grad(value(x), x)
    # linear: a difference is the derivative, but for the fp32 roundings of some 480 terms
    step = value((x + d).detach()) - value((x - d).detach())
    size = (2 * (x.abs() + d.abs()) * weight.abs() / 0.7).sum().item()
    assert abs(step.item() - 2 * (dx.double() * d).sum().item()) < 2.0 ** -21 * size


@gpu
def test_a_seed_that_was_written_is_noticed():
    x = make((16, 16), torch.float32).requires_grad_()
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    y = feedforward.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    # the tensors that are not looked at again may be written
    r = make((16, 16), torch.float32, 1).requires_grad_()
    a, b = x * 1, r * 1
    y = feedforward.dropout(a, 0.5, seed, residual=b)
    a.detach().zero_()
    b.detach().zero_()
    y.sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))


@gpu
def test_second_derivatives_and_forward_mode_raise():
    import torch.autograd.forward_ad as forward_ad
    x, dy = make((8, 16), torch.float32, 1).requires_grad_(), make((8, 16), torch.float32, 2).requires_grad_()
    g, = torch.autograd.grad(feedforward.dropout(x, 0.5, 1), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum() + (2 * dy).sum(), dy)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: feedforward.dropout(dual, 0.5, 1), lambda: feedforward.dropout(x, 0.5, 1, residual=dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@gpu
def test_refusals_on_the_gpu():
    x = make((4, 16), torch.float16)
    one = torch.ones(1, dtype=torch.int64, device="cuda")
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            feedforward.dropout(x, p, 1)
    for seed in (one.int(), torch.ones(2, dtype=torch.int64, device="cuda"), one.cpu(), one.float(),
                 torch.ones(0, dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="seed"):
            feedforward.dropout(x, 0.1, seed)
    for site in (-1, 2 ** 32):
        with pytest.raises(ValueError, match="site"):
            feedforward.dropout(x, 0.1, 1, site=site)
    for residual in (x.float(), x.cpu(), x[:2], x.view(16, 4)):
        with pytest.raises(ValueError, match="residual"):
            feedforward.dropout(x, 0.1, 1, residual=residual)
    for bad in (x.double(), x.int(), x.to_sparse()):
        with pytest.raises(ValueError, match="x must"):
            feedforward.dropout(bad, 0.1, 1)
    with pytest.raises(ValueError, match="plain"):
        feedforward.dropout(torch._neg_view(x), 0.1, 1)
    # nothing to do
    assert feedforward.dropout(x[:0], 0.1, 1).shape == (0, 16)
    e = x[:0].requires_grad_()
    assert torch.autograd.grad(feedforward.dropout(e, 0.1, 1, residual=e).sum(), e)[0].shape == (0, 16)


@gpu
def test_streams():
    x = make((1 << 22,), torch.bfloat16)
    want = [feedforward.dropout(x, 0.2, s) for s in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            got.append(feedforward.dropout(x, 0.2, s))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_captured_and_replayed_with_seeds_that_move_on():
    x, r, dy = (make((300, 40), torch.bfloat16, s) for s in (1, 2, 3))
    x.requires_grad_()
    seed = torch.full((1,), 100, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(feedforward.dropout(x, 0.3, seed, residual=r), x, dy)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = feedforward.dropout(x, 0.3, seed, residual=r)
        dx, = torch.autograd.grad(y, x, dy)
        seed.add_(1)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        eager = feedforward.dropout(x.detach(), 0.3, 100 + step, residual=r)
        assert torch.equal(y.detach(), eager) and torch.equal(dx, feedforward.dropout(dy, 0.3, 100 + step))
        assert seed.item() == 101 + step


@gpu
def test_recorded_and_compiled():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, r = make((20, 24), torch.float16, 1), make((20, 24), torch.float16, 2)
    seed = torch.full((1,), 17, dtype=torch.int64, device="cuda")

    def call(a, b):
        return feedforward.dropout(a, 0.3, 17, site=1, residual=b)

    def at(a, b):
        return feedforward.dropout(a, 0.3, seed, site=1, residual=b)

    want = call(x, r)
    graph = make_fx(call)(r, x)
    assert torch.equal(graph(x, r), want)
    assert torch.equal(torch.jit.trace(call, (r, x), check_trace=False)(x, r), want)
    leaves = [x.clone().requires_grad_(), r.clone().requires_grad_()]
    for f in (call, at):
        torch._dynamo.reset()
        compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
        assert torch.equal(compiled(x, r), want)
        got = torch.autograd.grad(compiled(*leaves), leaves, x)
        ref = torch.autograd.grad(call(*leaves), leaves, x)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))


@gpu
def test_blocks_with_dropout():
    """FeedForward and Mlp in training mode are the operators in their order; in eval mode nothing is
    dropped."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((3, 37, 64), device="cuda", generator=gen).bfloat16()
    block = feedforward.FeedForward(64, 136, dropout=0.2, device="cuda")
    plain = feedforward.FeedForward(64, 136, device="cuda")
    plain.load_state_dict(block.state_dict())
    y, r = block(x, next_weight=plain.pre_weight, seed=5, site=3)
    n, _ = feedforward.residual_norm(x, pre_weight=block.pre_weight)
    h = feedforward.dropout(streamk.gated(n, block.gate_up), 0.2, 5, site=6)
    z = feedforward.dropout(streamk.linear(h, block.down), 0.2, 5, site=7)
    want = feedforward.residual_norm(x, z, post_weight=block.post_weight, pre_weight=plain.pre_weight)
    # (there the product is rounded once more, before the mask's factor)
    for a, b in zip((y, r), want):
        assert (a.double() - b.double()).norm() <= 2 * 2.0 ** -8 * b.double().norm()
    with pytest.raises(ValueError, match="needs a seed"):
        block(x)
    block.eval()
    assert all(torch.equal(a, b) for a, b in zip(block(x)[1:], plain(x)[1:]))
    mlp = feedforward.Mlp(64, 136, dropout=0.2, device="cuda")
    with torch.no_grad():
        mlp.up_bias.normal_(generator=gen)
        mlp.down_bias.normal_(generator=gen)
    y, r = mlp(x, next_weight=plain.pre_weight, seed=5, site=3)
    n, _ = feedforward.residual_norm(x, pre_weight=mlp.pre_weight)
    h = streamk.linear(n, mlp.up, mlp.up_bias, "gelu", dropout=0.2, seed=5, site=6)
    want = streamk.linear(h, mlp.down, mlp.down_bias, residual=x, dropout=0.2, seed=5, site=7)
    assert torch.equal(r, want)
    assert torch.equal(y, feedforward.residual_norm(want, pre_weight=plain.pre_weight)[0])
    assert mlp(x, seed=5)[0] is None
    grads = torch.autograd.grad(r.float().sum(), list(mlp.parameters()))
    assert all(torch.isfinite(g).all() and g.any() for g in grads)
    with pytest.raises(ValueError, match="needs a seed"):
        mlp(x)
    mlp.eval()
    assert torch.equal(mlp(x)[1], mlp(x, seed=9)[1])
