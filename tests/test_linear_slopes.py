"""What a product with an activation keeps of it for its backward pass: slopes that are good relative to their size
also where a unit is far on the negative side, and the C entries that keep and take them.

The products here are with ones and zeros, so that their sums are the inputs exactly, or have a bias that
takes whole units far out.  Of a slope s are off, at most,
  by how it is kept: bfloat16 2^-8 |s| (a number of eight bits) or 2^-16 where that is less (steps of 2^-15), fp16
  2^-11 |s|, 2^-16 or, below 2^-16, 2^-27 (numbers of eleven bits down to 2^-16, steps of 2^-26 below);
  by its computation in fp32: with t the sigmoid's argument, 2^-24 (16 + 8 |t|) of it from z = -4 down (the argument is off
  by some 4 2^-24 |t|, the exponential's and reciprocal's own errors and the roundings are 8 of 2^-24, and where the slope
  is sigma (1 + z t' (1 - sigma)) with z t' below -4 the sum is at least 3/5 of its terms); elsewhere 2^-18;
and dz = dy s is rounded to the type once, e of it, half a step.
"""
import ctypes
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
import streamk  # noqa: E402

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
ACTS = ["silu", "gelu"]
BIG = [(160, 256), (192, 256), (224, 256), (256, 256)]
TILES = [(32, 32), (32, 64), (64, 64), (64, 128), (96, 128), (128, 128), (96, 256), (128, 256)] + BIG
FP32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):  # half the smallest step of all
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -134


def argument(z, act):
    """t and dt/dz of sigma(t)"""
    if act == "silu":
        return z, torch.ones_like(z)
    c = np.sqrt(8 / np.pi)
    return c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z * z)


def slope64(z, act):
    t, dt = argument(z, act)
    # (sigma (1 - sigma) without the difference)
    s, bend = torch.sigmoid(t), torch.sigmoid(t) * torch.sigmoid(-t)
    return s + z * dt * bend


def off_slope(z, act, type):
    """by how it is kept, and by its computation"""
    s = slope64(z, act).abs()
    if type == torch.bfloat16:
        kept = torch.minimum(2.0 ** -8 * s, torch.full_like(s, 2.0 ** -16))
    else:
        kept = torch.minimum(2.0 ** -11 * s, torch.full_like(s, 2.0 ** -16)).clamp(min=2.0 ** -27)
    t, _ = argument(z, act)
    return kept + torch.where(z <= -4, FP32 * (16 + 8 * t.abs()) * s, torch.full_like(s, 2.0 ** -18))


def farthest(act, type):
    """down to where slopes are 2^-57 (bfloat16) or nothing (fp16); sigma itself is then above 2^-126"""
    return {"silu": -40.0, "gelu": -8.0}[act] if type == torch.bfloat16 else {"silu": -24.0, "gelu": -6.5}[act]


def check_units(z, act, dy, grad):
    """grad = dy act'(z), element by element, z exact."""
    type, z = grad.dtype, z.double()
    want = dy.double() * slope64(z, act)
    bound = dy.double().abs() * off_slope(z, act, type)
    bound = (bound + half_step(type) * want.abs()) * (1 + 2.0 ** -6) + least(type)
    err = (grad.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # A slope above 2^-22 is kept in fp16, off by 2^-27 (a thirty-second), and its product with dy is something wherever it
    # is above 2^-25, half fp16's smallest step: where it is to be 2^-24.  In bfloat16 all slopes here are kept.
    there = (want.abs() > 2.0 ** -22 * dy.double().abs()) & (want.abs() > 2.0 ** -24) if type == torch.float16 else want != 0
    assert (grad[there] != 0).all()


def values(m, n, act, type, seed):
    """From far on the negative side to where slopes are one."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lo = farthest(act, type)
    return (lo + (8 - lo) * torch.rand((m, n), device="cuda", generator=gen)).to(type)


def gradient(z, act, dy):
    eye = torch.eye(z.shape[1], device="cuda").to(z.dtype)
    leaf = z.clone().requires_grad_()
    return torch.autograd.grad(streamk.linear(leaf, eye, None, act), leaf, dy)[0]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 16, 50, 300])
def test_slopes_of_every_size(m, act, type):
    z = values(m, 264, act, type, m)
    for size in (1.0, 4.0, -3.0):
        dy = torch.full_like(z, size)
        check_units(z, act, dy, gradient(z, act, dy))


@gpu
@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("tile", [(16, 16), (16, 32)] + TILES)
def test_slopes_of_every_size_by_every_tile(tile, slices):
    for type in TYPES:
        for act in ACTS:
            m = 50 if tile[0] == 16 else 333
            z, dy = values(m, 520, act, type, 3), torch.ones((m, 520), dtype=type, device="cuda")
            eye = torch.eye(520, device="cuda").to(type)
            leaf = z.clone().requires_grad_()
            try:
                streamk.force_product_tile(*tile, slices)
                y = streamk.linear(leaf, eye, None, act)
            finally:
                streamk.force_product_tile(0)
            check_units(z, act, dy, torch.autograd.grad(y, leaf, dy)[0])


FAR = [("silu", -4, 0.3), ("silu", -8, 1), ("silu", -12, 1), ("silu", -14, 1), ("gelu", -3.5, 0.2), ("gelu", -4.5, 0.3),
       ("gelu", -5, 0.25)]
FARTHER = [("silu", -16, 0.5), ("gelu", -7, 0.3)]  # (of these dz is below fp16's range)


@gpu
@pytest.mark.parametrize("m", [40, 300])
@pytest.mark.parametrize("act,mean,width,type", [(*unit, type) for type in TYPES for unit in FAR + FARTHER * (type == torch.bfloat16)])
def test_gradients_of_units_far_on_the_negative_side(m, act, mean, width, type):
    n, k = 72, 64
    gen = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn((m, k), device="cuda", generator=gen).to(type)
    w = (torch.randn((n, k), device="cuda", generator=gen) * width * k ** -0.5).to(type)
    bias = torch.full((n,), float(mean), device="cuda").to(type)
    dy = torch.randn((m, n), device="cuda", generator=gen).to(type)
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    dx, dw, db = torch.autograd.grad(streamk.linear(*leaves, act), leaves, dy)
    x, w, bias = (t.detach().double() for t in leaves)
    z = x @ w.t() + bias
    off_z = (k + 1) * FP32 * (x.abs() @ w.abs().t() + bias.abs())
    _, dt = argument(z - off_z, act)
    # |act''| is below |act'| (2 t' + 1) here: act' = sigma (1 + z t' (1 - sigma)), z t' below -4
    off = off_slope(z, act, type) + off_z * (2 * dt + 1) * slope64(z, act).abs()
    assert (z < -2.4).all()
    d, e = dy.double(), half_step(type)
    dz = d * slope64(z, act)
    assert dz.abs().max() < 0.5

    def within(got, want, bound):
        bound = (bound + e * want.abs()) * (1 + 2.0 ** -6) + least(type)
        err = (got.double() - want).abs()
        assert (err <= bound).all(), float((err / bound).max())

    within(db, dz.sum(0), (d.abs() * off).sum(0) + m * FP32 * dz.abs().sum(0))
    off = d.abs() * off + e * dz.abs() + least(type)
    within(dx, dz @ w, off @ w.abs() + n * FP32 * (dz.abs() @ w.abs()))
    within(dw, dz.t() @ x, off.t() @ x.abs() + m * FP32 * (dz.abs().t() @ x.abs()))
    assert (dw != 0).float().mean() > 0.9


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_slopes_that_are_exact(act):
    """Zero and one: far out on either side, and what a signed zero gives."""
    for type in TYPES:
        for size in (64.0, 200.0, float(torch.finfo(type).max) / 4):
            z = torch.full((3, 264), size, dtype=type, device="cuda")
            dy = torch.full_like(z, 1.5)
            assert torch.equal(gradient(z, act, dy), dy)
            assert not gradient(-z if act == "gelu" or size > 100 else torch.full_like(z, -200), act, dy).any()


@gpu
@pytest.mark.parametrize("m", [3, 300])
def test_nan_of_any_payload(m):
    for type, codes in ((torch.float16, (0x7e00, 0x7e01, 0x7fff, 0x7d55, -0x200, -1)),
                        (torch.bfloat16, (0x7fc0, 0x7fc1, 0x7fff, 0x7fd5, -0x40, -1))):
        for act in ACTS:
            z = torch.zeros((m, 72), dtype=type, device="cuda")
            for i, code in enumerate(codes):
                z.view(torch.int16)[m - 1, 8 * i] = code
            w = torch.ones((72, 72), dtype=type, device="cuda")
            leaf = z.clone().requires_grad_()
            g, = torch.autograd.grad(streamk.linear(leaf, w, None, act), leaf, torch.ones_like(z))
            assert g[m - 1].isnan().all() and torch.isfinite(g[:m - 1]).all()


# --- the C entries -------------------------------------------------------------------------

class DropArgs(ctypes.Structure):
    _fields_ = [("p", ctypes.c_double), ("seed", ctypes.c_longlong), ("seed_at", ctypes.c_void_p),
                ("site", ctypes.c_uint)]


P, L = ctypes.c_void_p, ctypes.c_longlong


def test_codes_of_the_entries():
    lib = streamk._lib

    def linear(entry, m=0, n=8, k=8, x=16, slopes=None, lds=8, type=0, act=0, p=None):
        drop = None if p is None else ctypes.byref(DropArgs(p, 0, None, 0))
        return entry(P(x), P(16), P(16), None, None, P(slopes), m, n, k, L(8), L(8), L(8), L(8), L(lds), type, act, drop,
                     None, L(0), 0, None)

    def grad(entry, m=0, n=8, dy=16, slopes=None, dz=16, dbias=None, lds=8, type=0, p=None, partials=None, count=0):
        drop = None if p is None else ctypes.byref(DropArgs(p, 0, None, 0))
        factor = [None] if entry == lib.feedforward_linear_backward else []
        return entry(P(dy), P(slopes), P(dz), P(dbias), m, n, L(8), L(lds), L(8), type, drop, P(partials), L(count), *factor,
                     0, None)

    for entry in (lib.feedforward_linear, lib.feedforward_linear_train):
        assert linear(entry) == 0 and linear(entry, slopes=16, act=2, p=0.5) == 0
        for bad in (dict(m=-1), dict(n=12), dict(type=2), dict(act=3), dict(x=8), dict(slopes=8, act=1),
                    dict(slopes=16, act=1, lds=4), dict(slopes=16), dict(p=2.0), dict(m=4, x=None)):
            assert linear(entry, **bad) == 1, bad
    for entry in (lib.feedforward_linear_grad, lib.feedforward_linear_backward):
        assert grad(entry) == 0 and grad(entry, slopes=16, p=0.5) == 0
        for bad in (dict(m=-1), dict(n=12), dict(type=2), dict(slopes=8), dict(slopes=16, lds=4), dict(p=-1.0),
                    dict(m=4, dy=None), dict(m=4, dz=None), dict(m=4096, dbias=16)):
            assert grad(entry, **bad) == 1, bad


def by_entries(forward, backward, x, w, bias, act, dy):
    """y, dz and dbias"""
    lib, (m, k), n, dev = streamk._lib, x.shape, len(w), x.device
    code, stream = int(x.dtype == torch.bfloat16), P(torch.cuda.current_stream().cuda_stream)
    y, dz = torch.empty((m, n), dtype=x.dtype, device=dev), torch.empty((m, n), dtype=x.dtype, device=dev)
    slopes = torch.empty((m, n), dtype=torch.int16, device=dev)
    db = torch.empty(n, dtype=x.dtype, device=dev)
    lib.feedforward_linear_grad_bytes.restype = L
    sums = torch.empty(max(lib.feedforward_linear_grad_bytes(m, n), 4), dtype=torch.uint8, device=dev)
    assert forward(P(x.data_ptr()), P(w.data_ptr()), P(y.data_ptr()), P(bias.data_ptr()), None, P(slopes.data_ptr()), m, n, k,
                   L(k), L(k), L(n), L(0), L(n), code, {"silu": 1, "gelu": 2}[act], None, None, L(0), 0, stream) == 0
    factor = [None] if backward == lib.feedforward_linear_backward else []
    assert backward(P(dy.data_ptr()), P(slopes.data_ptr()), P(dz.data_ptr()), P(db.data_ptr()), m, n, L(n), L(n), L(n), code,
                    None, P(sums.data_ptr()), L(sums.numel()), *factor, 0, stream) == 0
    return y, dz, db


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 50, 300])
def test_entries_of_either_form(m, act, type):
    n = 264
    z = values(m, n, act, type, m)
    eye, zero = torch.eye(n, device="cuda").to(type), torch.zeros(n, dtype=type, device="cuda")
    dy = torch.randn((m, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(type)
    lib = streamk._lib
    y, dz, db = by_entries(lib.feedforward_linear_train, lib.feedforward_linear_backward, z, eye, zero, act, dy)
    check_units(z, act, dy, dz)
    y2, dz2, db2 = by_entries(lib.feedforward_linear, lib.feedforward_linear_grad, z, eye, zero, act, dy)
    assert torch.equal(y, y2)
    # in steps of 2^-15: half a step of the slope, 2^-18 of its computation, one rounding
    d, s = dy.double(), slope64(z.double(), act)
    want, e = d * s, half_step(type)
    bound = (d.abs() * (2.0 ** -16 + 2.0 ** -18) + e * want.abs()) * (1 + 2.0 ** -6) + least(type)
    assert ((dz2.double() - want).abs() <= bound).all()
    for got, off in ((db, off_slope(z.double(), act, type)), (db2, 2.0 ** -16 + 2.0 ** -18)):
        total = want.sum(0)
        bound = (d.abs() * off).sum(0) + m * FP32 * want.abs().sum(0) + e * total.abs()
        assert ((got.double() - total).abs() <= bound * (1 + 2.0 ** -6) + least(type)).all()
