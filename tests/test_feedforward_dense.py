"""Dense products of the feed-forward block and their gradients: streamk.gated, streamk.linear.

The oracle is the definition in 64 bits on the rounded inputs.  Bounds, element by element, with e
half a step of the type (2^-11 fp16, 2^-8 bf16), S the sum of a product's magnitudes:
  a sum of k products in fp32 is off by at most k 2^-24 S, a result rounded to the type by e of it;
  the activations' slopes stay below 1.13, their second derivatives below 1, and in fp32 they are
  off by less than 2^-18 of their size (an exponential whose argument is good to 2^-24 of itself);
  for the gradients dg and du are rounded to the type.
"""
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
FP32 = 2.0 ** -24
ACT = 2.0 ** -18


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):  # half the smallest step of all
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -134


def act64(g, name):
    """value and slope"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    z = np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
    t = torch.tanh(z)
    return g / 2 * (1 + t), (1 + t) / 2 + g / 2 * (1 - t * t) * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * g * g)


def make(m, n, k, type, seed, dev="cuda", rows=None):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device=dev, generator=gen) * std).to(type)

    return randn(m, k), randn(rows or 2 * n, k, std=k ** -0.5), randn(m, n)


def within(got, want, bound, type, parts=1.5):
    bound = bound * (1 + 2.0 ** -6) + least(type)  # (roundings of what is off already)
    err = (got.double() - want).abs()
    assert got.dtype == type and got.shape == want.shape and torch.isfinite(got).all()
    assert (err <= bound).all(), float((err / bound).max())
    # roundings are independent of each other: together they stay near one of them
    assert err.norm() <= parts * half_step(type) * want.norm() + least(type) * want.numel() ** 0.5


class Gated64:
    def __init__(self, x, w, act):
        n, self.k = w.shape[0] // 2, w.shape[1]
        self.x, self.wg, self.wu = x.double(), w[:n].double(), w[n:].double()
        self.g, self.u = self.x @ self.wg.t(), self.x @ self.wu.t()
        self.sg, self.su = self.x.abs() @ self.wg.abs().t(), self.x.abs() @ self.wu.abs().t()
        self.value, self.slope = act64(self.g, act)

    def check_forward(self, h, type):
        dg, du = self.k * FP32 * self.sg, self.k * FP32 * self.su
        want = self.value * self.u
        bound = 1.13 * dg * (self.u.abs() + du) + self.value.abs() * du + (half_step(type) + 2 * ACT) * want.abs()
        within(h, want, bound, type, 1.01)

    def check_grads(self, dh, dx, dw, type):
        e, d = half_step(type), dh.double()
        eg, eu = self.k * FP32 * self.sg, self.k * FP32 * self.su
        g, u = d * self.u * self.slope, d * self.value
        off_g = d.abs() * ((self.u.abs() + eu) * (eg + ACT) + 1.13 * eu) + e * g.abs() + least(type)
        off_u = d.abs() * (1.13 * eg + ACT * self.value.abs()) + e * u.abs() + least(type)
        n2, m = 2 * self.g.shape[1], self.x.shape[0]
        if dx is not None:
            want = g @ self.wg + u @ self.wu
            size = g.abs() @ self.wg.abs() + u.abs() @ self.wu.abs()
            bound = off_g @ self.wg.abs() + off_u @ self.wu.abs() + n2 * FP32 * size + e * want.abs()
            within(dx, want, bound, type)
        if dw is not None:
            want = torch.cat([g.t() @ self.x, u.t() @ self.x])
            ax = self.x.abs()
            size = torch.cat([g.abs().t() @ ax, u.abs().t() @ ax])
            bound = torch.cat([off_g.t() @ ax, off_u.t() @ ax]) + m * FP32 * size + e * want.abs()
            within(dw, want, bound, type)


def check_product(got, a, b, type):
    """got = a @ b.T"""
    a, b = a.double(), b.double()
    want = a @ b.t()
    bound = a.shape[1] * FP32 * (a.abs() @ b.abs().t()) + half_step(type) * want.abs()
    within(got, want, bound, type, 1.01)


# --- without a GPU -------------------------------------------------------------------------

def test_refuses_host_tensors_and_unknown_activations():
    x, w = torch.zeros(2, 16).half(), torch.zeros(32, 16).half()
    with pytest.raises(ValueError, match="on the GPU"):
        streamk.gated(x, w)
    with pytest.raises(ValueError, match="on the GPU"):
        streamk.linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        streamk.gated(x, w, "relu")
    with pytest.raises(TypeError, match="Tensor"):
        streamk.linear(None, w)


def test_refuses_forward_mode():
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.zeros(2, 16).half(), torch.zeros(32, 16).half()
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, x), w), (x, forward_ad.make_dual(w, w))):
            for call in (streamk.gated, streamk.linear):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)


@pytest.mark.parametrize("m,n,k,lda,ldb,ldc,type,code", [
    (-1, 8, 8, 8, 8, 8, 0, 1), (4, 12, 8, 8, 8, 16, 0, 1), (4, 8, 12, 16, 16, 8, 0, 1), (4, 8, 8, 8, 8, 8, 2, 1),
    (4, 8, 16, 8, 16, 8, 0, 1), (4, 8, 16, 20, 16, 8, 0, 1), (4, 8, 16, 16, 16, 4, 0, 1), (4, 8, 0, 8, 8, 8, 0, 1),
    (4, 8, 16, 1 << 22, 16, 8, 0, 1), (0, 8, 16, 16, 16, 8, 0, 0), (4, 0, 16, 16, 16, 8, 1, 0)])
def test_codes_of_the_entries(m, n, k, lda, ldb, ldc, type, code):
    import ctypes
    lib, L = streamk._lib, ctypes.c_longlong
    rc = lib.feedforward_product(None, None, None, m, n, k, L(lda), L(ldb), L(ldc), 0, type, None, L(0), 0, None)
    assert rc == code
    rc = lib.feedforward_gated(None, None, None, None, m, n, k, L(lda), L(ldb), L(ldc), L(2 * ldc), type, 1, None, L(0),
                               0, None)
    assert rc == code
    assert (len(lib.feedforward_last_error()) > 0) or code == 0


@pytest.mark.parametrize("m,n,k,lda,ldb,turned,code", [
    (0, 8, 16, 16, 8, 1, 0), (0, 8, 16, 8, 8, 1, 1), (0, 16, 16, 16, 8, 1, 1),  # B: k rows of n
    (0, 8, 13, 8, 8, 2, 0), (8, 0, 13, 8, 8, 2, 0), (8, 0, 13, 0, 8, 2, 1), (12, 0, 8, 16, 8, 2, 1),  # A: k rows of m
    (0, 8, 64, 64, 64, 3, 1), (0, 8, 64, 64, 64, 5, 1), (0, 8, 64, 64, 64, -1, 1)])
def test_codes_of_the_layouts(m, n, k, lda, ldb, turned, code):
    import ctypes
    lib, L = streamk._lib, ctypes.c_longlong
    rc = lib.feedforward_product(None, None, None, m, n, k, L(lda), L(ldb), L(n), turned, 0, None, L(0), 0, None)
    assert rc == code
    # scratch off 16 bytes
    assert lib.feedforward_product(ctypes.c_void_p(16), ctypes.c_void_p(16), ctypes.c_void_p(16), 8, 8, 8, L(8), L(8),
                                   L(8), 0, 0, ctypes.c_void_p(8), L(1024), 0, None) == 1


def test_codes_of_the_gradients():
    import ctypes
    lib, L = streamk._lib, ctypes.c_longlong

    def grad(m, n, lddh, ldpre, lddgu, type=0, act=1, dgu=16):
        return lib.feedforward_gated_grad(None, None, ctypes.c_void_p(dgu), m, n, L(lddh), L(ldpre), L(lddgu), type, act,
                                          0, None)

    assert grad(0, 40, 40, 96, 128) == 0
    assert grad(0, 40, 40, 96, 80) == 0
    assert grad(0, 40, 40, 96, 72) == 1
    assert grad(0, 40, 32, 96, 128) == 1
    assert grad(0, 40, 40, 88, 128) == 1      # 48 columns of gates and ups in turns of sixteen
    assert grad(0, 40, 40, 96, 128, act=0) == 1
    assert grad(0, 40, 40, 96, 128, type=5) == 1
    assert grad(0, 40, 40, 96, 128, dgu=8) == 1  # off 16 bytes
    # more than 2 GiB of a gated product's weights
    rc = lib.feedforward_gated(None, None, None, None, 1, 1 << 20, 1024, L(1024), L(1024), L(1 << 20), L(1 << 21), 0, 1,
                               None, L(0), 0, None)
    assert rc == 1 and b"2 GiB" in lib.feedforward_last_error()


def test_codes_of_missing_matrices_and_too_many_rows():
    import ctypes
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p

    def product(a, b, c, m=4):
        return lib.feedforward_product(a, b, c, m, 8, 8, L(8), L(8), L(8), 0, 0, None, L(0), 0, None)

    there = P(16)
    for t in ((None, there, there), (there, None, there), (there, there, None)):
        assert product(*t) == 1 and b"missing" in lib.feedforward_last_error()
    assert product(there, there, there, 0x7fffffff) == 1 and b"too many" in lib.feedforward_last_error()
    for t in ((None, there, there), (there, None, there), (there, there, None)):
        assert lib.feedforward_gated_grad(*t, 4, 16, L(16), L(32), L(64), 0, 1, 0, None) == 1
        assert b"missing" in lib.feedforward_last_error()


TILES = [(64, 64), (64, 128), (96, 128), (128, 128), (96, 256), (128, 256), (160, 256), (192, 256), (224, 256), (256, 256)]


def test_plans_of_nothing():
    with pytest.raises(ValueError, match="compute units"):
        streamk.product_plan(8, 8, 8, cus=0)
    with pytest.raises(ValueError, match="layout"):
        streamk.product_plan(8, 8, 8, turned=3)
    with pytest.raises(ValueError, match="4 MiB"):
        streamk.product_plan(8, (1 << 21) + 8, 8, gated=True)
    assert streamk.product_plan(0, 8, 8) is None and streamk.product_plan(8, 8, 8, cus=1) is not None


FEW = [(rows, cols) for rows in (16, 32, 48, 64) for cols in (16, 32)]


def test_plans_are_tiles_that_can_compute_the_problem():
    seen = set()
    rng = np.random.default_rng(0)
    for _ in range(8000):
        m, n, k = (int(2 ** rng.uniform(*r)) for r in ((0, 14), (3, 14), (3, 14)))
        n, k = 8 * max(1, n // 8), 8 * max(1, k // 8)
        for gated, turned in ((False, 0), (True, 0), (False, 1), (False, 2)):
            if turned == 2:
                m, k = 8 * max(1, m // 8), m
            t = streamk.product_plan(m, n, k, gated, turned)
            rows, cols, slices = t
            if cols <= 32:  # whole columns of all rows
                assert turned == 0 and m <= 64 and rows == -(-m // 16) * 16 and slices == 1
                seen.add(((rows, cols), 1))
            else:
                assert (rows, cols) in TILES and 1 <= slices <= min(8, -(-k // 64))
                assert rows != 96 or turned != 2
                seen.add(((rows, cols), min(slices, 2)))
            if turned == 2:
                m, k = k, m
    assert {t for t, _ in seen} == set(TILES + FEW)  # none that nothing reaches


# --- on the GPU ----------------------------------------------------------------------------

# up to 64 rows by blocks of columns; the tiles; depths and widths that nothing divides
FORWARD = [(1, 8, 8), (1, 10752, 4096), (2, 40, 72), (7, 1032, 520), (16, 5208, 4160), (17, 2744, 1032), (33, 24, 8),
           (40, 8200, 1096), (48, 16, 4096), (64, 4104, 968), (65, 8, 8), (65, 72, 136), (100, 1000, 1000),
           (300, 520, 4160), (777, 5208, 4160), (1025, 264, 64), (2100, 1544, 192)]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("m,n,k", FORWARD)
def test_forward(m, n, k, type):
    x, w, _ = make(m, n, k, type, m + n + k)
    for act in ("silu", "gelu"):
        Gated64(x, w, act).check_forward(streamk.gated(x, w, act), type)
    check_product(streamk.linear(x, w), x, w, type)


@gpu
@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k", [(1, 8, 64), (300, 520, 192), (257, 136, 1096), (130, 264, 128), (333, 304, 640)])
def test_every_tile(tile, m, n, k, slices):
    try:
        streamk.force_product_tile(*tile, slices)
        for type in TYPES:
            x, w, dh = make(m, n, k, type, 5)
            x.requires_grad_()
            w.requires_grad_()
            ref = Gated64(x.detach(), w.detach(), "gelu")
            ref.check_forward(streamk.gated(x.detach(), w.detach(), "gelu"), type)
            h = streamk.gated(x, w, "gelu")
            ref.check_forward(h.detach(), type)
            ref.check_grads(dh, *torch.autograd.grad(h, (x, w), dh), type)
            y = streamk.linear(x, w[:n])
            check_product(y.detach(), x.detach(), w[:n].detach(), type)
            dx, dw = torch.autograd.grad(y, (x, w), dh)
            check_product(dx, dh, w[:n].detach().t(), type)
            check_product(dw[:n], dh.t(), x.detach().t(), type)
    finally:
        streamk.force_product_tile(0)


@gpu
@pytest.mark.parametrize("cols", [16, 32])
@pytest.mark.parametrize("m,n,k", FORWARD[:10])
def test_whole_columns_of_few_rows(m, n, k, cols):
    try:
        streamk.force_product_tile(16, cols)
        for type in TYPES:
            x, w, _ = make(m, n, k, type, m + n)
            Gated64(x, w, "silu").check_forward(streamk.gated(x, w), type)
            check_product(streamk.linear(x, w), x, w, type)
    finally:
        streamk.force_product_tile(0)


@gpu
@pytest.mark.parametrize("turned", [0, 1, 2])
def test_layouts_beside_rows_that_hold_nan(turned):
    """Matrices inside larger ones: what lies beside them, and behind their last row, is NaN."""
    import ctypes
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
    for tile in (0, (16, 16), (16, 32), (64, 64), (128, 128), (128, 256), (160, 256), (256, 256)):
        for m, n, k in ((72, 200, 136), (328, 264, 320), (64, 24, 56)):
            gen = torch.Generator(device="cuda").manual_seed(m)
            a, b = (torch.randn(r, k, device="cuda", generator=gen).half() for r in (m, n))

            def inside(x):
                rows, cols = x.shape
                room = torch.full((rows + 80, cols + 96), float("nan"), dtype=torch.float16, device="cuda")
                room[8:8 + rows, 16:16 + cols] = x
                return room, room[8:8 + rows, 16:16 + cols]

            ra, va = inside(a.t().contiguous() if turned == 2 else a)
            rb, vb = inside(b.t().contiguous() if turned else b)
            rc, vc = inside(torch.zeros(m, n, device="cuda").half())
            before = rc.clone()
            room = torch.empty(3 * m * n, device="cuda")
            try:
                streamk.force_product_tile(*(tile if tile else (0,)), slices=2 if m == 328 and tile else 0)
                code = lib.feedforward_product(P(va.data_ptr()), P(vb.data_ptr()), P(vc.data_ptr()), m, n, k, L(va.stride(0)),
                                               L(vb.stride(0)), L(vc.stride(0)), turned, 0, P(room.data_ptr()),
                                               L(4 * room.numel()), 0, P(torch.cuda.current_stream().cuda_stream))
            finally:
                streamk.force_product_tile(0)
            assert code == 0
            check_product(vc, a, b, torch.float16)
            vc.copy_(before[8:8 + m, 16:16 + n])
            assert torch.equal(rc.isnan(), before.isnan()) and not rc.nan_to_num().any()  # nothing else was written


GRADS = [(1, 8, 8), (3, 40, 72), (65, 64, 64), (64, 520, 136), (200, 1032, 264), (777, 200, 1000), (1237, 2744, 1032),
         (2048, 512, 512)]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("m,n,k", GRADS)
def test_gradients(m, n, k, type):
    x, w, dh = make(m, n, k, type, m * n + k)
    x.requires_grad_()
    w.requires_grad_()
    for act in ("silu", "gelu"):
        h = streamk.gated(x, w, act)
        ref = Gated64(x.detach(), w.detach(), act)
        ref.check_forward(h.detach(), type)
        dx, dw = torch.autograd.grad(h, (x, w), dh)
        ref.check_grads(dh, dx, dw, type)
    y = streamk.linear(x, w[:n])
    dx, dw = torch.autograd.grad(y, (x, w), dh)
    check_product(y.detach(), x.detach(), w[:n].detach(), type)
    check_product(dx, dh, w[:n].detach().t(), type)
    check_product(dw[:n], dh.t(), x.detach().t(), type)
    assert not dw[n:].any()


@gpu
def test_gradients_against_differences():
    """The loss sum(h c) along a direction, by differences of the definition in 64 bits: the step t
    leaves a relative t^2 of the third derivative and 2^-52 / t of cancellation."""
    m, n, k = 24, 40, 48
    for act in ("silu", "gelu"):
        x, w, c = make(m, n, k, torch.float16, 3)
        x.requires_grad_()
        w.requires_grad_()
        dx, dw = torch.autograd.grad(streamk.gated(x, w, act), (x, w), c)
        gen = torch.Generator(device="cuda").manual_seed(4)
        vx = torch.randn(x.shape, device="cuda", generator=gen, dtype=torch.float64)
        vw = torch.randn(w.shape, device="cuda", generator=gen, dtype=torch.float64) * k ** -0.5

        def loss(t):
            xd, wd = x.detach().double() + t * vx, w.detach().double() + t * vw
            return (act64(xd @ wd[:n].t(), act)[0] * (xd @ wd[n:].t()) * c.double()).sum()

        t = 1e-4
        slope = (loss(t) - loss(-t)) / (2 * t)
        terms = torch.cat([(dx.double() * vx).flatten(), (dw.double() * vw).flatten()])
        # every term of the inner product is off by some half steps: 6 of them, as independent errors
        assert (terms.sum() - slope).abs() <= 6 * 2.0 ** -11 * 3 * terms.norm() + 1e-5 * terms.abs().sum()


@gpu
def test_only_the_gradients_that_are_wanted():
    x, w, dh = make(70, 72, 136, torch.bfloat16, 1)
    both = [t.clone().requires_grad_() for t in (x, w)]
    dx, dw = torch.autograd.grad(streamk.gated(*both), both, dh)
    xg = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(streamk.gated(xg, w), xg, dh)[0], dx)
    wg = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(streamk.gated(x, wg), wg, dh)[0], dw)
    with torch.no_grad():
        assert not streamk.gated(xg, wg).requires_grad
    assert torch.equal(streamk.gated(x, w), streamk.gated(xg, wg).detach())


@gpu
@pytest.mark.parametrize("m", [5, 200])
def test_strides_alignment_and_shapes(m):
    n, k = 72, 136
    x, w, dh = make(m, n, k, torch.float16, 2)
    want, want_y = streamk.gated(x, w), streamk.linear(x, w)
    wide = torch.full((m, k + 24), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 8:8 + k] = x
    deep = torch.full((2 * n, k + 8), float("nan"), dtype=torch.float16, device="cuda")
    deep[:, :k] = w
    room = torch.empty(x.numel() + 1, dtype=torch.float16, device="cuda")[1:].view(x.shape).copy_(x)
    for a in (x, wide[:, 8:8 + k], x.t().contiguous().t(), room):
        for b in (w, deep[:, :k], w.t().contiguous().t()):
            assert torch.equal(streamk.gated(a, b), want)
            assert torch.equal(streamk.linear(a, b), want_y)
            a_, b_ = a.detach().requires_grad_(), b.detach().requires_grad_()
            for got, ref in zip(torch.autograd.grad(streamk.gated(a_, b_), (a_, b_), dh),
                                torch.autograd.grad(streamk.gated(x.requires_grad_(), w.requires_grad_()), (x, w), dh)):
                assert torch.equal(got, ref)
            x, w = x.detach(), w.detach()
    assert torch.equal(streamk.gated(x.view(1, m, k), w), want.view(1, m, n))
    assert streamk.gated(x[0], w).shape == (n,)
    # a gradient that is one value everywhere has no strides
    x.requires_grad_()
    w.requires_grad_()
    one = torch.autograd.grad(streamk.gated(x, w).float().sum(), (x, w))
    ones = torch.autograd.grad(streamk.gated(x, w), (x, w), torch.ones((m, n), dtype=torch.float16, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(one, ones))


@gpu
def test_rows_further_apart_than_the_kernels_address():
    x, w, _ = make(3, 16, 64, torch.float16, 4)
    room = torch.zeros(3, (1 << 21) + 8, dtype=torch.float16, device="cuda")
    room[:, :64] = x
    assert torch.equal(streamk.linear(room[:, :64], w), streamk.linear(x, w))
    assert torch.equal(streamk.gated(room[:, :64], w), streamk.gated(x, w))


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements of x, of both sums and of their gradients; the last rows and the sums
    over all of them."""
    m, n, k = 1050000, 1024, 2064
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 1 << 31 and 2 * n * m > 1 << 31
    x.normal_(generator=gen)
    w = torch.randn(2 * n, k, device="cuda", generator=gen).mul_(k ** -0.5).bfloat16()
    dh = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    last = slice(m - 300, m)
    dh[last].normal_(generator=gen)
    x.requires_grad_()
    w.requires_grad_()
    h = streamk.gated(x, w)
    ref = Gated64(x.detach()[last], w.detach(), "silu")
    ref.check_forward(h.detach()[last], torch.bfloat16)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    # (only the last rows have a gradient: the others add exact zeros to that of w)
    ref.check_grads(dh[last], dx[last], dw, torch.bfloat16)
    assert not dx[:m - 300].any()


@gpu
def test_empty():
    x, w, _ = make(0, 72, 136, torch.float16, 2)
    x.requires_grad_()
    w.requires_grad_()
    for y in (streamk.gated(x, w), streamk.linear(x, w)):
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == (0, 136) and not dw.any()
    assert streamk.linear(torch.zeros(3, 16, device="cuda").half(), torch.zeros(0, 16, device="cuda").half()).shape == (3, 0)


@gpu
def test_refusals_on_the_gpu():
    x, w, _ = make(4, 16, 32, torch.float16, 0)
    with pytest.raises(ValueError, match="GPU"):
        streamk.gated(x.float(), w.float())
    with pytest.raises(ValueError, match="one type"):
        streamk.linear(x.bfloat16(), w)
    with pytest.raises(ValueError, match="two dimensions"):
        streamk.linear(x, w[:, :16])
    with pytest.raises(ValueError, match="multiples of 8"):
        streamk.linear(x[:, :12], w[:, :12])
    with pytest.raises(ValueError, match="multiples of 8"):
        streamk.linear(x, w[:4])
    with pytest.raises(ValueError, match="as many of up"):
        streamk.gated(x, w[:31])
    with pytest.raises(ValueError, match="not 0"):
        streamk.linear(x[:, :0], w[:, :0])
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        g, = torch.autograd.grad(streamk.gated(x, w).float().sum(), x, create_graph=True)
        g.float().sum().backward()
    with pytest.raises(RuntimeError, match="differentiable once"):
        g, = torch.autograd.grad(streamk.linear(x, w).float().square().sum(), x, create_graph=True)
        g.float().sum().backward()


@gpu
def test_infinities_and_nan_stay_in_their_rows():
    for m in (20, 300):
        x, w, _ = make(m, 72, 200, torch.bfloat16, 8)
        want = streamk.gated(x, w)
        bad = x.clone()
        bad[3] = float("nan")
        bad[9, 7] = float("inf")
        got = streamk.gated(bad, w)
        keep = [i for i in range(m) if i not in (3, 9)]
        assert torch.equal(got[keep], want[keep]) and got[3].isnan().all()
    # far out the activations are g and 0 and their slopes 1 and 0, without NaN
    x = torch.full((70, 8), 100.0, dtype=torch.bfloat16, device="cuda")
    w = torch.eye(8, device="cuda").repeat(2, 1).bfloat16()
    w[1, 1] = -1
    x.requires_grad_()
    w.requires_grad_()
    for act in ("silu", "gelu"):
        h = streamk.gated(x, w, act)
        assert (h[:, 0] == 9984).all() and (h[:, 1] == 0).all()
        dx, dw = torch.autograd.grad(h.float().sum(), (x, w))
        assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


@gpu
def test_streams_and_two_at_once():
    problems = [make(m, 264, 520, torch.bfloat16, m) for m in (30, 90, 700)]
    want = [streamk.gated(x, w) for x, w, _ in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    out = []
    for _ in range(4):
        for (x, w, dh), stream in zip(problems, streams):
            with torch.cuda.stream(stream):
                a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
                h = streamk.gated(a, b)
                out.append((h.detach(), torch.autograd.grad(h, (a, b), dh)))
    torch.cuda.synchronize()
    for i, (h, grads) in enumerate(out):
        assert torch.equal(h, want[i % 3])
        assert all(torch.equal(a, b) for a, b in zip(grads, out[i % 3][1]))


@gpu
@pytest.mark.parametrize("m", [1, 64, 200])
def test_captured_and_replayed(m):
    n, k = 136, 264
    x, w, dh = make(m, n, k, torch.float16, 6)
    x.requires_grad_()
    w.requires_grad_()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(streamk.gated(x, w), (x, w), dh)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        h = streamk.gated(x, w)
        y = streamk.linear(x, w)
        dx, dw = torch.autograd.grad(h, (x, w), dh)
    for seed in range(3):
        nx, nw, ndh = make(m, n, k, torch.float16, 20 + seed)
        with torch.no_grad():
            x.copy_(nx), w.copy_(nw), dh.copy_(ndh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a, b = nx.requires_grad_(), nw.requires_grad_()
        ref = streamk.gated(a, b)
        assert torch.equal(h, ref) and torch.equal(y, streamk.linear(nx, nw))
        assert all(torch.equal(p, q) for p, q in zip((dx, dw), torch.autograd.grad(ref, (a, b), ndh)))


@gpu
def test_a_captured_backward_pass_beside_an_eager_graph_of_its_leaves():
    # made on the capture's own stream the eager graph is no hindrance, on another it is refused
    # before the engine draws that stream into the capture
    x, w, dh = make(70, 72, 136, torch.float16, 6)
    x.requires_grad_()
    w.requires_grad_()
    side = torch.cuda.Stream()
    for forward in (lambda: streamk.gated(x, w), lambda: streamk.linear(x, w[:72])):
        with torch.cuda.stream(side):
            want = torch.autograd.grad(forward(), (x, w), dh)
            alive = forward()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(forward(), (x, w), dh)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        del alive, got, graph
    alive = streamk.gated(x, w)
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            torch.autograd.grad(streamk.gated(x, w), (x, w), dh)
    torch.cuda.synchronize()
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(alive, (x, w), dh))


@gpu
def test_under_a_compiler():
    x, w, dh = make(70, 72, 136, torch.bfloat16, 1)
    leaves = [t.requires_grad_() for t in (x, w)]

    def loss(a, b):
        return (streamk.gated(a, b, "gelu") * 2, streamk.linear(a, b))

    compiled = torch.compile(loss, backend="aot_eager", fullgraph=True)
    for got, want in zip(compiled(*leaves), loss(*leaves)):
        assert torch.equal(got, want)
    got = torch.autograd.grad(compiled(*leaves)[0], leaves, dh)
    want = torch.autograd.grad(loss(*leaves)[0], leaves, dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        for got, want in zip(compiled(*leaves), loss(*leaves)):
            assert torch.equal(got, want)
    plain = [t.detach() for t in leaves]
    for got, want in zip(compiled(*plain), loss(*plain)):
        assert torch.equal(got, want) and not got.requires_grad
    # the sums are kept for gradients alone
    names = []

    def record(graph, example):
        names.append([str(node.target) for node in graph.graph.nodes])
        return graph.forward

    torch.compile(loss, backend=record, fullgraph=True)(*plain)
    torch.compile(lambda a, b: streamk.gated(a, b), backend=record, fullgraph=True)(*leaves)
    assert any("gated_alone" in n for n in names[0]) and not any("gated_dense" in n for n in names[0])
    assert any("gated_dense" in n for n in names[1])


@gpu
def test_forward_mode_is_refused_beside_tensors_without_tangents():
    import torch.autograd.forward_ad as forward_ad
    x, w, _ = make(20, 16, 32, torch.float16, 0)
    want = streamk.linear(x, w)
    with forward_ad.dual_level():
        assert torch.equal(streamk.linear(x, w), want)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for a in (dual, dual[:5], dual * 2):
            for call in (streamk.gated, streamk.linear):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(a, w)
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            streamk.linear(dual, w)


@gpu
def test_second_derivatives_beside_another_path_to_the_same_input():
    """Asked for by inputs, where no node that is on no way to them would be run."""
    for call in (streamk.gated, streamk.linear):
        x, w, dh = make(20, 16, 32, torch.float16, 0)
        dh = call(x, w).clone()
        leaves = [t.requires_grad_() for t in (x, w, dh)]
        for i in (0, 1):
            g, = torch.autograd.grad(call(x, w), leaves[i], dh, create_graph=True)
            for leaf in leaves:
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(g.float().sum() + leaf.float().sum(), leaf, retain_graph=True)
            # what has nothing to do with them is none of theirs
            z = torch.ones(3, device="cuda", requires_grad=True)
            assert torch.autograd.grad(g.float().sum() + (2 * z).sum(), z)[0].eq(2).all()


# A forced tile is the calling thread's, and the autograd engine's threads are others: what follows
# makes the backward passes' calls on this thread, and asks it for the plan that they take.

def forced_plan(tile, slices, m, n, k, turned):
    """The plan is the forced one: its tile, unless that layout has no such height, and its slices,
    unless there are not as many stages of 64."""
    rows, cols, got = streamk.product_plan(m, n, k, False, turned)
    if tile[0] != 96 or turned != 2:
        assert (rows, cols) == tile
        assert got == slices or -(-k // 64) < slices
    return True


@gpu
@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,n,k", [(1, 8, 64), (300, 520, 192), (257, 136, 1096), (130, 264, 128), (333, 304, 640)])
def test_gradients_by_every_tile(tile, m, n, k, slices):
    binding = streamk._torch_binding
    for type in TYPES:
        x, w, dh = make(m, n, k, type, 5)
        ref = Gated64(x, w, "gelu")
        try:
            streamk.force_product_tile(*tile, slices)
            assert forced_plan(tile, slices, m, k, 2 * n, 1) and forced_plan(tile, slices, 2 * n, k, m, 2)
            assert forced_plan(tile, slices, m, k, n, 1) and forced_plan(tile, slices, n, k, m, 2)
            h, sums = binding.gated_sums(x, w, 2)
            dx, dw = binding.gated_grads(dh, sums, x, w, 2, True, True)
            lx, lw = binding.linear_grads(dh, x, w[:n], True, True)
        finally:
            streamk.force_product_tile(0)
        ref.check_forward(h, type)
        ref.check_grads(dh, dx, dw, type)
        check_product(lx, dh, w[:n].t(), type)
        check_product(lw, dh.t(), x.t(), type)


@gpu
@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("tile,turned", [(t, turned) for t in TILES for turned in (0, 1, 2) if t[0] != 96 or turned != 2])
def test_every_tile_beside_rows_that_hold_nan(tile, turned, type, slices):
    """Matrices inside larger ones, as above, by every tile, in both types, whole and in slices."""
    import ctypes
    lib, L, P = streamk._lib, ctypes.c_longlong, ctypes.c_void_p
    for m, n, k in ((72, 200, 136), (328, 264, 320), (264, 520, 456)):
        gen = torch.Generator(device="cuda").manual_seed(m)
        a, b = (torch.randn(r, k, device="cuda", generator=gen).to(type) for r in (m, n))

        def inside(x):
            rows, cols = x.shape
            room = torch.full((rows + 80, cols + 96), float("nan"), dtype=type, device="cuda")
            room[8:8 + rows, 16:16 + cols] = x
            return room, room[8:8 + rows, 16:16 + cols]

        ra, va = inside(a.t().contiguous() if turned == 2 else a)
        rb, vb = inside(b.t().contiguous() if turned else b)
        rc, vc = inside(torch.zeros(m, n, device="cuda").to(type))
        before = rc.clone()
        room = torch.empty(3 * m * n, device="cuda")
        try:
            streamk.force_product_tile(*tile, slices)
            assert forced_plan(tile, slices, m, n, k, turned)
            code = lib.feedforward_product(P(va.data_ptr()), P(vb.data_ptr()), P(vc.data_ptr()), m, n, k, L(va.stride(0)),
                                           L(vb.stride(0)), L(vc.stride(0)), turned, int(type == torch.bfloat16),
                                           P(room.data_ptr()), L(4 * room.numel()), 0,
                                           P(torch.cuda.current_stream().cuda_stream))
        finally:
            streamk.force_product_tile(0)
        assert code == 0
        check_product(vc, a, b, type)
        vc.copy_(before[8:8 + m, 16:16 + n])
        assert torch.equal(rc.isnan(), before.isnan()) and not rc.nan_to_num().any()  # nothing else was written


@gpu
def test_gradients_that_are_views_to_be_read_negated():
    x, w, dh = make(20, 16, 32, torch.float16, 0)
    leaves = [t.requires_grad_() for t in (x, w)]
    for call in (streamk.gated, streamk.linear):
        h = call(x, w)
        dh = torch.randn_like(h)
        want = torch.autograd.grad(h, leaves, dh, retain_graph=True)
        got = torch.autograd.grad(h, leaves, torch._neg_view(-dh))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
