"""Two slices of a big tile that finish it together, through the C entries: inside matrices with NaN all round, and to the bit
what a launch that adds both slices' sums makes of them -- sums, slopes and results alike, with every epilogue."""
import ctypes
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import streamk  # noqa: E402
import test_linear_epilogue as epilogue  # noqa: E402

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
BIG = [(160, 256), (192, 256), (224, 256), (256, 256)]
P, L = ctypes.c_void_p, ctypes.c_longlong


@pytest.fixture
def polls():
    lib = streamk._lib
    lib.feedforward_force_polls.argtypes = [ctypes.c_int]
    lib.feedforward_force_polls.restype = None
    yield lib.feedforward_force_polls
    lib.feedforward_force_polls(-1)
    streamk.force_product_tile(0)


def room_of(m, n, k, gated, turned=0):
    """What slices that meet take, more than the sums of both alone."""
    lib = streamk._lib
    lib.feedforward_product_bytes.restype = L
    columns = -(-n // 16) * 32 if gated == 1 else n
    bytes = lib.feedforward_product_bytes(m, n, k, gated, turned, 0)
    assert bytes > 8 * m * columns
    return bytes, 8 * m * columns


def at(t):
    return P(None if t is None else t.data_ptr())


def apart(t):
    return L(0 if t is None else t.stride(0))


def linear(x, w, y, bias, residual, slopes, act, drop, room, train=True):
    lib, (m, k), n = streamk._lib, x.shape, len(w)
    scratch = torch.full((room,), 255, dtype=torch.uint8, device="cuda")
    entry = lib.feedforward_linear_train if train else lib.feedforward_linear
    assert entry(at(x), at(w), at(y), at(bias), at(residual), at(slopes), m, n, k, apart(x), apart(w), apart(y),
                 apart(residual), apart(slopes), int(x.dtype == torch.bfloat16), act,
                 None if drop is None else ctypes.byref(drop), at(scratch), L(room), 0,
                 P(torch.cuda.current_stream().cuda_stream)) == 0


def gated(x, w, h, pre, act, room):
    lib, (m, k), n = streamk._lib, x.shape, len(w) // 2
    scratch = torch.full((room,), 255, dtype=torch.uint8, device="cuda")
    assert lib.feedforward_gated(at(x), at(w), at(h), at(pre), m, n, k, apart(x), apart(w), apart(h), apart(pre),
                                 int(x.dtype == torch.bfloat16), act, at(scratch), L(room), 0,
                                 P(torch.cuda.current_stream().cuda_stream)) == 0


def inside(t, fill=float("nan")):
    """A larger matrix, and t inside it."""
    rows, cols = t.shape
    room = torch.full((rows + 80, cols + 96), fill, dtype=t.dtype, device="cuda")
    view = room[8:8 + rows, 16:16 + cols]
    view.copy_(t)
    return room, view


def untouched(room, view, fill=float("nan")):
    """Everything but the view is as it was."""
    view.fill_(fill)
    return (room.isnan() if fill != fill else room == fill).all()


@gpu
@pytest.mark.parametrize("tile", BIG)
@pytest.mark.parametrize("m,n,k", [(40, 200, 136), (328, 264, 320), (264, 520, 456)])
def test_inside_rows_that_hold_nan(m, n, k, tile, polls):
    for type in TYPES:
        x, w, bias, residual, _ = epilogue.make(m, n, k, type, m)
        (_, vx), (_, vw), (_, vr) = inside(x), inside(w), inside(residual)
        vb = inside(bias[None])[1]
        streamk.force_product_tile(*tile, 2)
        for act, name in ((0, None), (2, "gelu")):
            ref = epilogue.Full64(x, w, bias, name, residual, 0.3, 77, 2)
            drop = epilogue.DropArgs(0.3, 77, None, 2)
            for count in (-1, 0, 1):
                polls(count)
                for room in room_of(m, n, k, 2):
                    (ry, vy), (rs, vs) = inside(torch.zeros_like(residual)), inside(torch.zeros((m, n), dtype=torch.int16, device="cuda"), -7)
                    slopes = vs if act else None
                    linear(vx, vw, vy, vb, vr, slopes, act, drop, room, train=False)
                    ref.check_forward(vy)
                    if act:
                        epilogue.Full64(x, w, bias, name, None).check_slopes(vs)
                    y = vy.clone()
                    linear(vx, vw, vy, vb, vr, slopes, act, drop, room)
                    assert torch.equal(vy, y)
                    assert untouched(ry, vy) and untouched(rs, vs, -7)
        # gated
        n2 = n // 2 // 8 * 8
        vw = inside(w[:2 * n2])[1]
        for count in (-1, 0):
            polls(count)
            for room in room_of(m, n2, k, 1):
                (rh, vh), (rp, vp) = inside(torch.zeros((m, n2), dtype=type, device="cuda")), inside(
                    torch.zeros((m, -(-n2 // 16) * 32), device="cuda"), 5.0)
                gated(vx, vw, vh, vp, 1, room)
                # columns of the sums by turns of sixteen; the last turn's columns that are none stay as they are
                sums = x.double() @ w[:2 * n2].double().t()
                off = (k + 1) * epilogue.FP32 * (x.double().abs() @ w[:2 * n2].double().abs().t())
                for c in range(0, n2, 16):
                    wide = min(16, n2 - c)
                    for half, col in ((0, 2 * c), (n2, 2 * c + 16)):
                        got, want = vp[:, col:col + wide].double(), sums[:, half + c:half + c + wide]
                        assert ((got - want).abs() <= off[:, half + c:half + c + wide]).all()
                        assert (vp[:, col + wide:col + 16] == 0).all()
                g, u = sums[:, :n2], sums[:, n2:]
                value, slope = epilogue.act64(g, "silu")
                bound = (1.13 * off[:, :n2] + epilogue.ACT * value.abs()) * (u.abs() + off[:, n2:]) + off[:, n2:] * value.abs()
                want = value * u
                bound = (bound + epilogue.half_step(type) * want.abs()) * (1 + 2.0 ** -6) + epilogue.least(type)
                assert ((vh.double() - want).abs() <= bound).all()
                assert untouched(rh, vh) and untouched(rp, vp, 5.0)


@gpu
@pytest.mark.parametrize("tile", BIG)
@pytest.mark.parametrize("m,n,k", [(333, 528, 640), (100, 144, 1096), (8, 16, 136)])
def test_to_the_bit_what_a_launch_that_adds_makes(m, n, k, tile, polls):
    for type in TYPES:
        x, w, bias, residual, _ = epilogue.make(m, n, k, type, 5)
        streamk.force_product_tile(*tile, 2)
        full, alone = room_of(m, n, k, 2)
        for i, (has_bias, name, has_residual, p) in enumerate(epilogue.FORMS):
            act = {None: 0, "silu": 1, "gelu": 2}[name]
            for train in (True, False):
                out = []
                for count, room in ((-1, alone), (-1, full), (0, full), (1, full)):
                    polls(count)
                    y = torch.full((m, n), float("nan"), dtype=type, device="cuda")
                    slopes = torch.full((m, n), -7, dtype=torch.int16, device="cuda") if act else None
                    linear(x, w, y, bias if has_bias else None, residual if has_residual else None, slopes, act,
                           epilogue.DropArgs(p, 9, None, i), room, train)
                    out.append((y, y if slopes is None else slopes))
                for y, slopes in out[1:]:
                    assert torch.equal(y, out[0][0]) and torch.equal(slopes, out[0][1])
        full, alone = room_of(m, n // 2, k, 1)
        for act in (1, 2):
            out = []
            for count, room in ((-1, alone), (-1, full), (0, full), (1, full)):
                polls(count)
                h = torch.full((m, n // 2), float("nan"), dtype=type, device="cuda")
                pre = torch.full((m, -(-n // 32) * 32), -1.0, device="cuda")
                gated(x, w, h, pre, act, room)
                out.append((h, pre))
            for h, pre in out[1:]:
                assert torch.equal(h, out[0][0]) and torch.equal(pre, out[0][1])
