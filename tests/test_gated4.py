"""Gated projections with 4-bit weights: marlin.GatedLayer, marlin.gated_mul, feedforward_gated_w4.

The oracle is the definition in 64 bits with the weights (q - 8) s.  What the kernels may be off by,
element by element: a weight is rounded to fp16 once (2^-11 of it; not at all, or the sums instead,
where a kernel scales these), a sum of k products in fp32 loses at most k 2^-24 of the sum of their
magnitudes, the activations' slopes are below 1.13, and the result is rounded once (2^-11, and half
of fp16's smallest step).
"""
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
import marlin  # noqa: E402

gpu = pytest.mark.gpu


def act64(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    return g / 2 * (1 + torch.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))


def problem(m, n, k, group, seed=0, dev="cpu"):
    gen = torch.Generator().manual_seed(seed)
    groups = 1 if group == -1 else k // group
    x = torch.randn((m, k), generator=gen).half()
    q = torch.randint(0, 16, (2, n, k), generator=gen)
    s = (torch.rand((2, n, groups), generator=gen) * 0.019 + 0.001).half()
    fake = ((q - 8).half().reshape(2, n, groups, -1) * s.unsqueeze(-1)).reshape(2, n, k)
    return x.to(dev), q.to(dev), s.to(dev), fake.to(dev)


def layer_of(q, s, fake, group, act):
    _, n, k = q.shape
    layer = marlin.GatedLayer(k, n, group, act).to(q.device)
    layer.pack(marlin._Weight(fake[0]), marlin._Weight(fake[1]), s[0], s[1])
    return layer


def check(y, x, q, s, act):
    k = x.shape[-1]
    w = (q - 8).double().reshape(q.shape[0], q.shape[1], s.shape[2], -1) * s.double().unsqueeze(-1)
    w = w.reshape(q.shape)
    xd = x.double()
    g, u = xd @ w[0].t(), xd @ w[1].t()
    size = [xd.abs() @ w[i].abs().t() for i in range(2)]
    want = act64(g, act) * u
    off = 2.0 ** -11 + k * 2.0 ** -24
    dg, du = off * size[0], off * size[1]
    bound = 1.13 * dg * (u.abs() + du) + act64(g, act).abs() * du + 2.0 ** -11 * want.abs() + 2.0 ** -25
    bound = bound * (1 + 2.0 ** -10)  # (the rounding of what is off already)
    err = (y.double() - want).abs()
    assert torch.isfinite(y).all()
    assert (err <= bound).all(), float((err / bound).max())
    # the roundings are independent of each other: all of them together stay near one
    assert err.norm() <= 3 * 2.0 ** -11 * want.norm()


# --- without a GPU -------------------------------------------------------------------------

def test_pack_puts_gate_and_up_in_turns_of_eight():
    n, k = 128, 256
    _, q, s, fake = problem(1, n, k, 128)
    layer = layer_of(q, s, fake, 128, "silu")
    both = torch.stack([q[0].reshape(n // 8, 8, k), q[1].reshape(n // 8, 8, k)], 1).reshape(2 * n, k)
    scales = torch.stack([s[0].reshape(n // 8, 8, -1), s[1].reshape(n // 8, 8, -1)], 1).reshape(2 * n, -1)
    assert torch.equal(layer.B, marlin.pack_weights(both.t().contiguous().int()))
    assert torch.equal(layer.s, marlin.pack_scales(scales.t().contiguous(), True))


def test_refuses_what_it_cannot_compute():
    with pytest.raises(ValueError, match="128"):
        marlin.GatedLayer(256, 192)
    with pytest.raises(ValueError, match="activation"):
        marlin.GatedLayer(256, 128, activation="relu")
    with pytest.raises(ValueError, match="groupsize"):
        marlin.GatedLayer(256, 128, groupsize=64)
    layer = marlin.GatedLayer(256, 128)
    half = torch.nn.Linear(256, 128, bias=False).half()
    with pytest.raises(ValueError, match="weights must be"):
        layer.pack(half, torch.nn.Linear(128, 128, bias=False).half(), torch.ones(128, 1).half(), torch.ones(128, 1).half())
    with pytest.raises(ValueError, match="half"):
        layer.pack(half, torch.nn.Linear(256, 128, bias=False), torch.ones(128, 1).half(), torch.ones(128, 1).half())
    with pytest.raises(RuntimeError, match="GPU tensor"):
        layer(torch.zeros(1, 256).half())
    with pytest.raises(ValueError, match="activation"):
        marlin.gated_mul(None, None, None, None, None, activation="tanh")


@pytest.mark.parametrize("m,n,k,rows,numel,act,par,code", [
    (1, 128, 256, 2, 10 ** 6, 3, 16, 2),      # an unknown activation
    (1, 128, 256, 2, 10 ** 6, 0, 16, 2),
    (1, 64, 256, 2, 10 ** 6, 1, 16, 1),       # columns
    (1, 128, 192, 1, 10 ** 6, 1, 16, 1),      # depth
    (-1, 128, 256, 2, 10 ** 6, 1, 16, 1),
    (1, 128, 256, 0, 10 ** 6, 1, 16, 4),      # groups
    (1, 128, 256, 3, 10 ** 6, 1, 16, 4),
    (1, 128, 512, 8, 10 ** 6, 1, 16, 2),      # groups of 64
    (1, 128, 256, 2, 31, 1, 16, 5),           # workspace
    (1, 128, 256, 2, 10 ** 6, 1, 0, 5),
    (1, 128, 0, 1, 10 ** 6, 1, 16, 1),
    (0, 128, 256, 2, 32, 1, 16, 0),           # nothing to do
])
def test_codes_of_the_entry(m, n, k, rows, numel, act, par, code):
    import ctypes
    err = ctypes.create_string_buffer(256)
    lib = marlin._lib
    rc = lib.feedforward_gated_w4(None, None, None, None, m, n, k, rows, None, ctypes.c_longlong(numel), act, 0, None, par,
                          err, 256)
    assert rc == code
    assert (len(err.value) > 0) == (code != 0)


# --- on the GPU ----------------------------------------------------------------------------

# one row to many: column strips, rows, streaming and prefill kernels, whole tiles and slices
SIZES = [(1, 128, 256, 128), (2, 384, 128, -1), (1, 10752, 4096, 128), (5, 4096, 1024, -1), (8, 640, 11008, 128),
         (9, 1024, 512, 128), (16, 10752, 4096, 128), (17, 768, 640, -1), (33, 2048, 4096, 128),
         (45, 13568, 5120, -1), (64, 14336, 8192, 128), (65, 640, 1024, 128), (100, 384, 8192, 128),
         (203, 2560, 5120, 128), (300, 384, 8192, -1), (513, 1024, 1024, -1), (777, 5504, 4096, 128)]


@gpu
@pytest.mark.parametrize("m,n,k,group", SIZES)
def test_matches_the_definition(m, n, k, group):
    x, q, s, fake = problem(m, n, k, group, seed=m + n, dev="cuda")
    for act in ("silu", "gelu"):
        layer = layer_of(q, s, fake, group, act)
        check(layer(x), x, q, s, act)
        assert not layer.workspace.any()


@gpu
@pytest.mark.parametrize("force", [("kernel", 1), ("kernel", 2), ("kernel", 3), ("k_slices", 3), ("rows", (2, 3)),
                                   ("rows", (8, 2)), ("rows", (8, 3)), ("rows", (8, 4)), ("rows", (1, 1)),
                                   ("tile", 80), ("tile", 96), ("tile", 112), ("tile", 128)])
@pytest.mark.parametrize("group", [128, -1])
def test_every_kernel(force, group):
    m, n, k = 50, 512, 5120  #
    x, q, s, fake = problem(m, n, k, group, seed=3, dev="cuda")
    layer = layer_of(q, s, fake, group, "silu")
    kind, value = force
    try:
        if kind == "kernel":
            marlin.force_kernel(value)
        elif kind == "k_slices":
            marlin.force_kernel(2)
            marlin.force_k_slices(value)
        elif kind == "rows":
            marlin.force_rows(*value)
        else:
            marlin.force_kernel(2)
            marlin.force_tile_rows(value)
            marlin.force_k_slices(2)
        check(layer(x), x, q, s, "silu")
    finally:
        marlin.force_kernel(0)
        marlin.force_k_slices(0)
        marlin.force_rows(0)
        marlin.force_tile_rows(0)


@gpu
def test_agrees_with_a_layer_of_both_projections():
    """The plan is that of a layer of 2n columns, and so are the sums."""
    m, n, k = 3, 256, 512
    x, q, s, fake = problem(m, n, k, 128, seed=5, dev="cuda")
    layer = layer_of(q, s, fake, 128, "silu")
    product = marlin.Layer(k, 2 * n, 128).to("cuda")
    product.B, product.s = layer.B, layer.s
    both = product(x).reshape(m, n // 8, 2, 8)
    g, u = both[:, :, 0].reshape(m, n).double(), both[:, :, 1].reshape(m, n).double()
    want = act64(g, "silu") * u
    # g and u are rounded to fp16 there, 2^-11 each, slopes of at most 1.13 and |act(g)| <= |g|
    bound = 2.0 ** -11 * (1.13 * g.abs() * u.abs() + 2 * want.abs()) * 1.01 + 2.0 ** -24 * (1 + g.abs() + u.abs())
    assert ((layer(x).double() - want).abs() <= bound).all()


@gpu
def test_shapes_strides_and_rows_behind_the_last():
    n, k = 256, 384
    x, q, s, fake = problem(12, n, k, -1, seed=6, dev="cuda")
    layer = layer_of(q, s, fake, -1, "gelu")
    want = layer(x)
    assert torch.equal(layer(x.reshape(3, 4, k)), want.reshape(3, 4, n))
    wide = torch.zeros((12, k + 40), dtype=torch.half, device="cuda")
    wide[:, 8:8 + k] = x
    assert torch.equal(layer(wide[:, 8:8 + k]), want)
    assert layer(x[:0]).shape == (0, n)
    assert layer(x[0]).shape == (n,)
    # rows of C behind those of A are left as they were
    C = torch.full((20, n), 7.0, dtype=torch.half, device="cuda")
    marlin.gated_mul(x, layer.B, C[:12], layer.s, layer.workspace, "gelu")
    assert torch.equal(C[:12], want) and (C[12:] == 7).all()


@gpu
def test_operands_off_sixteen_bytes():
    for m in (4, 12, 40):
        x, q, s, fake = problem(m, 256, 1024, 128, seed=m, dev="cuda")
        layer = layer_of(q, s, fake, 128, "silu")
        room = torch.empty(x.numel() + 1, dtype=torch.half, device="cuda")
        off = room[1:].view(x.shape)
        off.copy_(x)
        check(layer(off), x, q, s, "silu")


@gpu
def test_infinities_and_nan_stay_in_their_rows():
    n, k = 256, 512
    x, q, s, fake = problem(20, n, k, 128, seed=8, dev="cuda")
    layer = layer_of(q, s, fake, 128, "silu")
    want = layer(x)
    bad = x.clone()
    bad[3, 5] = float("nan")
    bad[9, 7] = float("inf")
    got = layer(bad)
    keep = [i for i in range(20) if i not in (3, 9)]
    assert torch.equal(got[keep], want[keep])
    assert got[3].isnan().all()
    # sums far beyond the exponential's range: act(-300) = -0, act(300) = 300
    huge = torch.zeros((1, k), dtype=torch.half, device="cuda")
    huge[0, 0] = 40000.0
    out = layer(huge)
    assert not out.isnan().any()


@gpu
def test_refusals_on_the_gpu():
    n, k = 128, 256
    x, q, s, fake = problem(2, n, k, -1, dev="cuda")
    layer = layer_of(q, s, fake, -1, "silu")
    with pytest.raises(ValueError, match="half"):
        layer(x.float())
    with pytest.raises(ValueError, match="gated product takes"):
        layer(x[:, :128].contiguous())
    C = torch.empty((2, n), dtype=torch.half, device="cuda")
    with pytest.raises(RuntimeError, match="workspace"):
        marlin.gated_mul(x, layer.B, C, layer.s, layer.workspace[:8])
    with pytest.raises(ValueError, match="gated product takes"):
        marlin.gated_mul(x, layer.B, torch.empty((3, n), dtype=torch.half, device="cuda"), layer.s, layer.workspace)
    with pytest.raises(RuntimeError, match="contiguous"):
        marlin.gated_mul(x, layer.B, torch.empty((n, 2), dtype=torch.half, device="cuda").t(), layer.s, layer.workspace)


@gpu
@pytest.mark.parametrize("m", [1, 16, 48, 300])
def test_captured_and_replayed(m):
    n, k = 1024, 1024
    x, q, s, fake = problem(m, n, k, 128, seed=m, dev="cuda")
    layer = layer_of(q, s, fake, 128, "silu")
    side = torch.cuda.Stream()
    static = x.clone()
    with torch.cuda.stream(side):
        layer(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = layer(static)
    for seed in range(3):
        y = problem(m, n, k, 128, seed=seed + 50, dev="cuda")[0]
        static.copy_(y)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        check(out, y, q, s, "silu")


@gpu
def test_under_a_compiler():
    n, k = 256, 256
    x, q, s, fake = problem(4, n, k, -1, seed=9, dev="cuda")
    layer = layer_of(q, s, fake, -1, "gelu")
    compiled = torch.compile(lambda t: layer(t) * 2, backend="eager", fullgraph=True)
    assert torch.equal(compiled(x), layer(x) * 2)


@gpu
def test_strided_rows_under_a_compiler():
    """What the call copies eagerly it copies there as well."""
    n, k = 256, 256
    x, q, s, fake = problem(6, n, k, -1, seed=9, dev="cuda")
    layer = layer_of(q, s, fake, -1, "silu")
    wide = torch.zeros((6, k + 40), dtype=torch.half, device="cuda")
    wide[:, 8:8 + k] = x
    want = layer(x)
    for backend in ("eager", "aot_eager"):
        compiled = torch.compile(lambda t: layer(t) * 1, backend=backend, fullgraph=True)
        for a in (wide[:, 8:8 + k], x.t().contiguous().t(), x.reshape(2, 3, k).transpose(0, 1)):
            assert torch.equal(compiled(a), layer(a))
        assert torch.equal(compiled(wide[:, 8:8 + k]), want)
    assert not layer.workspace.any()


def test_an_activation_is_what_the_layer_says():
    layer = marlin.GatedLayer(256, 128)
    layer.activation = "relu"
    with pytest.raises(ValueError, match="activation"):
        layer(torch.zeros(1, 256).half())


@gpu
def test_an_activation_that_is_changed():
    """Eagerly and under a compiler it is the layer's attribute that counts."""
    n, k = 128, 256
    x, q, s, fake = problem(3, n, k, 128, seed=4, dev="cuda")
    layer = layer_of(q, s, fake, 128, "silu")
    want = layer_of(q, s, fake, 128, "gelu")(x)
    layer.activation = "gelu"
    assert torch.equal(layer(x), want)
    assert torch.equal(torch.compile(lambda t: layer(t) * 1, backend="eager", fullgraph=True)(x), want)


def test_what_has_no_gradients_says_so():
    """The result of products that have none, wherever a gradient would pass through it."""
    x, out = torch.ones(3, requires_grad=True), torch.full((3,), 2.0)
    mark = marlin._torch_binding.without_gradients
    y = mark(out, x)
    assert torch.equal(y.detach(), out) and y.requires_grad
    for backward in (lambda: (x + y).sum().backward(), lambda: torch.autograd.grad((x + y).sum(), x),
                     lambda: torch.autograd.grad((x * 2 + mark(out, x * 3)).sum(), x)):
        with pytest.raises(RuntimeError, match="4-bit weights have no gradients"):
            backward()
    with torch.no_grad():
        assert not mark(out, x).requires_grad
    assert not mark(out, x.detach()).requires_grad


@gpu
def test_gradients_are_not_lost_without_a_word():
    n = k = 256
    x, q, s, fake = problem(3, n, k, 128, seed=4, dev="cuda")
    layer = layer_of(q, s, fake, 128, "silu")
    want = layer(x)
    x.requires_grad_()
    y = layer(x)
    assert torch.equal(y, want)
    with pytest.raises(RuntimeError, match="no gradients"):
        (x + y).sum().backward()
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.autograd.grad((x + layer(x)).sum(), x)
    C = torch.empty_like(want)
    with pytest.raises(RuntimeError, match="gated_mul"):
        marlin.gated_mul(x, layer.B, C, layer.s, layer.workspace)
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.compile(lambda t: t + layer(t), backend="aot_eager", fullgraph=True)(x)
    with torch.no_grad():
        assert not layer(x).requires_grad
        marlin.gated_mul(x, layer.B, C, layer.s, layer.workspace)
        assert torch.equal(torch.compile(lambda t: layer(t) * 1, backend="aot_eager", fullgraph=True)(x), want)
    assert torch.equal(C, want)


def test_refuses_forward_mode():
    import torch.autograd.forward_ad as forward_ad
    layer = marlin.GatedLayer(256, 128)
    x, C = torch.zeros(1, 256).half(), torch.zeros(1, 128).half()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            layer(dual)
        with pytest.raises(RuntimeError, match="forward-mode"):
            marlin.gated_mul(dual, layer.B, C, layer.s, layer.workspace)


@pytest.mark.parametrize("m,n,k,code", [(80000, 14336, 128, 3), (8192, 128, 1 << 17, 3), (1, 1 << 17, 1 << 14, 3)])
def test_operands_of_more_than_two_gib_are_refused(m, n, k, code):
    import ctypes
    err = ctypes.create_string_buffer(256)
    rc = marlin._lib.feedforward_gated_w4(None, None, None, None, m, n, k, 1, None, ctypes.c_longlong(1 << 30), 1, 0,
                                          None, 16, err, 256)
    assert rc == code and b"2 GiB" in err.value and f"m={m} n={n} k={k}".encode() in err.value


@gpu
def test_as_many_rows_as_make_two_gib_of_results():
    """The product has twice C's columns, and would be more; the first rows, the last and some between."""
    n, k, m = 14336, 128, 74880
    assert 1.99 * 2 ** 30 < 2 * m * n < 2 ** 31
    x, q, s, fake = problem(m, n, k, -1, seed=1, dev="cuda")
    layer = layer_of(q, s, fake, -1, "silu")
    y = layer(x)
    for first in (0, 37440, m - 200):
        check(y[first:first + 200], x[first:first + 200], q, s, "silu")


@gpu
def test_views_to_be_read_negated():
    x, q, s, fake = problem(2, 128, 256, -1, dev="cuda")
    layer = layer_of(q, s, fake, -1, "silu")
    C = torch.empty((2, 128), dtype=torch.half, device="cuda")
    for call in (layer, lambda a: marlin.gated_mul(a, layer.B, C, layer.s, layer.workspace)):
        with pytest.raises(ValueError, match="plain tensor"):
            call(torch._neg_view(x))
