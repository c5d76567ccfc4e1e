"""The norms around a block (feedforward.residual_norm), its gate and the residual's scale.

The oracle is the definition in 64 bits.  Bounds, element by element, with e half a step of the type
(2^-11, 2^-8, 2^-24) and F = 48 x 2^-24 for what fp32 loses inside: a sum of up to 16384 squares is
sixteen terms to a lane and ten additions in pairs, a length one root and one division, a term a few
products.  The backward pass reads r as the forward pass rounded it.
"""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
import feedforward  # noqa: E402
from feedforward import residual_norm  # noqa: E402

gpu = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
F = 48 * 2.0 ** -24
EPS = 1e-6


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[t]


def within(got, want, bound, type, name):
    bound = bound * (1 + 2.0 ** -6) + least(type)
    err = (got.double() - want).abs()
    assert got.dtype == type and got.shape == want.shape and torch.isfinite(got).all(), name
    assert (err <= bound).all(), (name, float((err / bound).max()))


def make(shape, type, gate, seed, post=True, pre=True, block=True, dev="cuda"):
    gen = torch.Generator(device=dev).manual_seed(seed)
    d = shape[-1]

    def randn(*s, std=1.0, mean=0.0):
        return (torch.randn(s, device=dev, generator=gen) * std + mean).to(type)

    t = {"residual": randn(*shape), "block": randn(*shape) if block else None,
         "post_weight": randn(d, std=0.1, mean=1.0) if post else None,
         "pre_weight": randn(d, std=0.1, mean=1.0) if pre else None, "gate": None}
    if gate == "channel":
        t["gate"] = randn(d, std=0.2, mean=0.5)
    elif gate == "sequence":
        t["gate"] = randn(*shape[:1], *[1] * (len(shape) - 2), d, std=0.2, mean=0.5)
    elif gate == "row":
        t["gate"] = randn(*shape, std=0.2, mean=0.5)
    return t, randn(*shape, std=0.1), randn(*shape, std=0.1)


class Norm64:
    def __init__(self, t, scale):
        f = {k: None if v is None else v.detach().double() for k, v in t.items()}
        self.t, self.type, self.scale = f, t["residual"].dtype, scale
        one = torch.ones((), dtype=torch.float64, device=t["residual"].device)
        self.post = one if f["post_weight"] is None else f["post_weight"]
        self.pre = one if f["pre_weight"] is None else f["pre_weight"]
        self.gate = one if f["gate"] is None else f["gate"]
        if f["block"] is None:
            self.r, self.off = f["residual"], torch.zeros_like(f["residual"])
        else:
            b = f["block"]
            self.rstd1 = one if f["post_weight"] is None else (b.square().mean(-1, keepdim=True) + EPS).rsqrt()
            self.bh = b * self.rstd1
            p = self.gate * self.bh * self.post
            self.r = scale * f["residual"] + p
            self.off = F * (abs(scale) * f["residual"].abs() + p.abs())
        self.rstd2 = (self.r.square().mean(-1, keepdim=True) + EPS).rsqrt()
        self.rh = self.r * self.rstd2
        # what the length of r is off by, relative to it
        self.delta = F + self.off.norm(dim=-1, keepdim=True) / self.r.norm(dim=-1, keepdim=True).clamp_min(1e-30)

    def check_forward(self, y, r):
        e = half_step(self.type)
        if self.t["block"] is not None:
            within(r, self.r, self.off + e * self.r.abs(), self.type, "r")
        if self.t["pre_weight"] is not None:
            want = self.rh * self.pre
            bound = (self.delta + F + e) * want.abs() + self.rstd2 * self.pre.abs() * self.off
            within(y, want, bound, self.type, "y")

    def check_grads(self, dy, dr, got):
        e, ty = half_step(self.type), self.type
        rows = self.r.numel() // self.r.shape[-1]
        zero = torch.zeros_like(self.r)
        dy = zero if dy is None or self.t["pre_weight"] is None else dy.double()
        dr = zero if dr is None else dr.double()
        rh, rstd2 = self.rh, self.rstd2
        a = e + F + self.delta
        off_rh = a * rh.abs() + rstd2 * (self.off + least(ty))
        dyp = dy * self.pre
        m1 = (dyp * rh).mean(-1, keepdim=True)
        off_m1 = (dyp.abs() * off_rh).mean(-1, keepdim=True) + F * (dyp * rh).abs().mean(-1, keepdim=True)
        dt = dr + rstd2 * (dyp - rh * m1)
        off_dt = rstd2 * (rh.abs() * off_m1 + m1.abs() * off_rh) + (F + self.delta) * (
            dr.abs() + rstd2 * (dyp.abs() + (rh * m1).abs()))
        sums = rows * 2.0 ** -24 + F
        scale = 1.0 if self.t["block"] is None else self.scale
        if got.get("residual") is not None:
            within(got["residual"], scale * dt, abs(scale) * off_dt + e * (scale * dt).abs(), ty, "dresidual")
        if got.get("pre_weight") is not None:
            lead = tuple(range(dy.dim() - 1))
            want = (dy * rh).sum(lead)
            bound = (dy.abs() * off_rh).sum(lead) + sums * (dy * rh).abs().sum(lead) + e * want.abs()
            within(got["pre_weight"], want, bound, ty, "dpre")
        if self.t["block"] is None:
            return
        lead = tuple(range(dy.dim() - 1))
        gp = self.gate * self.post
        gpb = (gp * self.bh).abs()
        off_bh = F * self.bh.abs()
        if got.get("block") is not None:
            w = dt * gp
            if self.t["post_weight"] is None:
                want, off_m2, m2 = w, torch.zeros_like(m1), torch.zeros_like(m1)
            else:
                m2 = (w * self.bh).mean(-1, keepdim=True)
                want = self.rstd1 * (w - self.bh * m2)
                off_m2 = (gpb * off_dt).mean(-1, keepdim=True) + 4 * (F + self.delta) * (
                    gpb * (dr.abs() + rstd2 * (dyp.abs() + (rh * m1).abs()))).mean(-1, keepdim=True)
            bound = self.rstd1 * (gp.abs() * off_dt + self.bh.abs() * off_m2 + F * (w.abs() + (self.bh * m2).abs()))
            within(got["block"], want, bound + e * want.abs(), ty, "dblock")
        q, off_q = dt * self.bh, self.bh.abs() * off_dt + dt.abs() * off_bh
        if got.get("post_weight") is not None:
            want = (self.gate * q).sum(lead)
            bound = (self.gate.abs() * (off_q + sums * q.abs())).sum(lead) + (e + F) * want.abs()
            within(got["post_weight"], want, bound, ty, "dpost")
        if got.get("gate") is not None:
            shape = self.t["gate"].shape

            def over(x):
                return x.sum(lead) if len(shape) == 1 else x.sum_to_size(shape)

            want = over(q * self.post)
            bound = over(self.post.abs() * (off_q + sums * q.abs())) + (e + F) * want.abs()
            within(got["gate"], want, bound, ty, "dgate")


NAMES = ("residual", "block", "post_weight", "gate", "pre_weight")


def run(t, scale=0.75):
    return residual_norm(**t, scale=scale, eps=EPS)


def grads_of(t, outs, grads, names=NAMES):
    names = [n for n in names if t[n] is not None]
    return dict(zip(names, torch.autograd.grad(outs, [t[n] for n in names], grads)))


def leaves(t):
    return {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}


# --- without a GPU -------------------------------------------------------------------------

def test_refuses_host_tensors():
    with pytest.raises(ValueError, match="on the GPU"):
        residual_norm(torch.zeros(2, 16), pre_weight=torch.ones(16))
    with pytest.raises(TypeError, match="Tensor"):
        residual_norm(None, pre_weight=torch.ones(16))
    with pytest.raises(ValueError, match="multiples of 8"):
        feedforward.FeedForward(20, 16)
    with pytest.raises(ValueError, match="activation"):
        feedforward.FeedForward(16, 16, "relu")


def test_refuses_forward_mode():
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.zeros(2, 16), torch.ones(16)
    with forward_ad.dual_level():
        for args in (dict(residual=forward_ad.make_dual(x, x), pre_weight=w),
                     dict(residual=x, pre_weight=forward_ad.make_dual(w, w)),
                     dict(residual=x, block=forward_ad.make_dual(x, x)),
                     dict(residual=x, block=x, post_weight=forward_ad.make_dual(w, w)),
                     dict(residual=x, block=x, gate=forward_ad.make_dual(w, w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                residual_norm(**args)


def test_codes_and_scratch_of_the_entries():
    import ctypes
    import marlin
    lib = marlin._lib
    L, I, D, P = ctypes.c_longlong, ctypes.c_int, ctypes.c_float, ctypes.c_void_p
    lib.feedforward_norm_grad_bytes.restype = L
    nbytes = lib.feedforward_norm_grad_bytes

    def norm(rows, d, per, type=0, ldr=None, block=None, r=None, pre=P(16), y=P(16), eps=1e-6, gate=None, post=None):
        return lib.feedforward_norm(P(16), L(d if ldr is None else ldr), block, L(d), post, gate, L(d), I(per), pre,
                                    D(1.0), D(eps), r, y, None, L(rows), I(d), I(type), I(0), None)

    assert norm(0, 64, 1) == 0
    assert norm(4, 0, 1) == 1 and norm(4, 16385, 1) == 1 and norm(-1, 64, 1) == 1
    assert norm(4, 64, 0) == 1 and norm(4, 64, 3) == 1       # rows that no gate's rows divide
    assert norm(4, 64, 4, type=3) == 1
    assert norm(4, 64, 4, ldr=63) == 1
    assert norm(4, 64, 4, eps=-1.0) == 1 and norm(4, 64, 4, eps=float("nan")) == 1
    assert norm(4, 64, 4, pre=None) == 1                     # nothing to compute
    assert norm(4, 64, 4, y=None) == 1 and norm(4, 64, 4, block=P(16)) == 1  # an output is missing
    assert norm(4, 64, 4, gate=P(16)) == 1 and norm(4, 64, 4, post=P(16)) == 1  # of no block
    assert nbytes(L(4), I(64), I(3), I(0)) == -1
    for rows, per in ((1, 1), (5, 5), (4096, 1024), (4096, 1), (6000, 2), (8192, 8192), (131072, 16)):
        for d in (1, 64, 1000, 4096, 16384):
            for type in (0, 2):
                assert 8 * d <= nbytes(L(rows), I(d), I(per), I(type)) <= 8 * d * rows

    def grad(rows, d, partials, have, **missing):
        a = dict(dy=P(16), r=P(16), block=P(16), post=P(16), gate=P(16), pre=P(16), stats=P(16), dpost=P(16))
        a.update(missing)
        return lib.feedforward_norm_grad(a["dy"], L(d), None, L(d), a["r"], L(d), a["block"], L(d), a["post"], a["gate"],
                                         L(d), I(rows or 1), a["pre"], D(1.0), a["stats"], None, None, a["dpost"], None,
                                         None, partials, L(have), L(rows), I(d), I(0), I(0), None)

    assert grad(0, 64, None, 0) == 0
    need = nbytes(L(4), I(64), I(4), I(0))
    assert grad(4, 64, None, need) == 1 and grad(4, 64, P(16), need - 1) == 1
    for name in ("dy", "r", "stats", "block", "post"):
        assert grad(4, 64, P(16), need, **{name: None}) == 1, name


# --- on the GPU ----------------------------------------------------------------------------

SHAPES = [(1, 1, 4096), (2, 3, 8), (1, 7, 64), (3, 5, 520), (2, 33, 1032), (1, 2, 1), (2, 9, 77), (3, 4, 1001),
          (1, 40, 4096), (2, 5, 8192), (1, 3, 8200), (1, 3, 16384), (1, 2, 9001), (1, 2, 16383)]


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_definition(shape, type):
    for gate in ("none", "channel", "sequence"):
        t, dy, dr = make(shape, type, gate, seed=sum(shape))
        ref = Norm64(t, 0.75)
        ref.check_forward(*run(t))
        v = leaves(t)
        y, r = run(v)
        ref.check_forward(y.detach(), r.detach())
        ref.check_grads(dy, dr, grads_of(v, (y, r), (dy, dr)))


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("shape,gate", [((4096, 64), "none"), ((5000, 3, 72), "sequence"), ((6000, 136), "row"),
                                        ((3, 1500, 1024), "sequence"), ((700, 9, 33), "sequence"), ((513, 2048), "channel"),
                                        ((130, 8, 4096), "row"), ((2, 300, 8192), "sequence"), ((300, 16384), "row")])
def test_sums_over_many_rows(shape, gate, type):
    """Parts of a gate's rows, whole gates of several rows, and a gate to a row."""
    t, dy, dr = make(shape, type, gate, seed=len(shape))
    v = leaves(t)
    y, r = run(v)
    ref = Norm64(t, 0.75)
    ref.check_forward(y.detach(), r.detach())
    ref.check_grads(dy, dr, grads_of(v, (y, r), (dy, dr)))


@gpu
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel"])
def test_parts_that_are_left_out(block, post, pre, gate):
    t, dy, dr = make((3, 70, 264), torch.bfloat16, gate, 5, post, pre, block)
    if not block and (post or gate != "none" or not pre):
        with pytest.raises(ValueError, match="block"):
            run(t)
        return
    ref = Norm64(t, 0.75)
    y, r = run(t)
    assert (y is None) == (not pre) and (block or r is t["residual"])
    ref.check_forward(y, r)
    v = leaves(t)
    y, r = run(v)
    outs, grads = ([y], [dy]) if not block else ([r], [dr]) if not pre else ([y, r], [dy, dr])
    got = grads_of(v, outs, grads)
    ref.check_grads(dy, dr if block else None, got)
    if block and pre:  # a gradient of one output alone
        y, r = run(v)
        ref.check_grads(dy, None, grads_of(v, [y], [dy]))
        y, r = run(v)
        names = [n for n in NAMES if n != "pre_weight"]
        ref.check_grads(None, dr, grads_of(v, [r], [dr], names))
        loss = residual_norm(**v, scale=0.75)[1].float().sum()
        assert not torch.autograd.grad(loss, v["pre_weight"])[0].any()


@gpu
def test_only_the_gradients_that_are_wanted_and_the_same_bits_each_time():
    t, dy, dr = make((2, 300, 520), torch.bfloat16, "sequence", 5)
    v = leaves(t)
    want = grads_of(v, run(v), (dy, dr))
    for _ in range(3):
        for name in NAMES:
            one = {k: x.detach().requires_grad_(k == name) for k, x in t.items()}
            y, r = run(one)
            outs = [(o, g) for o, g in ((y, dy), (r, dr)) if o.requires_grad]
            got, = torch.autograd.grad([o for o, _ in outs], [one[name]], [g for _, g in outs])
            assert torch.equal(got, want[name]), name


@gpu
def test_gradients_against_differences():
    for gate in ("none", "sequence"):
        t, dy, dr = make((2, 6, 40), torch.float32, gate, 9)
        v = leaves(t)
        got = grads_of(v, run(v), (dy, dr))
        gen = torch.Generator(device="cuda").manual_seed(1)
        along = {k: torch.randn(x.shape, device="cuda", generator=gen, dtype=torch.float64) for k, x in got.items()}

        def loss(step):
            moved = {k: None if x is None else x.double() + step * along[k] for k, x in t.items()}
            ref = Norm64(moved, 0.75)
            return (ref.rh * ref.pre * dy.double()).sum() + (ref.r * dr.double()).sum()

        step = 1e-5
        slope = (loss(step) - loss(-step)) / (2 * step)
        terms = torch.cat([(got[k].double() * along[k]).flatten() for k in got])
        # fp32 terms, each off by some F; the differences by step^2 and 2^-52 / step of the loss's terms
        assert (terms.sum() - slope).abs() <= (F + 1e-8) * terms.abs().sum() * 4


@gpu
@pytest.mark.parametrize("type", TYPES)
def test_strides_alignment_and_shapes(type):
    t, dy, dr = make((3, 50, 264), type, "channel", 3)
    want = run(t)
    v = leaves(t)
    want_g = grads_of(v, run(v), (dy, dr))

    def wide(x):
        room = torch.full((*x.shape[:-1], x.shape[-1] + 24), float("nan"), dtype=type, device="cuda")
        room[..., 8:8 + x.shape[-1]] = x
        return room[..., 8:8 + x.shape[-1]]

    def off(x):
        return torch.empty(x.numel() + 1, dtype=type, device="cuda")[1:].view(x.shape).copy_(x)

    def turned(x):
        return x.transpose(0, -1).contiguous().transpose(0, -1)

    for how in (wide, off, turned):
        u = {k: how(x) for k, x in t.items() if x is not None}
        near = 0.0 if how is wide else 1.0  # (one element at a time: other sums)
        for a, b in zip(run(u), want):
            assert torch.equal(a, b) if not near else (a.double() - b.double()).abs().max() <= 4 * half_step(type) * b.abs().max()
        ref = Norm64(t, 0.75)
        ref.check_forward(*run(u))
        w = {k: x.detach().requires_grad_() for k, x in u.items()}
        ref.check_grads(dy, dr, grads_of(w, run(w), (how(dy), how(dr))))
    # one value everywhere has no strides
    y, r = run(v)
    one = dict(zip(v, torch.autograd.grad((y.float().sum() + r.float().sum()), [x for x in v.values()])))
    Norm64(t, 0.75).check_grads(torch.ones_like(dy), torch.ones_like(dr), one)
    assert all(want_g[k].shape == t[k].shape for k in want_g)
    y, r = residual_norm(t["residual"][0, 0], pre_weight=t["pre_weight"])
    assert y.shape == (264,)


@gpu
def test_a_residual_that_is_overwritten_before_the_backward_pass():
    """r is what the gradients are made from: the residual itself may go."""
    t, dy, dr = make((2, 5, 72), torch.bfloat16, "channel", 8)
    v = leaves(t)
    want = grads_of(v, run(v), (dy, dr))
    v = leaves(t)
    residual = v["residual"] * 1
    out = run({**v, "residual": residual})
    with torch.no_grad():
        residual.fill_(float("nan"))
    got = grads_of(v, out, (dy, dr))
    assert all(torch.equal(got[k], want[k]) for k in want)


@gpu
def test_offsets_beyond_32_bits():
    rows, d = 265000, 8192
    gen = torch.Generator(device="cuda").manual_seed(1)
    v = {k: torch.empty(rows, d, dtype=torch.float16, device="cuda").normal_(generator=gen) for k in ("residual", "block")}
    assert v["block"].numel() > 1 << 31
    w = {k: torch.rand(d, device="cuda", generator=gen).half() for k in ("post_weight", "pre_weight")}
    last = slice(rows - 20, rows)
    dy = torch.zeros_like(v["block"])
    dy[last].normal_(generator=gen)
    small = {k: x[last].clone() for k, x in v.items()}
    got, want = [], []
    for inputs, grad, out in ((v, dy, got), (small, dy[last].clone(), want)):
        a = {k: x.detach().requires_grad_() for k, x in {**inputs, **w}.items()}
        y, r = residual_norm(a["residual"], a["block"], post_weight=a["post_weight"], pre_weight=a["pre_weight"])
        out += [y.detach(), r.detach()] + list(torch.autograd.grad((y, r), list(a.values()), (grad, grad)))
    for i, (a, b) in enumerate(zip(got, want)):
        if a.dim() == 2:
            assert torch.equal(a[last], b), i
        else:  # twenty terms of about one each, added in fp32 in two orders, each sum rounded once
            assert ((a.double() - b.double()).abs() <= half_step(torch.float16) * 2.01 * b.double().abs().clamp_min(0.1)).all()
    assert not got[2][:rows - 20].any() and not got[3][:rows - 20].any()


@gpu
def test_no_rows():
    t, dy, dr = make((2, 0, 64), torch.float16, "sequence", 3)
    v = leaves(t)
    y, r = run(v)
    got = grads_of(v, (y, r), (dy, dr))
    assert y.shape == r.shape == (2, 0, 64)
    assert all(got[k].shape == t[k].shape and not got[k].any() for k in got)


@gpu
def test_zero_rows_infinities_and_nan_stay_in_their_rows():
    t, dy, dr = make((1, 40, 136), torch.float16, "channel", 3)
    want = run(t)
    v = leaves(t)
    want_g = grads_of(v, run(v), (dy, dr), ("residual", "block"))
    for name in ("residual", "block"):
        t[name][0, 3] = float("nan")
        t[name][0, 9, 5] = float("inf")
        t[name][0, 11] = 0
    v = leaves(t)
    y, r = run(v)
    keep = [i for i in range(40) if i not in (3, 9, 11)]
    assert torch.equal(y[0, keep], want[0][0, keep]) and torch.equal(r[0, keep], want[1][0, keep])
    assert y[0, 3].isnan().all() and not y[0, 11].any() and not r[0, 11].any()
    got = grads_of(v, (y, r), (dy, dr), ("residual", "block"))
    for k in got:
        assert torch.equal(got[k][0, keep], want_g[k][0, keep])
        # a row of zeros has the length 1 / sqrt(eps) = 1000: its gradient is 1000 dy pre and, through
        # the norm after the block, a thousand times that, which is beyond fp16 from dy = 0.07 on
        assert not got[k][0, 11].isnan().any()
    # the largest halves: their squares' sum is far beyond fp16
    big = torch.full((2, 4096), 65504.0, dtype=torch.float16, device="cuda")
    y, _ = residual_norm(big, pre_weight=torch.ones(4096, device="cuda").half())
    assert (y == 1).all()


@gpu
def test_refusals_on_the_gpu():
    t, _, _ = make((2, 3, 64), torch.float16, "sequence", 3)
    bad = [dict(gate=t["gate"][[0, 1, 1]]), dict(gate=t["gate"].expand(2, 3, 64)[:, :2]), dict(gate=t["gate"][..., :32]),
           dict(gate=torch.ones((), device="cuda").half()), dict(gate=torch.ones((3, 64), device="cuda").half()),
           dict(post_weight=t["post_weight"][:32]), dict(pre_weight=t["pre_weight"].reshape(1, 64)),
           dict(pre_weight=t["pre_weight"].float()), dict(block=t["block"].float()), dict(block=t["block"][:1]),
           dict(block=t["block"].cpu()), dict(eps=-1.0)]
    for change in bad:
        with pytest.raises(ValueError):
            residual_norm(**{**t, **change})
    with pytest.raises(ValueError, match="neither|belong"):
        residual_norm(t["residual"])
    with pytest.raises(ValueError, match="1 to 16384"):
        residual_norm(torch.zeros(1, 16385, device="cuda"), pre_weight=torch.ones(16385, device="cuda"))
    with pytest.raises(ValueError, match="last dimension"):
        residual_norm(torch.zeros(1, 0, device="cuda"), pre_weight=torch.ones(0, device="cuda"))


@gpu
def test_captured_replayed_and_beside_an_eager_graph_of_its_leaves():
    t, dy, dr = make((2, 40, 520), torch.bfloat16, "sequence", 3)
    v = leaves(t)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        grads_of(v, run(v), (dy, dr))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, r = run(v)
        got = grads_of(v, (y, r), (dy, dr))
    for seed in range(3):
        nt, ndy, ndr = make((2, 40, 520), torch.bfloat16, "sequence", 30 + seed)
        with torch.no_grad():
            for k in v:
                v[k].copy_(nt[k])
            dy.copy_(ndy), dr.copy_(ndr)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        w = leaves(nt)
        out = run(w)
        assert torch.equal(y, out[0]) and torch.equal(r, out[1])
        ref = grads_of(w, out, (ndy, ndr))
        assert all(torch.equal(got[k], ref[k]) for k in ref)
    del y, r, got, graph
    alive = run(v)
    with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            grads_of(v, run(v), (dy, dr))
    torch.cuda.synchronize()
    assert all(torch.isfinite(g).all() for g in grads_of(v, alive, (dy, dr)).values())


@gpu
def test_under_a_compiler():
    t, dy, dr = make((2, 40, 520), torch.bfloat16, "sequence", 3)
    v = leaves(t)
    compiled = torch.compile(lambda **kw: residual_norm(**kw, scale=0.75, eps=EPS), backend="aot_eager", fullgraph=True)
    for a, b in zip(compiled(**v), run(v)):
        assert torch.equal(a, b)
    got, want = grads_of(v, compiled(**v), (dy, dr)), grads_of(v, run(v), (dy, dr))
    assert all(torch.equal(got[k], want[k]) for k in want)
    first = torch.compile(lambda x, w: residual_norm(x, pre_weight=w)[0], backend="aot_eager", fullgraph=True)
    x, w = v["residual"], v["pre_weight"]
    a, b = first(x, w), residual_norm(x, pre_weight=w)[0]
    assert torch.equal(a, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(a, (x, w), dy), torch.autograd.grad(b, (x, w), dy)))


# --- the block -----------------------------------------------------------------------------

def block64(params, x, activation, scale, inner, gate=None):
    """y without a next norm: the definition, differentiable, in 64 bits"""
    def rms(v, w):
        return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

    y = rms(x, params["pre_weight"])
    g, u = y @ params["gate_up"][:inner].t(), y @ params["gate_up"][inner:].t()
    act = g * torch.sigmoid(g) if activation == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
    out = (act * u) @ params["down"].t()
    out = rms(out, params["post_weight"]) if "post_weight" in params else out
    gate = params.get("gate", 1.0) if gate is None else gate
    return scale * x + gate * out


@gpu
@pytest.mark.parametrize("type", TYPES[:2])
@pytest.mark.parametrize("tokens", [1, 90])
def test_the_block_and_its_gradients(type, tokens):
    """The norm of the difference: y, h, the down projection and the sum are each rounded, and so are
    in the backward pass the gradients of the block, dh, dg and du, those of g and u by their own
    rounding, y's and the result: some ten roundings, each less than e, as independent errors."""
    torch.manual_seed(0)
    for activation, gate in (("silu", False), ("gelu", True)):
        block = feedforward.FeedForward(264, 520, activation, gate=gate, scale=0.9, dtype=type, device="cuda")
        x = torch.randn(3, tokens, 264, device="cuda").to(type).requires_grad_()
        y, r = block(x, next_weight=block.pre_weight)
        params = {k: v.detach().double().requires_grad_() for k, v in block.named_parameters()}
        xd = x.detach().double().requires_grad_()
        want = block64(params, xd, activation, 0.9, 520)
        e = half_step(type)
        assert (r.detach().double() - want.detach()).norm() <= 10 * e * want.norm()
        dr = torch.randn(r.shape, device="cuda").to(type)
        got = torch.autograd.grad(r, [x, *block.parameters()], dr)
        ref = torch.autograd.grad(want, [xd, *params.values()], dr.double())
        for name, a, b in zip(["x", *params], got, ref):
            assert (a.double() - b).norm() <= 10 * e * b.norm(), name


@gpu
def test_two_blocks_share_the_norm_between_them_and_take_a_gate_per_sequence():
    torch.manual_seed(1)
    a, b = (feedforward.FeedForward(136, 264, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x = torch.randn(2, 5, 136, device="cuda").bfloat16()
    gate = torch.rand(2, 1, 136, device="cuda").bfloat16()
    y, r = a(x, gate, b.pre_weight)
    _, out = b.after_norm(y, r)
    mid = block64({k: v.double() for k, v in a.named_parameters()}, x.double(), "silu", 1.0, 264, gate.double())
    want = block64({k: v.double() for k, v in b.named_parameters()}, mid, "silu", 1.0, 264)
    assert (r.double() - mid).norm() <= 10 * 2.0 ** -8 * mid.norm()
    assert (out.double() - want).norm() <= 20 * 2.0 ** -8 * want.norm()


@gpu
@pytest.mark.parametrize("tokens", [1, 60])
def test_the_block_in_four_bits(tokens):
    """Against the dense block with the weights that four bits leave, both in fp16."""
    torch.manual_seed(2)
    dense = feedforward.FeedForward(512, 1024, "gelu", gate=True, dtype=torch.float16, device="cuda")
    four = dense.quantize(128)
    import marlin
    with torch.no_grad():
        for weight in (dense.gate_up, dense.down):
            weight.copy_(marlin.quantize(weight.half().t().contiguous(), 128)[0].t())
    x = torch.randn(tokens, 512, device="cuda").half()
    with torch.no_grad():
        want, got = dense(x)[1], four(x)[1]
        want_y, got_y = dense(x, next_weight=dense.pre_weight)[0], four(x, next_weight=four.pre_weight)[0]
    # the same weights; g, u and the down projection by other kernels, h and the sum rounded
    assert (got.double() - want.double()).norm() <= 10 * 2.0 ** -11 * want.double().norm()
    assert (got_y.double() - want_y.double()).norm() <= 10 * 2.0 ** -11 * want_y.double().norm()
    assert not any(p.requires_grad for p in four.parameters())
    with pytest.raises(ValueError):
        feedforward.FeedForward(264, 520, device="cuda").quantize()


@gpu
def test_a_training_step_in_a_graph():
    """Forward, backward and update of the whole block, captured once and replayed: every replay
    against the same step made eagerly."""
    torch.manual_seed(3)
    block = feedforward.FeedForward(136, 264, gate=True, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(70, 136, device="cuda").bfloat16()
    aim = torch.randn(70, 136, device="cuda").bfloat16()
    params = list(block.parameters())

    def step():
        _, r = block(x)
        grads = torch.autograd.grad(r, params, (r - aim).detach())
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.sub_(g, alpha=0.01)
        return r.detach()

    start = [p.detach().clone() for p in params]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()

    def reset():
        with torch.no_grad():
            for p, s in zip(params, start):
                p.copy_(s)
        torch.cuda.synchronize()

    reset()
    want = []
    for _ in range(3):
        r = step()
        want.append((r.clone(), [p.detach().clone() for p in params]))
    reset()
    for r, after in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, r)
        assert all(torch.equal(p.detach(), q) for p, q in zip(params, after))


@gpu
def test_the_block_in_four_bits_has_no_gradients_and_says_so():
    torch.manual_seed(2)
    four = feedforward.FeedForward(256, 256, gate=True, dtype=torch.float16, device="cuda").quantize(128)
    x = torch.randn(5, 256, device="cuda").half()
    with torch.no_grad():
        want = four(x, next_weight=four.pre_weight)
    # of the norms and the gate there are gradients, where none has to pass through the products
    gate = torch.rand(256, device="cuda").half().requires_grad_()
    y, r = four(x, gate, four.pre_weight)
    assert all(torch.isfinite(g).all() and g.any() for g in torch.autograd.grad((y.float() + r.float()).sum(), gate))
    x.requires_grad_()
    for backward in (lambda r: r.float().sum().backward(), lambda r: torch.autograd.grad(r.float().sum(), x)):
        y, r = four(x, next_weight=four.pre_weight)
        assert torch.equal(r, want[1]) and torch.equal(y, want[0])
        with pytest.raises(RuntimeError, match="4-bit weights have no gradients"):
            backward(r)
    normed, _ = residual_norm(x, pre_weight=four.pre_weight)
    with pytest.raises(RuntimeError, match="4-bit weights have no gradients"):
        torch.autograd.grad(four.after_norm(normed, x.detach())[1].float().sum(), x)
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.compile(lambda t: four(t)[1], backend="aot_eager", fullgraph=True)(x)
    with torch.no_grad():
        assert torch.equal(torch.compile(lambda t: four(t)[1], backend="aot_eager", fullgraph=True)(x), want[1])


@gpu
def test_second_derivatives_beside_another_path_to_the_same_input():
    t, dy, dr = make((2, 5, 72), torch.float32, "channel", 8)
    v = leaves(t)
    dy.requires_grad_()
    for name in NAMES:
        g, = torch.autograd.grad(run(v), v[name], (dy, dr), create_graph=True)
        for leaf in (*v.values(), dy):
            with pytest.raises(RuntimeError, match="differentiable once"):
                torch.autograd.grad(g.sum() + leaf.sum(), leaf, retain_graph=True)
    x, w = v["residual"], v["pre_weight"]
    g, = torch.autograd.grad(residual_norm(x, pre_weight=w)[0], w, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum() + x.sum(), x)


@gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("d", [72, 1001, 16384])
def test_infinities_of_a_block_without_a_norm_are_no_part_of_its_gradient(d, type):
    """r = scale residual + gate block is linear in the block: its gradient is gate dr, whatever is in it."""
    for gate in ("none", "channel", "sequence"):
        t, _, dr = make((2, 9, d), type, gate, 5, post=False, pre=False)
        v = leaves(t)
        want = torch.autograd.grad(run(v)[1], (v["residual"], v["block"]), dr)
        gp = 1.0 if t["gate"] is None else t["gate"].double()
        assert ((want[1].double() - gp * dr.double()).abs() <= half_step(type) * (gp * dr.double()).abs() + least(type)).all()
        t["block"][0, 3, 5] = float("inf")
        t["block"][1, 0, 70] = float("-inf")
        t["block"][1, 4] = float("nan")
        v = leaves(t)
        got = torch.autograd.grad(run(v)[1], (v["residual"], v["block"]), dr)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_the_entries_take_one_scale_for_both_passes():
    """Without a block r is the residual itself, and its gradient is that of the norm alone, whatever
    the scale."""
    import ctypes
    import marlin
    lib, L, I, D, P = marlin._lib, ctypes.c_longlong, ctypes.c_int, ctypes.c_float, ctypes.c_void_p
    rows, d = 6, 136
    t, dy, _ = make((rows, d), torch.float32, "none", 4, block=False, post=False)
    v = leaves(t)
    want_y = run(v)[0]
    want, = torch.autograd.grad(want_y, v["residual"], dy)
    x, w = t["residual"], t["pre_weight"]
    y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, 2, device="cuda")

    def at(t):
        return P(t.data_ptr())

    torch.cuda.synchronize()
    for scale in (1.0, 0.5):
        dx.fill_(float("nan"))
        stream = P(torch.cuda.current_stream().cuda_stream)
        assert lib.feedforward_norm(at(x), L(d), None, L(d), None, None, L(d), I(rows), at(w), D(scale), D(EPS), None,
                                    at(y), at(stats), L(rows), I(d), I(2), I(0), stream) == 0
        assert lib.feedforward_norm_grad(at(dy), L(d), None, L(d), at(x), L(d), None, L(d), None, None, L(d), I(rows),
                                         at(w), D(scale), at(stats), at(dx), None, None, None, None, None, L(0), L(rows),
                                         I(d), I(2), I(0), stream) == 0
        assert torch.equal(y, want_y) and torch.equal(dx, want), scale


@gpu
def test_gradients_that_are_views_to_be_read_negated():
    """As the imaginary part of a conjugate is, and what autograd makes of one."""
    for d in (1, 64):
        t, dy, dr = make((5, d), torch.float32, "channel", 4)
        v = leaves(t)
        outs = run(v)
        negated = [torch.imag(torch.complex(torch.zeros_like(g), -g).conj()) for g in (dy, dr)]
        assert all(n.is_neg() and torch.equal(n, g) for n, g in zip(negated, (dy, dr)))
        want = torch.autograd.grad(outs, list(v.values()), (dy, dr), retain_graph=True)
        for grads in (negated, [torch._neg_view(-g) for g in (dy, dr)]):
            got = torch.autograd.grad(outs, list(v.values()), grads, retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
