"""Calls that something looks at: dispatch modes, make_fx, fake tensors, torch.jit.trace.

The calls launch behind torch's dispatcher, where a recorder sees the outputs' allocation and nothing
of what fills them.  Where one is at work they go through operators of their own, marlin_amd::*, and
what was recorded gives, run again on other inputs, what the calls give.
"""
import os
import sys

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "awesome-cute_amd"))
import feedforward  # noqa: E402
import marlin  # noqa: E402
import streamk  # noqa: E402

gpu = pytest.mark.gpu


def layers(dev):
    """A gated layer and a plain one of the same weights."""
    gen = torch.Generator().manual_seed(0)
    out = []
    for layer in (marlin.GatedLayer(256, 256, 128, "gelu"), marlin.Layer(256, 256, 128)):
        layer.B.copy_(torch.randint(-2 ** 31, 2 ** 31 - 1, layer.B.shape, generator=gen))
        layer.s.copy_(torch.rand(layer.s.shape, generator=gen) * 0.02)
        out.append(layer.to(dev))
    return out


def calls(dev="cpu"):
    """name -> (function, input shapes, the operators it is made of)"""
    gated_layer, layer = layers(dev)

    def into(mul, layer, width):
        def call(x):
            C = x.new_zeros(x.shape[0], width)
            mul(x, layer.B, C, layer.s, layer.workspace)
            return C
        return call

    return {
        "gated": (lambda x, w: streamk.gated(x, w, "gelu"), ((20, 64), (96, 64)), ["gated_alone"]),
        "linear": (lambda x, w: streamk.linear(x, w), ((20, 64), (96, 64)), ["linear_dense"]),
        "gemm": (lambda x, w: streamk.gemm(x, w), ((20, 64), (256, 64)), ["gemm"]),
        "norm": (lambda x, w: feedforward.residual_norm(x, pre_weight=w)[0], ((3, 5, 64), (64,)), ["residual_norm"]),
        "norms": (lambda x, b, w: feedforward.residual_norm(x, b, post_weight=w, gate=w, pre_weight=w),
                  ((20, 64), (20, 64), (64,)), ["residual_norm"]),
        "gated layer": (lambda x: gated_layer(x), ((3, 5, 256),), ["gated_linear"]),
        "layer": (lambda x: layer(x), ((15, 256),), ["mul"]),
        "gated mul": (into(marlin.gated_mul, gated_layer, 256), ((15, 256),), ["gated_mul"]),
        "mul": (into(marlin.mul, layer, 256), ((15, 256),), ["mul"]),
    }


NAMES = sorted(calls())


def make(shapes, seed, dev="cuda"):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=gen).half().to(dev) for shape in shapes]


def operators(graph):
    return [str(n.target).split(".")[1] for n in graph.graph.nodes if str(n.target).startswith("marlin_amd.")]


def same(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("name", NAMES)
def test_fake_tensors_record_the_operators(name):
    call, shapes, want = calls()[name]
    with torch.no_grad():
        graph = make_fx(call, tracing_mode="fake", _allow_non_fake_inputs=True)(*make(shapes, 0, "cpu"))
    assert operators(graph) == want


def test_fake_tensors_record_the_backward_passes():
    def step(x, w, b, p):
        h = streamk.linear(streamk.gated(x, w), b)
        y, r = feedforward.residual_norm(x, h, pre_weight=p)
        return torch.autograd.grad((y, r), (x, w, b, p), (y, r))

    inputs = [t.requires_grad_() for t in make(((20, 64), (96, 64), (64, 48), (64,)), 0, "cpu")]
    graph = make_fx(step, tracing_mode="fake")(*inputs)
    assert operators(graph) == ["gated_dense", "linear_dense", "residual_norm", "norm_grads", "linear_grads", "gated_grads"]


class Record(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "marlin_amd":
            self.seen.append(func.name().split("::")[1].split(".")[0])
        return func(*args, **(kwargs or {}))


@gpu
@pytest.mark.parametrize("name", NAMES)
def test_modes_see_the_operators(name):
    call, shapes, want = calls("cuda")[name]
    inputs = make(shapes, 1)
    eager = call(*inputs)
    with Record() as record:
        got = call(*inputs)
    assert record.seen == want and same(got, eager)
    assert same(call(*inputs), eager)


@gpu
@pytest.mark.parametrize("name", NAMES)
def test_what_was_recorded_is_the_call(name):
    call, shapes, want = calls("cuda")[name]
    first, other = make(shapes, 1), make(shapes, 2)
    with torch.no_grad():
        graph = make_fx(call)(*first)
        traced = torch.jit.trace(call, tuple(first), check_trace=False)
    assert operators(graph) == want
    assert all(f"marlin_amd::{op}" in str(traced.graph) for op in want)
    for inputs in (other, first):
        eager = call(*inputs)
        assert same(graph(*inputs), eager)
        assert same(traced(*inputs), eager)


@gpu
def test_gradients_under_a_mode():
    x, w, dy = make(((20, 64), (96, 64), (20, 96)), 3)
    x.requires_grad_()
    w.requires_grad_()
    want = torch.autograd.grad(streamk.linear(x, w), (x, w), dy)
    with Record() as record:
        got = torch.autograd.grad(streamk.linear(x, w), (x, w), dy)
    assert same(got, want) and record.seen[0] == "linear_dense"


def backward_calls(call, inputs):
    """The backward operators' nodes of a compiled call, and the gradients that it gives."""
    from torch._dynamo.backends.common import aot_autograd
    from functorch.compile import make_boxed_func
    nodes = []

    def backward(graph, example):
        nodes.extend(n for n in graph.graph.nodes if "_grads" in str(n.target))
        return make_boxed_func(graph.forward)

    torch._dynamo.reset()
    compiled = torch.compile(call, backend=aot_autograd(fw_compiler=lambda g, e: make_boxed_func(g.forward),
                                                        bw_compiler=backward), fullgraph=True)
    wanted = [t for t in inputs if t.requires_grad]
    outs = compiled(*inputs)
    outs = outs if isinstance(outs, tuple) else (outs,)
    return nodes, torch.autograd.grad(outs, wanted, [o.detach() for o in outs])


@gpu
@pytest.mark.parametrize("frozen", [0, 1])
@pytest.mark.parametrize("name", ["gated", "linear"])
def test_compiled_backward_passes_compute_what_is_wanted(name, frozen):
    call, shapes, _ = calls("cuda")[name]
    inputs = make(shapes, 4)
    inputs[1 - frozen].requires_grad_()
    nodes, got = backward_calls(call, inputs)
    out = call(*inputs)
    assert same(got, torch.autograd.grad(out, inputs[1 - frozen], out.detach()))
    assert [n.args[-2:] for n in nodes] == [(frozen == 1, frozen == 0)]


@gpu
def test_compiled_backward_passes_of_norms_compute_what_is_wanted():
    shapes = ((20, 64), (20, 64), (64,), (64,), (64,))

    def call(x, b, post, gate, pre):
        return feedforward.residual_norm(x, b, post_weight=post, gate=gate, pre_weight=pre)

    for wanted in ((0, 1), (2, 4), (3,), (0, 1, 2, 3, 4)):
        inputs = [t.requires_grad_(i in wanted) for i, t in enumerate(make(shapes, 5))]
        nodes, got = backward_calls(call, inputs)
        outs = call(*inputs)
        assert same(got, torch.autograd.grad(outs, [inputs[i] for i in wanted], [o.detach() for o in outs]))
        assert [n.args[-1] for n in nodes] == [[i in wanted for i in range(5)]]
