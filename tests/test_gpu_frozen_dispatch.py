"""GPU: the operators of test_gpu_frozen.py as the dispatcher sees them: active modes, tracing with real tensors, views with a pending negation,
forward-mode derivatives."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from lycoris_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rnd(gen, shape, dt=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dt).to(DEV)


class Heard(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


def problem(seed):
    gen = torch.Generator().manual_seed(seed)
    wq, sw = ops.int8_quantize(rnd(gen, (64, 48), torch.float32, 1 / math.sqrt(48)))
    return gen, rnd(gen, (50, 48)), wq, sw, rnd(gen, (64, 48), scale=0.15)


def test_a_dispatch_mode_hears_every_operator():
    gen, x, wq, sw, w = problem(1)
    base, g = rnd(gen, (50, 64)), rnd(gen, (50, 64))
    calls = {"int8_quantize": lambda x, w: ops.int8_quantize(x)[0].float(), "int8_matmul": lambda x, w: ops.int8_matmul(wq, sw, wq, sw),
             "int8_linear": lambda x, w: ops.int8_linear(x, wq, sw, None, base), "gated_linear": lambda x, w: ops.gated_linear(x, w, base=base),
             "gated_int8": lambda x, w: ops.gated_linear(x, wq, weight_scale=sw)}
    want = {name: call(x, w) for name, call in calls.items()}
    for name, call in calls.items():
        with Heard() as mode:
            y = call(x, w)
        assert torch.equal(y, want[name])
        op = "gated_linear" if name == "gated_int8" else name
        assert f"lycoris_amd::{op}" in mode.names and "aten::empty.memory_format" not in mode.names, (name, mode.names)
    for name, op, back in (("int8_linear", "int8_linear", "_int8_linear_backward"), ("gated_linear", "_gated_linear_forward", "_gated_linear_backward"),
                           ("gated_int8", "_gated_linear_forward", "_gated_linear_backward")):
        def step():
            leaves = [x.clone().requires_grad_(True)] + ([w.clone().requires_grad_(True)] if name == "gated_linear" else [])
            y = calls[name](*(leaves * 2)[:2])
            return [y.detach(), *torch.autograd.grad(y, leaves, g[:, :y.shape[-1]])]
        plain = step()
        with Heard() as mode:
            seen = step()
        assert all(torch.equal(a, b) for a, b in zip(plain, seen)), name
        assert f"lycoris_amd::{op}" in mode.names and f"lycoris_amd::{back}" in mode.names and "aten::empty.memory_format" not in mode.names, (name, mode.names)


def test_a_trace_of_real_tensors_computes_on_other_inputs():
    gen, x, wq, sw, w = problem(2)

    def f(x):
        return ops.int8_linear(x, wq, sw), ops.gated_linear(x, w, act="silu"), ops.gated_linear(x, wq, weight_scale=sw)

    traced = make_fx(f, tracing_mode="real")(x)
    other = rnd(gen, (50, 48))
    assert all(torch.equal(a, b) for a, b in zip(traced(other), f(other)))


def test_a_view_with_its_negation_pending_is_read_negated():
    gen, x, wq, sw, w = problem(3)
    for call in (lambda x, w: ops.int8_linear(x, wq, sw), lambda x, w: ops.gated_linear(x, w), lambda x, w: ops.gated_linear(x, wq, weight_scale=sw)):
        assert torch.equal(call(torch._neg_view(x), w), call(-x, w))
        for view in (torch._neg_view, torch.neg):
            xl = x.clone().requires_grad_(True)
            y = call(view(xl), w)
            gx, = torch.autograd.grad(y, xl, torch.ones_like(y))
            if view is torch._neg_view:
                first = (y.detach(), gx)
        assert torch.equal(first[0], y) and torch.equal(first[1], gx)
    assert torch.equal(ops.gated_linear(x, torch._neg_view(w)), ops.gated_linear(x, -w))


def test_forward_mode_is_refused():
    gen, x, wq, sw, w = problem(4)
    base = rnd(gen, (50, 64))
    for i, call in enumerate((lambda d: ops.int8_linear(d(x), wq, sw), lambda d: ops.int8_linear(x, wq, sw, base=d(base)), lambda d: ops.gated_linear(d(x), w),
                              lambda d: ops.gated_linear(x, d(w)), lambda d: ops.gated_linear(x, w, base=d(base)), lambda d: ops.gated_linear(d(x), wq, weight_scale=sw))):
        for grad in (True, False):
            with fwad.dual_level(), torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                call(lambda t: fwad.make_dual(t, torch.ones_like(t)))
                pytest.fail(f"call {i} was accepted")
