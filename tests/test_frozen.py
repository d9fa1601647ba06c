"""Host side of the 8-bit frozen layer and the gated projection: the forms for host tensors against the formulas in 64 bits, refusals,
argument checks of the C ABI (before any launch), tracing shapes, and the modules under adapters."""
import math
import re
import shutil
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.nn as nn

import lycoris_amd
from lycoris_amd import _native as N
from lycoris_amd import ops
from lycoris_amd.modules import GatedLinear, Int8Linear, LoConModule, LokrModule, quantize_frozen

GEN = torch.Generator().manual_seed(0)


def rnd(*shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=GEN) * scale).to(dtype)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 4, 33), (0, 5)])
def test_quantize(shape, dt):
    x = rnd(*shape, dtype=dt)
    q, s = ops.int8_quantize(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == x.shape[:-1] and s.dtype == torch.float32
    if x.numel():
        x64 = x.double()
        amax = x64.abs().amax(-1, keepdim=True)
        assert torch.equal(q.double(), torch.round(127 * x64 / amax)) and int(q.abs().max()) == 127
        assert ((q.double() * s.double()[..., None] - x64).abs() <= amax / 254 * (1 + 1e-6)).all()
    z = torch.zeros(2, 4, dtype=dt)
    z[1, 2] = float("inf")
    q, s = ops.int8_quantize(z)
    assert (q == 0).all() and s[0] == 0 and math.isnan(s[1])


def test_linear_and_its_gradient():
    x, w = rnd(5, 12), rnd(8, 12)
    wq, sw = ops.int8_quantize(w)
    bias, base = rnd(8), rnd(5, 8).requires_grad_(True)
    xl = x.clone().requires_grad_(True)
    y = ops.int8_linear(xl, wq, sw, bias, base)
    q, s = ops.int8_quantize(x)
    want = (q.double() @ wq.double().t()) * s.double()[:, None] * sw.double() + bias.double() + base.detach().double()
    assert (y.double() - want).abs().max() <= 8 * 2.0 ** -24 * (want.abs().max() + 10)
    g = rnd(5, 8)
    dx, db = torch.autograd.grad(y, [xl, base], g)
    assert torch.allclose(dx, g @ (wq.float() * sw[:, None]), atol=1e-5) and torch.equal(db, g)
    assert torch.allclose(ops.int8_matmul(q, s, wq, sw, bias, dtype=torch.float32), want.float() - base.detach(), atol=1e-5)


@pytest.mark.parametrize("act", sorted(ops.ACTIVATIONS))
@pytest.mark.parametrize("gate_first", [False, True])
def test_gated(act, gate_first):
    x, w, b, base = rnd(4, 6).double(), rnd(10, 6).double(), rnd(10).double(), rnd(4, 10).double()
    y = ops.gated_linear(x, w, b, base, act=act, gate_first=gate_first)
    p = x @ w.t() + b + base
    v, t = (p[:, 5:], p[:, :5]) if gate_first else (p[:, :5], p[:, 5:])
    a = {"silu": lambda t: t / (1 + torch.exp(-t)), "gelu": lambda t: t * 0.5 * (1 + torch.erf(t / 2 ** 0.5)),
         "gelu_tanh": lambda t: 0.5 * t * (1 + torch.tanh((2 / math.pi) ** 0.5 * (t + 0.044715 * t ** 3)))}[act](t)
    assert torch.allclose(y, v * a, atol=1e-12)
    wq, sw = ops.int8_quantize(w.float())
    xf = x.float().requires_grad_(True)
    yq = ops.gated_linear(xf, wq, b.float(), base.float(), act=act, gate_first=gate_first, weight_scale=sw)
    ref = ops.int8_linear(xf, wq, sw, b.float(), base.float())
    v, t = (ref[:, 5:], ref[:, :5]) if gate_first else (ref[:, :5], ref[:, 5:])
    g = rnd(4, 5)
    acts = {"silu": nn.functional.silu, "gelu": nn.functional.gelu, "gelu_tanh": lambda t: nn.functional.gelu(t, approximate="tanh")}
    want = v * acts[act](t)
    assert torch.allclose(yq, want, atol=1e-6)
    assert torch.allclose(torch.autograd.grad(yq, xf, g)[0], torch.autograd.grad(want, xf, g)[0], atol=1e-5)


def test_refusals():
    wq, sw = ops.int8_quantize(rnd(8, 12))
    x = rnd(3, 12)
    for call in (lambda: ops.int8_linear(rnd(3, 11), wq, sw), lambda: ops.int8_linear(x, wq.float(), sw), lambda: ops.int8_linear(x, wq, sw, base=rnd(3, 1)),
                 lambda: ops.int8_linear(x, wq, sw, rnd(8).requires_grad_(True)), lambda: ops.int8_linear(x, wq, sw.clone().requires_grad_(True)),
                 lambda: ops.gated_linear(x, wq), lambda: ops.gated_linear(x, rnd(7, 12)), lambda: ops.gated_linear(x, rnd(8, 12), base=rnd(3, 4)),
                 lambda: ops.gated_linear(x, rnd(8, 12), act="relu"), lambda: ops.gated_linear(x, rnd(8, 12, dtype=torch.bfloat16)),
                 lambda: ops.gated_linear(x, wq, weight_scale=sw.clone().requires_grad_(True)), lambda: ops.int8_matmul(wq, sw, wq[:, :8], sw),
                 lambda: ops.int8_quantize(x[:, :0]), lambda: ops.int8_quantize(torch.tensor(1.0))):
        with pytest.raises((RuntimeError, ValueError)):
            call()


def test_c_abi_refuses_before_any_launch():
    bf, p = N.LYC_BF16, 4096  # never dereferenced: every call below fails a check
    bad = [("lyc_int8_quantize", (p, 8, p, 16, p, 2, 8, 7, None), "dtype"), ("lyc_int8_quantize", (p, 8, p, 16, p, 2, 0, bf, None), "bad dims"),
           ("lyc_int8_quantize", (None, 8, p, 16, p, 2, 8, bf, None), "null"), ("lyc_int8_quantize", (p, 4, p, 16, p, 2, 8, bf, None), "pitch of x"),
           ("lyc_int8_quantize", (p, 8, p, 24, p, 2, 8, bf, None), "multiple of 16"), ("lyc_int8_quantize", (p, 8, p + 8, 16, p, 2, 8, bf, None), "aligned"),
           ("lyc_int8_quantize", (p, 1 << 18, p, 1 << 18, p, 2, 1 << 18, bf, None), "exceed"),
           ("lyc_int8_quantize", (p, 8, p, 16, p, (1 << 26) + 1, 8, bf, None), "exceed"),
           ("lyc_int8_matmul", (p, 1 << 17, p, p, 1 << 17, p, None, 0, None, p, p, 2, 3, 1 << 17, bf, None), "exceed"),  # 2^17 (-128)^2 = 2^31
           ("lyc_int8_matmul", (p, 16, p, p, 8, p, None, 0, None, p, p, 2, 3, 8, bf, None), "multiple of 16"),
           ("lyc_int8_matmul", (p, 16, None, p, 16, p, None, 0, None, p, p, 2, 3, 8, bf, None), "null"),
           ("lyc_int8_linear_fwd", (p, p, 16, p, None, 0, None, p, None, 64, 3, 8, bf, None), "workspace"),
           ("lyc_int8_linear_fwd", (p, p, 16, p, None, 0, None, p, p, -1, 3, 8, bf, None), "bad dims"),
           ("lyc_int8_linear_bwd", (p + 2, p, 16, p, p, p, 2, 3, 8, bf, None), "aligned"),
           ("lyc_gated_linear_fwd", (p, p, 0, None, None, 0, None, p, None, p, 2, 8, 0, 0, 0, bf, None), "bad dims"),
           ("lyc_gated_linear_fwd", (p, p, 0, None, None, 0, None, p, None, p, 2, 8, 4, 3, 0, bf, None), "activation"),
           ("lyc_gated_linear_fwd", (p, p, 8, p, None, 0, None, p, None, p, 2, 8, 4, 0, 0, bf, None), "multiple of 16"),
           ("lyc_gated_linear_fwd", (p + 4, p, 0, None, None, 0, None, p, None, p, 2, 8, 4, 0, 0, bf, None), "aligned"),
           ("lyc_gated_linear_fwd", (p, p, 0, None, None, 0, None, p, None, p, 2, 1 << 15, 1 << 16, 0, 0, bf, None), "1 GiB"),
           ("lyc_gated_linear_bwd", (p, p, p, p, 16, p, None, p, p, None, p, 2, 8, 4, 0, 0, bf, None), "frozen"),
           ("lyc_gated_linear_bwd", (p, None, p, p, 0, None, None, p, None, None, p, 2, 8, 4, 0, 0, bf, None), "null")]
    for name, args, word in bad:
        with pytest.raises(RuntimeError, match=word):
            N.call(name, *args)
    lib = N.load()
    assert lib.lyc_int8_linear_workspace_bytes(4, 8, 0, bf, 0) == -1 and lib.lyc_gated_linear_workspace_bytes(4, 8, 0, bf, 0) == -1
    assert lib.lyc_int8_linear_workspace_bytes(64, 8, 20, bf, 0) >= 64 * 32 + 256 and lib.lyc_int8_linear_workspace_bytes(4, 8, 20, bf, 0) == 0
    assert lib.lyc_gated_linear_workspace_bytes(4, 64, 8, bf, 0) == 0  # nothing to stage
    for name in ("lyc_int8_quantize", ):  # nothing to do is no error
        N.call(name, None, 8, None, 16, None, 0, 8, bf, None)


def test_tracing_shapes():
    N.load_torch_ops()
    m = dict(device="meta")
    ns = torch.ops.lycoris_amd
    x = torch.empty(2, 5, 40, dtype=torch.bfloat16, requires_grad=True, **m)
    wq, sw = torch.empty(12, 40, dtype=torch.int8, **m), torch.empty(12, **m)
    q, s = ns.int8_quantize(x.detach())
    assert q.shape == x.shape and q.stride(-2) == 128 and s.shape == (2, 5)
    y = ns.int8_linear(x, wq, sw, None, None)
    assert y.shape == (2, 5, 12) and torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == x.shape
    assert ns.int8_matmul(q, s, wq, sw, None, torch.float16).shape == (2, 5, 12)
    w, b = torch.empty(12, 40, dtype=torch.bfloat16, requires_grad=True, **m), torch.empty(12, requires_grad=True, **m)
    base = torch.empty(2, 5, 12, dtype=torch.bfloat16, requires_grad=True, **m)
    h = ns.gated_linear(x, w, None, b, base, 0, False)
    gs = torch.autograd.grad(h, [x, w, b, base], torch.empty_like(h))
    assert h.shape == (2, 5, 6) and [g.shape for g in gs] == [x.shape, w.shape, b.shape, base.shape]


class Block(nn.Module):
    def __init__(self, c, f, gated=True):
        super().__init__()
        self.to_q, self.to_out = nn.Linear(c, c, bias=False), nn.Linear(f, c)
        proj = nn.Linear(c, 2 * f)
        self.ff = GatedLinear(proj) if gated else proj

    def forward(self, x):
        h = x + self.to_q(x)
        if isinstance(self.ff, GatedLinear):
            return h + self.to_out(self.ff(h))
        v, t = self.ff(h).chunk(2, -1)
        return h + self.to_out(v * nn.functional.gelu(t))


def test_quantize_frozen_replaces_layers():
    torch.manual_seed(0)
    net = Block(16, 24).requires_grad_(False)
    net.shared = net.to_q
    want = {n: l.weight.clone() for n, l in net.named_modules() if isinstance(l, nn.Linear)}
    names = quantize_frozen(net, where=lambda n, l: n != "to_out")
    assert sorted(names) == ["ff.proj", "to_q"] and net.shared is net.to_q and type(net.to_out) is nn.Linear
    assert isinstance(net.ff.proj, Int8Linear) and isinstance(net.to_q, nn.Linear)
    for n in names:
        layer = net.get_submodule(n)
        step = want[n].abs().amax(1, keepdim=True) / 127
        assert ((layer.weight - want[n]).abs() <= step * 0.5001).all() and layer.weight.shape == want[n].shape
        assert not any(p.requires_grad for p in layer.parameters())
    with pytest.raises(TypeError):
        Int8Linear.from_linear(net.to_q)
    assert quantize_frozen(net) == ["to_out"] and quantize_frozen(net) == []
    fresh = Block(16, 24)
    quantize_frozen(fresh)
    fresh.shared = fresh.to_q
    fresh.load_state_dict(net.state_dict())
    x = rnd(3, 16)
    assert torch.equal(fresh(x), net(x))
    half = net.to(torch.float16)
    assert half.to_q.weight_scale.dtype == torch.float32 and half.to_q.weight.dtype == torch.float16 and half.to_q.weight_q.dtype == torch.int8


@pytest.mark.parametrize("algo", [LoConModule, LokrModule])
def test_adapters_on_an_int8_gated_block(algo):
    torch.manual_seed(1)
    nets = [Block(16, 24, gated) for gated in (True, False)]
    for a, b in zip(nets[0].parameters(), nets[1].parameters()):
        b.data.copy_(a.data)
    outs = []
    for net in nets:
        net.requires_grad_(False)
        quantize_frozen(net)
        layers = [net.to_q, net.ff.proj if isinstance(net.ff, GatedLinear) else net.ff, net.to_out]
        torch.manual_seed(2)
        mods = [algo(f"m{i}", l, lora_dim=4, alpha=2.0) for i, l in enumerate(layers)]
        with torch.no_grad():
            for m in mods:
                assert m.is_quant and m.bypass_mode
                for p in m.parameters():
                    p.copy_(torch.randn(p.shape) * 0.2)
        for m in mods:
            m.apply_to()
        with pytest.raises(RuntimeError, match="already carries"):
            net.extra = nn.Linear(16, 16)
            LoConModule("x", net.extra, lora_dim=4).apply_to()
            quantize_frozen(net)
        del net.extra
        for call in (mods[0].merge_to, mods[0].onfly_merge):
            with pytest.raises(NotImplementedError, match="8-bit"):
                call()
        torch.manual_seed(3)
        x = torch.randn(5, 16).requires_grad_(True)
        y = net(x)
        grads = torch.autograd.grad(y.square().sum(), [x] + [p for m in mods for p in m.parameters()])
        outs.append([y, *grads])
    for a, b in zip(*outs):
        assert torch.allclose(a, b, atol=1e-4 * float(b.detach().abs().max()) + 1e-6)


def test_casting_an_int8_layer_keeps_its_scales():
    layer = Int8Linear.from_linear(nn.Linear(40, 24))
    scale, q = layer.weight_scale.clone(), layer.weight_q.clone()
    for cast in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.float(), lambda m: m.to("cpu"), lambda m: m.double()):
        cast(layer)
        assert torch.equal(layer.weight_scale, scale) and layer.weight_scale.dtype == torch.float32 and torch.equal(layer.weight_q, q)
        assert layer.weight.dtype == layer.bias.dtype == layer.dtype
    assert layer.to(device="meta").weight_scale.device.type == "meta"


def test_gated_layer_falls_back_to_the_projection_itself():
    torch.manual_seed(4)
    proj = nn.Linear(8, 12)
    layer = GatedLinear(proj, act="silu", gate_first=True)
    x = torch.randn(3, 8)
    want = layer(x)
    t, v = proj(x).chunk(2, -1)
    assert torch.allclose(want, v * nn.functional.silu(t), atol=1e-6)
    m = LoConModule("m", proj, lora_dim=4, module_dropout=0.5)
    with torch.no_grad():
        m.lora_up.weight.normal_()
    m.apply_to()
    m.eval()
    assert layer._adapters() == [m]
    got = layer(x)
    m.train()
    assert layer._adapters() is None
    m.eval()
    t, v = proj(x).chunk(2, -1)
    assert torch.allclose(got, v * nn.functional.silu(t), atol=1e-5) and not torch.allclose(got, want, atol=1e-3)
    m.restore()
    assert layer._adapters() == [] and torch.equal(layer(x), want)
    seen = []
    hook = proj.register_forward_hook(lambda mod, args, out: seen.append(out) or out + 1)
    t, v = proj(x).chunk(2, -1)
    assert torch.allclose(layer(x), v * nn.functional.silu(t), atol=1e-6) and len(seen) == 2
    with pytest.raises(RuntimeError, match="hooks"):
        quantize_frozen(layer)
    hook.remove()
    proj.forward = lambda x: nn.functional.linear(x, proj.weight * 2, proj.bias)  # somebody else's patch
    t, v = proj(x).chunk(2, -1)
    assert torch.allclose(layer(x), v * nn.functional.silu(t), atol=1e-6)
    with pytest.raises(TypeError):
        GatedLinear(nn.Linear(8, 7))
    with pytest.raises(ValueError):
        GatedLinear(nn.Linear(8, 6), act="relu")
    assert lycoris_amd.GatedLinear is GatedLinear


def test_forward_mode_is_refused_and_not_dropped():
    """the device operators have no jvp: a dual input, which need not require a gradient, is an error and not an output without its tangent"""
    N.load_torch_ops()
    ns, m = torch.ops.lycoris_amd, dict(device="meta")
    wq, sw = torch.empty(12, 40, dtype=torch.int8, **m), torch.empty(12, **m)
    x, w, bias, base = torch.empty(5, 40, **m), torch.empty(12, 40, **m), torch.empty(12, **m), torch.empty(5, 12, **m)
    calls = [(lambda x, sw, bias, base: ns.int8_linear(x, wq, sw, bias, base), (x, sw, bias, base)),
             (lambda x, sw, bias, base: ns.gated_linear(x, wq, sw, bias, base, 0, False), (x, sw, bias, base)),
             (lambda x, w, bias, base: ns.gated_linear(x, w, None, bias, base, 0, False), (x, w, bias, base))]
    for call, args in calls:
        for i in range(len(args)):
            for grad in (True, False):
                with fwad.dual_level(), torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                    call(*[fwad.make_dual(t, torch.empty_like(t)) if j == i else t for j, t in enumerate(args)])
        assert call(*args).shape[0] == 5  # and without a tangent nothing is
    # the host forms are differentiable either way
    x = rnd(3, 12, dtype=torch.float64)
    q, s = ops.int8_quantize(rnd(8, 12))
    t = rnd(3, 12, dtype=torch.float64)
    with fwad.dual_level():
        got = fwad.unpack_dual(ops.int8_linear(fwad.make_dual(x, t), q, s)).tangent
    assert torch.allclose(got, t @ (q.double() * s.double()[:, None]).t())


def test_every_product_kernel_has_its_own_lds_limit_flags():
    """the limit of dynamic LDS is raised per kernel and device, and remembered: one set of flags for all kernels of a type would leave it at
    the default for all but the first one launched"""
    N.load()
    nm = shutil.which("nm") or "/opt/rocm/llvm/bin/llvm-nm"
    names = subprocess.run([nm, N.lib_path()], check=True, capture_output=True, text=True).stdout.split()
    kernels = [n for n in names if re.search(r"__device_stub__fz_(gemm|skinny)_kernel", n)]
    flags = [n for n in names if "allow_lds" in n and n.endswith("E4done")]
    assert len(kernels) > 50 and len(set(flags)) == len(set(kernels))
