"""GPU: every tile and split of the products (frozen_plans.py) against the formulas in 64 bits.

Bounds, elementwise, from the arithmetic: u = eps / 2 of a type is one rounding to it, e = 2^-24 one to fp32, n e S the error of a sum of n fp32 terms of
magnitudes S.  8-bit products are exact integers.  Three-plane fp32 operands: 6 n e S (3 n e S beside exact integers).  The gradients' operands beside 16-bit
types: one rounding to 11 bits (bf16) or 22 (fp16) of a term, and 2^-39 of the largest of their row."""
import math

import pytest
import torch

from frozen_plans import BASE, BF16, F16, F32, INT8, KEEP, PLANS, PRODUCTS
from lycoris_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
ACT_ERR = 2.0 ** -17
DT = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
TERM = {F32: 0.0, BF16: 2.0 ** -11, F16: 2.0 ** -22}
STEP = {F32: 0.0, BF16: 2.0 ** -39, F16: 2.0 ** -39}
PLANES = {F32: 3, F16: 2, BF16: 1}


def normal(gen, shape, dt, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dt)


def held(gen, N, K):
    q, s = ops.int8_quantize(normal(gen, (N, K), torch.float32, 1 / math.sqrt(K)) * torch.exp(0.3 * normal(gen, (N, 1), torch.float32)))
    return q, s, q.double() * s.double()[:, None]


def within(got, want, bound, dtype, what):
    f = torch.finfo(DT[dtype])
    bound = bound + f.eps / 2 * (want.abs() + bound) + f.smallest_normal * f.eps / 2
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound).all(), (what, float((off - bound).max()), float((off / bound).max()), int((off > bound).sum()))


def poison(like):
    """NaNs in the memory that outputs and workspaces come from"""
    blocks = [torch.full((n,), float("nan"), device=DEV) for n in [1 << 20] * 16 + [1 << 24] * 4]
    del blocks


def silu64(t):
    s = torch.sigmoid(t)
    return t * s, s * (1 + t * (1 - s))


def label(c):
    return f"{PRODUCTS[c[0]]}-{('f32', 'f16', 'bf16')[c[1]]}-{c[2]}x{c[3]}x{c[4]}-{c[5]}-tile{c[6]}{'-parts' if c[7] else ''}"


@pytest.mark.parametrize("case", [c for c in PLANS if c[0] == 0], ids=label)
def test_int8_forward(case):
    _, dtype, M, K, N, _, tile, parts = case
    gen, dt = torch.Generator(device=DEV).manual_seed(M + K + N), DT[dtype]
    x = normal(gen, (M, K), dt)
    wq, sw, _ = held(gen, N, K)
    bias, base = normal(gen, (N,), dt, 0.2), normal(gen, (M, N), dt, 0.3)
    poison(x)
    y = ops.int8_linear(x, wq, sw, bias, base)
    x64 = x.double()
    top = x64.abs().amax(1, keepdim=True)
    q = torch.round(127.0 * x64 / top)
    p = (q @ wq.double().t().contiguous()) * (top.float() / 127.0).double() * sw.double()
    want, mag = p + bias.double() + base.double(), p.abs() + bias.double().abs() + base.double().abs()
    within(y, want, 6 * E * mag, dtype, "y")


@pytest.mark.parametrize("case", [c for c in PLANS if c[0] == 1], ids=label)
def test_int8_dx(case):
    _, dtype, M, K, N, _, tile, parts = case
    gen, dt = torch.Generator(device=DEV).manual_seed(M + K + N), DT[dtype]
    g = normal(gen, (M, N), dt, 1 / math.sqrt(N))
    wq, sw, w64 = held(gen, N, K)
    x = torch.zeros(M, K, dtype=dt, device=DEV, requires_grad=True)
    y = ops.int8_linear(x, wq, sw)
    poison(x)
    dx, = torch.autograd.grad(y, x, g)
    g64 = g.double()
    want, mag = g64 @ w64, g64.abs() @ w64.abs()
    top = (g64 * sw.double()).abs().amax(1, keepdim=True)
    bound = (TERM[dtype] + 3 * E + (PLANES[dtype] * N + 8) * E) * mag * 1.01 + STEP[dtype] * top * wq.double().abs().sum(0)
    within(dx, want, bound, dtype, "dx")


def gated(case, gen):
    """operands, and p with what it may be off by"""
    _, dtype, M, K, F, flags, tile, parts = case
    dt, int8 = DT[dtype], bool(flags & INT8)
    x = normal(gen, (M, K), dt)
    sw = None
    bias, base = normal(gen, (2 * F,), dt, 0.2), normal(gen, (M, 2 * F), dt, 0.3) if flags & BASE else None
    x64 = x.double()
    if int8:
        w, sw, w64 = held(gen, 2 * F, K)
        top = x64.abs().amax(1, keepdim=True)
        p = (torch.round(127.0 * x64 / top) @ w.double().t().contiguous()) * (top.float() / 127.0).double() * sw.double()
        mag, terms = p.abs(), 6
    else:
        w = normal(gen, (2 * F, K), dt, 1 / math.sqrt(K))
        w64 = w.double()
        p, mag = x64 @ w64.t().contiguous(), x64.abs() @ w64.abs().t().contiguous()
        terms = K + 4 if dtype != F32 else 6 * K + 16
    for t in (bias, base):
        if t is not None:
            p, mag = p + t.double(), mag + t.double().abs()
    return x, w, sw, w64, bias, base, p, terms * E * mag


@pytest.mark.parametrize("case", [c for c in PLANS if c[0] == 2], ids=label)
def test_gated_forward(case):
    _, dtype, M, K, F, flags, tile, parts = case
    x, w, sw, w64, bias, base, p, ep = gated(case, torch.Generator(device=DEV).manual_seed(M + K + F))
    poison(x)
    gate_first = F % 2 == 0
    pre = None
    if flags & KEEP:
        h, pre = torch.ops.lycoris_amd._gated_linear_forward(x, w, sw, bias, base, ops.ACTIVATIONS["silu"], gate_first)
    else:
        h = ops.gated_linear(x, w, bias, base, act="silu", gate_first=gate_first, weight_scale=sw)
    (v, t), (ev, et) = (m.split(F, 1)[::-1] if gate_first else m.split(F, 1) for m in (p, ep))
    a = silu64(t)[0]
    within(h, v * a, a.abs() * ev + (v.abs() + ev) * (1.2 * et + ACT_ERR * (t.abs() + 1)), dtype, "h")
    if pre is None:
        return
    n = M * 2 * F
    if dtype == F32:
        kept = pre.view(torch.float32)
    else:
        kept = ((pre[:2 * n].view(torch.int16).int() << 16) | (pre[2 * n:].int() << 8)).view(torch.float32)
    off = (kept.double().view(M, 2 * F) - p).abs()
    bound = ep + (0.0 if dtype == F32 else 2.0 ** -16) * (p.abs() + ep)
    assert (off <= bound * 1.001 + 1e-30).all(), float((off - bound).max())


@pytest.mark.parametrize("case", [c for c in PLANS if c[0] >= 3], ids=label)
def test_gated_gradients(case):
    product, dtype, M, K, F, flags, tile, parts = case
    gen = torch.Generator(device=DEV).manual_seed(M + K + F)
    x, w, sw, w64, bias, base, p, ep = gated(case, gen)
    g = normal(gen, (M, F), DT[dtype], 1 / math.sqrt(F))
    xl, wl = x.clone().requires_grad_(product == 3), w.clone().requires_grad_(product == 4)
    h = ops.gated_linear(xl, wl, bias, act="silu", weight_scale=sw)
    poison(x)
    got, = torch.autograd.grad(h, xl if product == 3 else wl, g)
    ep = ep + (0.0 if dtype == F32 else 2.0 ** -16) * (p.abs() + ep)
    (v, t), (ev, et) = p.split(F, 1), ep.split(F, 1)
    g64, (a, da), afp = g.double(), silu64(t), ACT_ERR * (t.abs() + 1)
    dp = torch.cat((g64 * a, g64 * v * da), 1)
    e = torch.cat((g64.abs() * (1.2 * et + afp + E * a.abs()), g64.abs() * ((da.abs() + afp) * ev + (v.abs() + ev) * (et + afp) + 3 * E * (v * da).abs())), 1)
    c = sw.double() if sw is not None else 1.0
    top = (dp * c).abs().amax(1, keepdim=True)
    e = e + (TERM[dtype] + 3 * E) * (dp.abs() + e) + STEP[dtype] * top / c
    if product == 3:
        n, other, largest = (6 if dtype == F32 and sw is None else PLANES[dtype]) * 2 * F, w64, w64.abs().max() * (sw is None)
        want, mag, err = dp @ other, dp.abs() @ other.abs(), e @ other.abs()
        lost = STEP[dtype] * largest * dp.abs().sum(1, keepdim=True)
    else:
        n, other = (6 if dtype == F32 else PLANES[dtype]) * M, x.double()
        left = dp.t().contiguous()
        want, mag, err = left @ other, left.abs() @ other.abs(), e.t().contiguous() @ other.abs()
        lost = STEP[dtype] * 2 * top.max() * other.abs().max() * (dp.abs() / top).sum(0)[:, None]
    within(got, want, err * 1.01 + (n + 16) * E * mag * 1.01 + lost, dtype, "gradient")
