"""GPU: frozen layers held in 8 bits (ops.int8_quantize / int8_matmul / int8_linear) and the gated projection (ops.gated_linear) against
the formulas in 64 bits on the same inputs.

Bounds are elementwise and come from the arithmetic.  u = eps / 2 of the activation type is one rounding to it, e = 2^-24 one rounding to
fp32.  A sum of n fp32 terms is off by at most n e times the sum of their magnitudes S.  8-bit products are exact integers below 2^31, so
the 8-bit forward has no n: converting, two scales, bias and base are five roundings.  fp32 operands run as six bf16 products per term
(what is left out is below 3 e of a term): 6 n e S.  The backward pass reads p cut to its upper 24 bits (2^-15 |p|; fp32: as it is) and, over
an 8-bit weight, sw q or sw dp rounded to the activation type (u S)."""
import math

import pytest
import torch

from lycoris_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "f16", "f32"]


def u_of(dt):
    return torch.finfo(dt).eps / 2


def sub_of(dt):
    """half the spacing of the numbers below the smallest normal one (fp16: 2^-14 * 2^-10 / 2 = 2^-25): there a rounding is off by that much,
    whatever the value, and not by u of it"""
    f = torch.finfo(dt)
    return f.smallest_normal * f.eps / 2


def rnd(gen, shape, dt, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dt).to(DEV)


def f64(t):
    return None if t is None else t.detach().double().cpu()


def quantize64(x):
    """(q, scale) of the definition, both float64; scale as the fp32 the op returns"""
    x = x.double().cpu()
    amax = x.abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * x / torch.where(amax > 0, amax, torch.ones_like(amax)))
    return q, (amax.float() / 127.0).double()


def poison():
    """leave NaNs in the memory that the next calls' outputs and workspaces come from"""
    blocks = [torch.full((n,), float("nan"), device=DEV) for n in [1 << 17] * 24 + [1 << 22] * 4 + [1 << 25]]
    del blocks


def within(got, want, bound, what):
    sub = sub_of(got.dtype)
    got = f64(got).reshape(want.shape)
    over = (got - want).abs() - (bound + sub)
    assert torch.isfinite(got).all(), what
    assert (over <= 0).all(), f"{what}: off by {float((got - want).abs().max()):.3e}, {float(over.max()):.3e} over its bound"


def held(gen, N, K):
    w = torch.randn(N, K, generator=gen) / math.sqrt(K) * torch.exp(0.3 * torch.randn(N, 1, generator=gen))
    q, s = ops.int8_quantize(w.to(DEV))
    return q, s


# ---- int8_quantize -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 16), (3, 7), (2, 5, 200), (65, 640), (7, 1001), (3, 1536), (2, 4104), (5, 8200), (2, 20001), (0, 64), (300, 320)])
def test_quantize_is_exact(shape, dt):
    gen = torch.Generator().manual_seed(sum(shape))
    x = rnd(gen, shape, dt)
    q, s = ops.int8_quantize(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and s.shape == x.shape[:-1] and s.dtype == torch.float32
    if x.numel() == 0:
        return
    q64, s64 = quantize64(x)
    assert torch.equal(q.cpu().double(), q64)
    assert torch.equal(s.cpu().double(), s64[..., 0])


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_quantize_halves_zeros_extremes_and_non_finite_rows(dt):
    K = 200
    top = torch.finfo(dt).max
    rows = [torch.zeros(K), torch.arange(K) / 2.0 * (127.0 / 127.0), -torch.arange(K).float() / 4, torch.full((K,), 1.5),
            torch.where(torch.arange(K) % 2 == 0, 1.0, 0.5), torch.linspace(-1, 1, K) * top, torch.linspace(-1, 1, K) * torch.finfo(dt).tiny]
    rows[1][0] = 127.0  # max 127 -> halves are exact halves
    rows[1].clamp_(max=127.0)
    x = torch.stack(rows).to(dt).to(DEV)
    q, s = ops.int8_quantize(x)
    q64, s64 = quantize64(x)
    assert torch.equal(q.cpu().double(), q64) and torch.equal(s.cpu().double(), s64[:, 0])
    bad = torch.randn(4, K).to(dt)
    bad[0, 3], bad[1, 199], bad[2, 0] = float("inf"), float("nan"), -float("inf")
    q, s = ops.int8_quantize(bad.to(DEV))
    assert torch.isnan(s[:3]).all() and (q[:3] == 0).all() and torch.isfinite(s[3]) and (q[3] != 0).any()


def test_quantize_strided_and_misaligned_rows():
    gen = torch.Generator().manual_seed(5)
    big = rnd(gen, (40, 300), torch.bfloat16)
    column = rnd(gen, (300, 1), torch.bfloat16)
    q, s = ops.int8_quantize(column.t())  # one row whose pitch is 1
    assert torch.equal(q.cpu().double(), quantize64(column.t())[0])
    for x in (big[:, 3:203], big[::2, :128], big.t(), big[:, ::2], big[5:6].expand(4, 300), big[:, 8:264]):
        q, s = ops.int8_quantize(x)
        q64, s64 = quantize64(x)
        assert torch.equal(q.cpu().double(), q64) and torch.equal(s.cpu().double(), s64[..., 0])


# ---- int8_linear ---------------------------------------------------------------------------------------------------------------------------
LINEAR = [(1, 1, 1), (1, 64, 64), (1, 1280, 1280), (2, 48, 40), (5, 200, 17), (16, 1280, 640), (17, 129, 130), (77, 2048, 640), (64, 16, 8), (130, 640, 333),
          (257, 96, 1000), (333, 1001, 77), (513, 1280, 520), (1024, 320, 1280), (2100, 264, 1032)]


def linear_reference(x, wq, sw, bias, base):
    q, s = quantize64(x.reshape(-1, x.shape[-1]))
    p = (q @ f64(wq).t()) * s * f64(sw)
    mag = p.abs()
    for t in (bias, base):
        if t is not None:
            t = f64(t).reshape(-1, p.shape[1]) if t.dim() > 1 else f64(t)
            p, mag = p + t, mag + t.abs()
    return p, 6 * E * mag


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", LINEAR)
def test_linear_forward_and_dx(M, K, N, dt):
    gen = torch.Generator().manual_seed(M + K + N)
    lead = (2, M // 2) if M % 2 == 0 else (M,)
    x = rnd(gen, (*lead, K), dt)
    wq, sw = held(gen, N, K)
    bias = rnd(gen, (N,), dt if M % 3 else torch.float32, 0.1) if (M + N) % 2 else None
    base = rnd(gen, (*lead, N), dt, 0.3) if K % 3 else None
    xl = x.clone().requires_grad_(True)
    bl = None if base is None else base.clone().requires_grad_(True)
    poison()
    y = ops.int8_linear(xl, wq, sw, bias, bl)
    assert y.shape == (*lead, N) and y.dtype == dt
    want, err = linear_reference(x, wq, sw, bias, base)
    u = u_of(dt)
    within(y, want, err + u * (want.abs() + err), "y")
    g = rnd(gen, (*lead, N), dt, 1 / math.sqrt(N))
    grads = torch.autograd.grad(y, [xl] + ([] if bl is None else [bl]), g)
    w64, g64 = f64(wq) * f64(sw)[:, None], f64(g).reshape(-1, N)
    dx, S = g64 @ w64, g64.abs() @ w64.abs()
    # 16-bit: the weight's rounding; fp16's plane is rescaled by a power of two (exact).  fp32: g sw rounded, three products
    rel = (u + (N + 2) * E) if dt != torch.float32 else (3 * N + 8) * E
    within(grads[0], dx, rel * S * 1.01 + u * dx.abs(), "dx")
    assert grads[0].shape == x.shape
    if bl is not None:
        assert torch.equal(grads[1], g)
    with torch.no_grad():
        assert torch.equal(ops.int8_linear(x, wq, sw, bias, base), y)
    with torch.inference_mode():
        assert torch.equal(ops.int8_linear(x, wq, sw, bias, base), y)


@pytest.mark.parametrize("M,K,N,dt", [(3850, 5130, 3900, torch.bfloat16), (4090, 1276, 10250, torch.bfloat16), (4090, 1276, 10250, torch.float32)],
                         ids=["large", "long", "long_f32"])
def test_long_ragged_products(M, K, N, dt):
    """the largest tiles over many K steps, in one part and in several, with rows, columns and K that end inside a tile"""
    gen = torch.Generator(device=DEV).manual_seed(M)
    x, g = (torch.randn(M, n, generator=gen, device=DEV).to(dt) for n in (K, N))
    wq, sw = ops.int8_quantize(torch.randn(N, K, generator=gen, device=DEV) / math.sqrt(K))
    poison()
    xl = x.clone().requires_grad_(True)
    y = ops.int8_linear(xl, wq, sw)
    dx, = torch.autograd.grad(y, xl, g)
    assert torch.isfinite(y).all() and torch.isfinite(dx).all()
    rows = torch.cat((torch.arange(0, M, 97), torch.tensor([255, 256, M - 2, M - 1]))).to(DEV)
    want, err = linear_reference(x[rows], wq, sw, None, None)
    within(y[rows], want, err + u_of(dt) * (want.abs() + err), "y")
    w64, g64 = f64(wq) * f64(sw)[:, None], f64(g[rows])
    want, S = g64 @ w64, g64.abs() @ w64.abs()
    u = u_of(dt)
    rel = (u + (N + 2) * E) if dt != torch.float32 else (3 * N + 8) * E
    within(dx[rows], want, rel * S * 1.01 + u * want.abs(), "dx")


def test_linear_operands_of_other_layouts():
    gen = torch.Generator().manual_seed(3)
    M, K, N = 50, 203, 96
    wq, sw = held(gen, N, K)
    x = rnd(gen, (M, K), torch.bfloat16)
    want = ops.int8_linear(x, wq, sw)
    packed = wq.contiguous()  # pitch 203: copied inside
    assert packed.stride(0) == K and torch.equal(ops.int8_linear(x, packed, sw), want)
    wide = torch.full((N, 256), 77, dtype=torch.int8, device=DEV)  # a pitch with values behind K
    wide[:, :K] = wq
    assert torch.equal(ops.int8_linear(x, wide[:, :K], sw), want)
    assert torch.equal(ops.int8_linear(x, wq.t().contiguous().t(), sw), want)
    room = torch.empty(M * K + 1, dtype=torch.bfloat16, device=DEV)
    off = room[1:].view(M, K).copy_(x)
    assert off.data_ptr() % 16 and torch.equal(ops.int8_linear(off, wq, sw), want)
    assert torch.equal(ops.int8_linear(x.t().contiguous().t(), wq, sw), want)
    assert torch.equal(ops.int8_linear(x, wq, sw[:, None]), want)
    xl = x.clone().requires_grad_(True)
    ops.int8_linear(xl, packed, sw).sum().backward()  # an expanded gradient
    ref = x.clone().requires_grad_(True)
    ops.int8_linear(ref, wq, sw).backward(torch.ones(M, N, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(xl.grad, ref.grad)


def test_linear_empty_batch_and_non_finite_rows():
    gen = torch.Generator().manual_seed(4)
    wq, sw = held(gen, 64, 96)
    x = torch.empty(0, 96, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = ops.int8_linear(x, wq, sw)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == (0, 96)
    x = rnd(gen, (40, 96), torch.bfloat16)
    want = ops.int8_linear(x, wq, sw)
    x[7, 3] = float("nan")
    x[20, 95] = float("inf")
    y = ops.int8_linear(x, wq, sw)
    rest = [m for m in range(40) if m not in (7, 20)]
    assert torch.isnan(y[7]).all() and torch.isnan(y[20]).all() and torch.equal(y[rest], want[rest])
    x[0] = 0
    assert (ops.int8_linear(x, wq, sw)[0] == 0).all()


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_dx_of_weights_far_from_one(dt):
    """scales at both ends of what fp16 can hold: its weight plane is brought into range by a power of two"""
    gen = torch.Generator().manual_seed(9)
    M, K, N = 33, 64, 80
    for factor in (1e-7, 3e3):
        q, s = ops.int8_quantize((torch.randn(N, K, generator=gen) * factor).to(DEV))
        x = rnd(gen, (M, K), dt).requires_grad_(True)
        g = rnd(gen, (M, N), dt, 1e-2 / max(factor, 1e-3))
        y = ops.int8_linear(x, q, s)
        dx, = torch.autograd.grad(y, x, g)
        w64, g64 = f64(q) * f64(s)[:, None], f64(g)
        want, S = g64 @ w64, g64.abs() @ w64.abs()
        u = u_of(dt)
        rel = (u + (N + 2) * E) if dt != torch.float32 else (3 * N + 8) * E
        within(dx, want, rel * S * 1.01 + u * want.abs(), f"dx {factor}")


# ---- int8_matmul --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 640, 320), (3, 50, 9), (40, 77, 64), (129, 256, 200), (300, 1000, 520)])
def test_matmul(M, K, N, dt):
    gen = torch.Generator().manual_seed(M * K + N)
    aq = torch.randint(-128, 128, (M, K), generator=gen, dtype=torch.int8).to(DEV)
    bq = torch.randint(-128, 128, (N, K), generator=gen, dtype=torch.int8).to(DEV)
    sa, sb = (torch.rand(M, generator=gen) + 0.1).to(DEV), (torch.rand(N, generator=gen) / K).to(DEV)
    bias = rnd(gen, (N,), dt) if N % 2 else None
    p = (f64(aq) @ f64(bq).t()) * f64(sa)[:, None] * f64(sb)
    mag = p.abs() + (0 if bias is None else f64(bias).abs())
    want = p if bias is None else p + f64(bias)
    bound = 6 * E * mag + u_of(dt) * (want.abs() + 6 * E * mag)
    poison()
    within(ops.int8_matmul(aq, sa, bq, sb, bias, dtype=dt), want, bound, "y")
    pitch = (K + 15) // 16 * 16 + 16
    wide = torch.full((M, pitch), -5, dtype=torch.int8, device=DEV)  # rows with values behind K
    wide[:, :K] = aq
    within(ops.int8_matmul(wide[:, :K], sa, bq, sb, bias, dtype=dt), want, bound, "y of a slice")


def test_matmul_shares_one_quantised_input():
    gen = torch.Generator().manual_seed(8)
    x = rnd(gen, (2, 60, 320), torch.bfloat16)
    xq, sx = ops.int8_quantize(x)
    for N in (320, 100):
        wq, sw = held(gen, N, 320)
        assert torch.equal(ops.int8_matmul(xq, sx, wq, sw, dtype=torch.bfloat16), ops.int8_linear(x, wq, sw))


# ---- gated_linear ---------------------------------------------------------------------------------------------------------------------------
def act64(name, t):
    """act, act', and a bound on |act''|"""
    if name == "silu":
        s = torch.sigmoid(t)
        return t * s, s * (1 + t * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-t / math.sqrt(2))
        return t * c, c + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    s = torch.sigmoid(2 * k * (t + 0.044715 * t ** 3))
    return t * s, s + 2 * t * s * (1 - s) * k * (1 + 0.134145 * t * t)


ACT_ERR = 2.0 ** -17  # of the fp32 activation and its derivative, relative to |t| + 1: the exponential's argument is rounded (|t| e each way)


def gated_reference(x, w64, bias, base, act, gate_first, g, dt, held_weight, p_of_q=None):
    """{name: (value, bound)} of h and of every gradient"""
    u, K = u_of(dt), x.shape[-1]
    x64 = f64(x).reshape(-1, K)
    F = w64.shape[0] // 2
    if held_weight:
        p, Sp, terms = p_of_q, p_of_q.abs(), 6
    else:
        p, Sp = x64 @ w64.t(), x64.abs() @ w64.abs().t()
        terms = K + 4 if dt != torch.float32 else 6 * K + 16
    for t in (bias, base):
        if t is not None:
            t = f64(t).reshape(-1, 2 * F) if t.dim() > 1 else f64(t)
            p, Sp = p + t, Sp + t.abs()
    dp_err = terms * E * Sp
    half = lambda m: (m[:, F:], m[:, :F]) if gate_first else (m[:, :F], m[:, F:])  # noqa: E731  (value, gate)
    v, t = half(p)
    ev, et = half(dp_err)
    a, da = act64(act, t)
    afp = ACT_ERR * (t.abs() + 1)
    out = {}
    eh = a.abs() * ev + (v.abs() + ev) * (1.2 * et + afp)
    out["y"] = (v * a, eh + u * (v * a).abs() + u * eh)
    if g is None:
        return out
    g64 = f64(g).reshape(-1, F)
    cut = 0.0 if dt == torch.float32 else 2.0 ** -15  # 24 bits: sign, 8 of exponent, 15 of the fraction
    ev, et = ev + cut * (v.abs() + ev), et + cut * (t.abs() + et)
    dv, dt_ = g64 * a, g64 * v * da
    edv = g64.abs() * (1.2 * et + afp + E * a.abs())
    edt = g64.abs() * ((da.abs() + afp) * ev + (v.abs() + ev) * (1.0 * et + afp) + 3 * E * (v * da).abs())
    join = lambda m, n: torch.cat((n, m) if gate_first else (m, n), 1)  # noqa: E731
    dp, edp = join(dv, dt_), join(edv, edt)
    edp = edp + u * (dp.abs() + edp) + sub_of(dt)  # dp is held in the activation type
    out["dbase"] = (dp, edp)
    many = 1 if dt != torch.float32 else 6
    W = w64.abs()
    wr = u if held_weight and dt != torch.float32 else 0.0
    S = dp.abs() @ W
    edx = (edp @ W) * (1 + wr) + (wr + (many * 2 * F + 16) * E) * S * 1.05
    out["dx"] = (dp @ w64, edx + u * ((dp @ w64).abs() + edx))
    M = x64.shape[0]
    S = dp.abs().t() @ x64.abs()
    edw = edp.t() @ x64.abs() + (many * M + 16) * E * S * 1.05
    out["dw"] = (dp.t() @ x64, edw + u * ((dp.t() @ x64).abs() + edw))
    eb = edp.sum(0) + (M + 4) * E * dp.abs().sum(0) * 1.05
    out["dbias"] = (dp.sum(0), eb + u * (dp.sum(0).abs() + eb))
    return out


GATED = [(1, 16, 8), (1, 1280, 640), (3, 33, 5), (16, 320, 128), (40, 200, 77), (64, 64, 64), (130, 136, 200), (257, 640, 333), (333, 201, 505), (1000, 320, 256)]


@pytest.mark.parametrize("int8", [False, True], ids=["plain", "int8"])
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,K,F", GATED)
def test_gated_forward_and_gradients(M, K, F, dt, int8):
    gen = torch.Generator().manual_seed(M + K + F)
    act = ("gelu", "gelu_tanh", "silu")[(M + F) % 3]
    gate_first = bool(K % 2) or M == 64
    lead = (2, M // 2) if M % 2 == 0 else (M,)
    x = rnd(gen, (*lead, K), dt)
    bias = rnd(gen, (2 * F,), dt, 0.2) if M % 5 else None
    base = rnd(gen, (*lead, 2 * F), dt, 0.3) if F % 3 else None
    p_of_q = sw = None
    if int8:
        w, sw = held(gen, 2 * F, K)
        w64 = f64(w) * f64(sw)[:, None]
        q, s = quantize64(x.reshape(-1, K))
        p_of_q = (q @ f64(w).t()) * s * f64(sw)
    else:
        w = rnd(gen, (2 * F, K), dt, 1 / math.sqrt(K))
        w64 = f64(w)
    g = rnd(gen, (*lead, F), dt, 1 / math.sqrt(F))
    leaf = lambda t: None if t is None else t.clone().requires_grad_(True)  # noqa: E731
    poison()
    leaves = {"dx": leaf(x), "dw": None if int8 else leaf(w), "dbias": leaf(bias), "dbase": leaf(base)}
    y = ops.gated_linear(leaves["dx"], w if int8 else leaves["dw"], leaves["dbias"], leaves["dbase"], act=act, gate_first=gate_first, weight_scale=sw)
    assert y.shape == (*lead, F) and y.dtype == dt
    names = [n for n, t in leaves.items() if t is not None]
    got = dict(zip(names, torch.autograd.grad(y, [leaves[n] for n in names], g)), y=y)
    want = gated_reference(x, w64, bias, base, act, gate_first, g, dt, int8, p_of_q)
    for n in ["y"] + names:
        if n != "y":
            assert got[n].shape == leaves[n].shape and got[n].dtype == leaves[n].dtype
        within(got[n], *want[n], n)
    with torch.no_grad():  # without the backward pass's operand: the same bits
        assert torch.equal(ops.gated_linear(x, w, bias, base, act=act, gate_first=gate_first, weight_scale=sw), y)


def test_gated_gradients_agree_with_differences():
    """the formula's derivative against central differences of the op itself (fp32: h = 2^-6 leaves h^2 |f'''| / 6 < 1e-4 and 2 e |f| / h)"""
    gen = torch.Generator().manual_seed(2)
    M, K, F = 4, 24, 12
    x, w = rnd(gen, (M, K), torch.float32), rnd(gen, (2 * F, K), torch.float32, 0.2)
    b, base, g = rnd(gen, (2 * F,), torch.float32, 0.2), rnd(gen, (M, 2 * F), torch.float32, 0.2), rnd(gen, (M, F), torch.float32)
    for act in ops.ACTIVATIONS:
        ts = [t.clone().requires_grad_(True) for t in (x, w, b, base)]
        grads = torch.autograd.grad(ops.gated_linear(*ts, act=act), ts, g)
        for i, t in enumerate((x, w, b, base)):
            d = rnd(gen, t.shape, torch.float32)
            d /= d.norm()
            h = 2.0 ** -6
            f = [(ops.gated_linear(*[s + (sign * h * d if j == i else 0) for j, s in enumerate((x, w, b, base))], act=act).double() * g.double()).sum() for sign in (1, -1)]
            num, ana = float(f[0] - f[1]) / (2 * h), float((grads[i].double() * d.double()).sum())
            size = float(grads[i].double().norm())
            assert abs(num - ana) <= 2e-3 * max(size, 1.0), (act, i, num, ana)


def test_gated_only_what_is_asked_for():
    gen = torch.Generator().manual_seed(12)
    x, w = rnd(gen, (70, 72), torch.bfloat16), rnd(gen, (48, 72), torch.bfloat16, 0.1)
    bias, base, g = rnd(gen, (48,), torch.bfloat16), rnd(gen, (70, 48), torch.bfloat16), rnd(gen, (70, 24), torch.bfloat16)
    full = [t.clone().requires_grad_(True) for t in (x, w, bias, base)]
    all_ = torch.autograd.grad(ops.gated_linear(*full), full, g)
    for i in range(4):
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, bias, base))]
        assert torch.equal(torch.autograd.grad(ops.gated_linear(*ts), ts[i], g)[0], all_[i])
    e = [t[:0].clone().requires_grad_(True) if i in (0, 3) else t.clone().requires_grad_(True) for i, t in enumerate((x, w, bias, base))]
    ge = torch.autograd.grad(ops.gated_linear(*e), e, g[:0])
    assert (ge[1] == 0).all() and (ge[2] == 0).all() and ge[0].shape == (0, 72) and ge[3].shape == (0, 48)


def test_gated_large_gates_and_non_finite_rows():
    """gates far from zero (act -> 0 or the identity, no NaN from inf * 0), and a row that is not finite stays alone"""
    for act in ops.ACTIVATIONS:
        for dt in DTYPES:
            base = torch.zeros(4, 16, dtype=dt, device=DEV)
            base[:, :8] = 2.0
            base[0, 8:], base[1, 8:], base[2, 8:], base[3, 8:] = 1e4, -1e4, 50.0, -50.0
            base.requires_grad_(True)
            x, w = torch.zeros(4, 8, dtype=dt, device=DEV), torch.zeros(16, 8, dtype=dt, device=DEV)
            y = ops.gated_linear(x, w, base=base, act=act)
            ref = act64(act, f64(base)[:, 8:])
            within(y, 2 * ref[0], ACT_ERR * 2 * ref[0].abs() + u_of(dt) * 2.01 * ref[0].abs() + 1e-18, act)
            d, = torch.autograd.grad(y, base, torch.ones_like(y))
            within(d[:, 8:], 2 * ref[1], 1e-4 * ref[1].abs() + u_of(dt) * 2.01 * ref[1].abs() + 1e-15, act)
            if dt != torch.float16:  # t^2 and t^3 beyond fp32: the derivative is 1 or 0
                far = torch.tensor([1e20, -1e20, 1e30, -1e30], dtype=dt, device=DEV).repeat(4, 2)
                far = torch.cat((torch.ones_like(far), far), 1).requires_grad_(True)
                d, = torch.autograd.grad(ops.gated_linear(x, w, base=far, act=act).float().sum(), far)
                assert torch.equal(d[:, 8:].float(), (far[:, 8:] > 0).float()), act
    gen = torch.Generator().manual_seed(1)
    x, w = rnd(gen, (20, 64), torch.bfloat16), rnd(gen, (64, 64), torch.bfloat16, 0.1)
    want = ops.gated_linear(x, w)
    x[3, 5] = float("nan")
    y = ops.gated_linear(x, w)
    rest = [m for m in range(20) if m != 3]
    assert torch.isnan(y[3]).all() and torch.equal(y[rest], want[rest])


# ---- how they are called -------------------------------------------------------------------------------------------------------------------
def test_results_repeat_bit_for_bit_on_any_stream():
    gen = torch.Generator().manual_seed(6)
    wq, sw = held(gen, 1024, 320)
    x, g = rnd(gen, (500, 320), torch.bfloat16), rnd(gen, (500, 512), torch.bfloat16)
    w = rnd(gen, (1024, 320), torch.bfloat16, 0.05)

    def step():
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        a = ops.gated_linear(xs, wq, weight_scale=sw)
        b = ops.gated_linear(xs, ws)
        return (a.detach(), b.detach(), *torch.autograd.grad([a, b], [xs, ws], [g, g]), ops.int8_linear(x, wq, sw))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_captured_step_replays():
    gen = torch.Generator().manual_seed(7)
    wq, sw = held(gen, 640, 320)
    w = rnd(gen, (512, 320), torch.float16, 0.05).requires_grad_(True)
    bias = rnd(gen, (512,), torch.float16, 0.1).requires_grad_(True)
    x = rnd(gen, (260, 320), torch.float16).requires_grad_(True)
    g1, g2 = rnd(gen, (260, 640), torch.float16), rnd(gen, (260, 256), torch.float16)

    def step():
        y1, y2 = ops.int8_linear(x, wq, sw), ops.gated_linear(x, w, bias, act="silu")
        return [y1.detach(), y2.detach(), *torch.autograd.grad([y1, y2], [x, w, bias], [g1, g2])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(rnd(gen, (260, 320), torch.float16))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_outputs_past_32_bit_offsets():
    M, K, N = 290_000, 64, 8192  # 4.75 GB of output
    gen = torch.Generator().manual_seed(10)
    wq, sw = held(gen, N, K)
    x = torch.randn(M, K, dtype=torch.bfloat16, device=DEV)
    y = ops.int8_linear(x, wq, sw)
    rows = torch.tensor([0, 131071, 262143, 262144, 280001, M - 1], device=DEV)
    want, err = linear_reference(x[rows], wq, sw, None, None)
    within(y[rows], want, err + u_of(torch.bfloat16) * (want.abs() + err), "y")
    del y
    w = rnd(gen, (2 * 4096, K), torch.bfloat16, 0.1)
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    h = ops.gated_linear(xl, wl, act="silu")
    g = torch.zeros_like(h)
    g[rows] = 1.0
    dx, dw = torch.autograd.grad(h, [xl, wl], g)
    want = gated_reference(x[rows], f64(w), None, None, "silu", False, g[rows], torch.bfloat16, False)
    within(h[rows], *want["y"], "h")
    within(dx[rows], *want["dx"], "dx")
    within(dw, *want["dw"], "dw")  # the other rows' gradient is zero


def test_many_rows():
    """more rows than a launch of a workgroup a row, or a grid's second dimension, would take"""
    M, K, F = (1 << 22) + 101, 16, 8
    gen = torch.Generator().manual_seed(21)
    x = torch.randn(M, K, dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([0, (1 << 22) - 1, 1 << 22, M - 1], device=DEV)
    q, s = ops.int8_quantize(x)
    q64, s64 = quantize64(x[rows])
    assert torch.equal(f64(q[rows]), q64) and torch.equal(f64(s[rows]), s64[:, 0])
    w = rnd(gen, (2 * F, K), torch.bfloat16, 0.25)
    xl, wl = x.requires_grad_(True), w.requires_grad_(True)
    h = ops.gated_linear(xl, wl, act="gelu_tanh")
    g = torch.zeros_like(h)
    g[rows] = 1.0
    dx, dw = torch.autograd.grad(h, [xl, wl], g)
    want = gated_reference(x[rows], f64(w), None, None, "gelu_tanh", False, g[rows], torch.bfloat16, False)
    within(h[rows], *want["y"], "h")
    within(dx[rows], *want["dx"], "dx")
    within(dw, *want["dw"], "dw")  # the other rows' gradient is zero


def test_autocast_and_other_types_of_bias():
    gen = torch.Generator().manual_seed(13)
    wq, sw = held(gen, 64, 48)
    x = rnd(gen, (9, 48), torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ops.int8_linear(x, wq, sw, rnd(gen, (64,), torch.float32), base=rnd(gen, (9, 64), torch.float32))
        h = ops.gated_linear(x, rnd(gen, (64, 48), torch.float32))
    assert y.dtype == h.dtype == torch.bfloat16
    b = rnd(gen, (64,), torch.float16)
    xb = x.to(torch.bfloat16)
    assert torch.equal(ops.int8_linear(xb, wq, sw, b), ops.int8_linear(xb, wq, sw, b.float()))


def test_refusals_on_the_device():
    gen = torch.Generator().manual_seed(14)
    wq, sw = held(gen, 64, 48)
    x = rnd(gen, (9, 48), torch.bfloat16)
    bad = [lambda: ops.int8_linear(x[:, :40], wq, sw), lambda: ops.int8_linear(x, wq.float(), sw), lambda: ops.int8_linear(x, wq, sw[:60]),
           lambda: ops.int8_linear(x, wq, sw.half()), lambda: ops.int8_linear(x, wq.cpu(), sw), lambda: ops.int8_linear(x, wq, sw.cpu()),
           lambda: ops.int8_linear(x.double(), wq, sw), lambda: ops.int8_linear(x, wq, sw, torch.zeros(63, device=DEV)),
           lambda: ops.int8_linear(x, wq, sw, base=torch.zeros(9, 1, device=DEV, dtype=x.dtype)),
           lambda: ops.int8_linear(x, wq, sw, torch.zeros(64, device=DEV, requires_grad=True)),
           lambda: ops.int8_matmul(wq, sw, wq[:, :32], sw), lambda: ops.int8_matmul(wq, sw[:3], wq, sw), lambda: ops.int8_matmul(wq, sw, wq, sw, dtype=torch.float64),
           lambda: ops.int8_quantize(x.double()), lambda: ops.int8_quantize(x[:, :0]), lambda: ops.int8_quantize(torch.tensor(1.0, device=DEV)),
           lambda: ops.gated_linear(x, wq), lambda: ops.gated_linear(x, torch.zeros(63, 48, device=DEV, dtype=x.dtype)),
           lambda: ops.gated_linear(x, torch.zeros(64, 48, device=DEV)), lambda: ops.gated_linear(x, wq, weight_scale=sw[:32]),
           lambda: ops.gated_linear(x, wq, base=torch.zeros(9, 32, device=DEV, dtype=x.dtype), weight_scale=sw), lambda: ops.gated_linear(x, wq, act="relu", weight_scale=sw)]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was accepted")
    xl = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(ops.int8_linear(xl, wq, sw).float().pow(2).sum(), xl, create_graph=True)


def test_calls_from_two_threads():
    import threading
    gen = torch.Generator().manual_seed(21)
    wq, sw = held(gen, 640, 320)
    xs = [rnd(gen, (300 + 41 * i, 320), torch.bfloat16) for i in range(2)]
    want = [ops.int8_linear(x, wq, sw) for x in xs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got[i].append(ops.int8_linear(xs[i], wq, sw))
        st.synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_traced_block_equals_the_eager_one():
    gen = torch.Generator().manual_seed(22)
    wq, sw = held(gen, 128, 64)
    w, b = rnd(gen, (96, 128), torch.bfloat16, 0.1), rnd(gen, (96,), torch.bfloat16)

    def block(x, w):
        h = torch.ops.lycoris_amd.int8_linear(x, wq, sw, None, None)
        return torch.ops.lycoris_amd.gated_linear(h, w, None, b, None, 2, True)

    x = rnd(gen, (5, 7, 64), torch.bfloat16)
    g = rnd(gen, (5, 7, 48), torch.bfloat16)
    outs = []
    for f in (block, torch.compile(block, backend="aot_eager", fullgraph=True)):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = f(xl, wl)
        outs.append([y.detach(), *torch.autograd.grad(y, [xl, wl], g)])
    for a, c in zip(*outs):
        assert torch.equal(a, c)


# ---- together: a transformer block whose frozen layers are held in 8 bits, under adapters ------------------------------------------------
class Block(torch.nn.Module):
    def __init__(self, c, f):
        super().__init__()
        from lycoris_amd import GatedLinear
        self.to_q, self.to_out = torch.nn.Linear(c, c, bias=False), torch.nn.Linear(f, c)
        self.ff = GatedLinear(torch.nn.Linear(c, 2 * f))

    def forward(self, x):
        h = x + self.to_q(x)
        return h + self.to_out(self.ff(h))


@pytest.mark.parametrize("algo", ["locon", "lokr"])
@pytest.mark.parametrize("dt,tol", [(torch.float32, 2e-3), (torch.bfloat16, 3e-2)], ids=["f32", "bf16"])
def test_training_step_of_adapters_on_an_int8_block(algo, dt, tol):
    """One step of adapters on Int8Linear layers and a GatedLinear block, against the same modules on the host in 64 bits.  Both sides
    quantise their own activations: an element whose value differs by r of itself changes its integer with probability 127 r, by a step of
    1/127 of the row's maximum (four times its rms, say).  fp32: r = 1e-6, so that one element in 1e4 moves by 3 % of the rms: 3e-4 norm-wise
    a layer, three layers.  bf16: 2^-9 and more (the activations are rounded): a fifth of the elements, 1.4 % a layer."""
    from lycoris_amd import LoConModule, LokrModule, NATIVE_ALGOS, quantize_frozen
    assert NATIVE_ALGOS["locon"] is LoConModule
    torch.manual_seed(3)
    c, f = 320, 640
    nets = [Block(c, f).requires_grad_(False) for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    x = torch.randn(2, 150, c).to(dt)
    g = (torch.randn(2, 150, c) / c).to(dt)
    results = []
    for net, dev, ct in ((nets[0], DEV, dt), (nets[1], "cpu", torch.float64)):
        names = quantize_frozen(net)  # the same integers on both sides
        assert sorted(names) == ["ff.proj", "to_out", "to_q"]
        net.to(dev)
        layers = [net.to_q, net.ff.proj, net.to_out]
        torch.manual_seed(4)
        cls, kw = (LoConModule, dict(lora_dim=8, alpha=4.0)) if algo == "locon" else (LokrModule, dict(lora_dim=100000, factor=8))
        mods = [cls(f"m{i}", l, **kw) for i, l in enumerate(layers)]
        with torch.no_grad():
            for m in mods:
                for p in m.parameters():
                    p.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())) * 0.1)
        for m in mods:
            m.to(dev)
            if ct == torch.float64:
                m.double()
            m.apply_to()
        for l in layers:
            l.bias = None if l.bias is None else torch.nn.Parameter(l.bias.to(ct), requires_grad=False)
            l.dtype = ct
        xl = x.to(dev).to(ct).requires_grad_(True)
        y = net(xl)
        assert net.ff._adapters() == [mods[1]]
        params = [p for m in mods for p in m.parameters()]
        for p in params:
            p.grad = torch.zeros_like(p)
        if dev == DEV:
            ops.fused_grad_accumulation(True, None)
        try:
            y.backward(g.to(dev).to(ct))
        finally:
            ops.fused_grad_accumulation(False, None)
        results.append([y.detach(), xl.grad] + [p.grad for p in params])
        assert all(q.grad is None for l in layers for q in l.parameters())
    for i, (a, b) in enumerate(zip(*results)):
        a, b = f64(a), f64(b)
        assert float((a - b).norm() / b.norm()) <= tol, i


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_one_tensor_in_two_places_broadcast_operands_and_recomputation(dt):
    from torch.utils.checkpoint import checkpoint
    gen = torch.Generator().manual_seed(31)
    wq, sw = held(gen, 96, 96)
    w = rnd(gen, (96, 96), dt, 0.1)
    x, g, g2 = rnd(gen, (50, 96), dt), rnd(gen, (50, 96), dt), rnd(gen, (50, 48), dt)

    def grads(f, leaves, grad):
        leaves = [t.clone().requires_grad_(True) for t in leaves]
        y = f(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, grad)]

    for f, grad in ((lambda a, b: ops.int8_linear(a, wq, sw, base=b), g), (lambda a, b: ops.gated_linear(a, w, base=b), g2),
                    (lambda a, b: ops.gated_linear(a, wq, base=b, weight_scale=sw, gate_first=True), g2)):
        y, da, db = grads(f, [x, x], grad)  # two leaves of the same values
        one, d = grads(lambda a: f(a, a), [x], grad)
        assert torch.equal(one, y) and torch.equal(d, da + db)
        again, dc = grads(lambda a: checkpoint(lambda t: f(t, t), a, use_reentrant=False), [x], grad)
        assert torch.equal(again, y) and torch.equal(dc, d)
        row = x[:1].clone()  # a base that every row shares
        full, _, dfull = grads(f, [x, row.expand(50, 96).contiguous()], grad)
        shared, _, drow = grads(lambda a, r: f(a, r.expand(50, 96)), [x, row], grad)
        assert torch.equal(shared, full)
        within(drow, f64(dfull).sum(0, keepdim=True), (u_of(dt) * 2 + 50 * E) * f64(dfull).abs().sum(0, keepdim=True) + 1e-30, "shared base")
    wl = w.clone().requires_grad_(True)  # one weight in two calls
    y = ops.gated_linear(x, wl) + ops.gated_linear(x, wl, act="silu")
    dw, = torch.autograd.grad(y, wl, g2)
    parts = [grads(lambda v: ops.gated_linear(x, v, act=act), [w], g2)[1] for act in ("gelu", "silu")]
    assert torch.equal(dw, parts[0] + parts[1])


def test_two_captured_graphs_replayed_side_by_side():
    gen = torch.Generator().manual_seed(32)
    wq, sw = held(gen, 640, 320)
    inputs = [rnd(gen, (n, 320), torch.bfloat16).requires_grad_(True) for n in (700, 90)]
    g = [rnd(gen, (t.shape[0], 320), torch.bfloat16) for t in inputs]

    def step(x, grad):
        y = ops.gated_linear(x, wq, weight_scale=sw)
        z = ops.int8_linear(y, wq[:320], sw[:320])
        return z.detach(), torch.autograd.grad(z, x, grad)[0]

    want = [[t.clone() for t in step(x, grad)] for x, grad in zip(inputs, g)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in inputs], [], []
    for x, grad, st in zip(inputs, g, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(x, grad)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(step(x, grad))
        graphs.append(graph)
    for _ in range(4):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
            for a in got:
                a.zero_()
        step(inputs[0], g[0])  # eager work between the replays


def test_a_capture_beside_an_eager_graph_of_the_same_leaf_is_refused():
    """(its backward pass would end the process when the capture ends: refused by the forward call)"""
    gen = torch.Generator().manual_seed(33)
    wq, sw = held(gen, 64, 64)
    w = rnd(gen, (64, 64), torch.bfloat16, 0.1).requires_grad_(True)
    x = rnd(gen, (40, 64), torch.bfloat16).requires_grad_(True)
    alive = [ops.int8_linear(x, wq, sw), ops.gated_linear(x.detach(), w)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        plain = x.detach() * 2
        frozen = ops.int8_linear(x.detach(), wq, sw)  # nothing to differentiate: no matter
        for call in (lambda: ops.int8_linear(x, wq, sw), lambda: ops.gated_linear(x, wq, weight_scale=sw), lambda: ops.gated_linear(x.detach(), w),
                     lambda: ops.int8_linear(x.detach(), wq, sw, base=x)):
            with pytest.raises(RuntimeError, match="eager autograd graph"):
                call()
    want = alive[0].detach().clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(frozen, want) and torch.equal(plain, x.detach() * 2)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):  # nothing lives: captured
        y = ops.int8_linear(x, wq, sw)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        y = y.detach()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
