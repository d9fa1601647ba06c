"""GPU: what ops.gated_linear keeps in how many bits, against the formulas in 64 bits.  With x = 0 the projection is its bias and base alone, so
that every value of it is known exactly.  Bounds: u = eps / 2 of a type is one rounding to it, e = 2^-24 one rounding to fp32; the activation and its
derivative are off by 2^-17 (|t| + 1) at most, in fp32."""
import math

import pytest
import torch

from lycoris_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
ACT_ERR = 2.0 ** -17
HALVES = [torch.bfloat16, torch.float16]
IDS = ["bf16", "f16"]


def silu64(t):
    s = torch.sigmoid(t)
    return t * s, s * (1 + t * (1 - s))


@pytest.mark.parametrize("int8", [False, True], ids=["plain", "int8"])
@pytest.mark.parametrize("dt", HALVES, ids=IDS)
@pytest.mark.parametrize("M,F", [(1, 8), (70, 33), (300, 256), (1200, 64)])
def test_the_gradient_of_an_fp32_bias_keeps_32_bits(M, F, dt, int8):
    """sum_m dp in fp32: a term is off by the activation's error and three roundings, the sum of M by M e of the magnitudes; nothing is rounded to
    the activation type (u of the sum would be 2^-9 or 2^-12), and a sum beyond fp16 stays finite"""
    gen = torch.Generator().manual_seed(M + F)
    x, w = torch.zeros(M, 16, dtype=dt, device=DEV), torch.zeros(2 * F, 16, dtype=dt, device=DEV)
    sw = None
    if int8:
        w, sw = ops.int8_quantize(torch.randn(2 * F, 16, generator=gen).to(DEV))
    bias = torch.zeros(2 * F, device=DEV, requires_grad=True)
    base = torch.randn(M, 2 * F, generator=gen).to(dt).to(DEV)
    g = (torch.rand(M, F, generator=gen) * 600 + 100).to(dt).to(DEV)  # one sign: the sums grow with M
    h = ops.gated_linear(x, w, bias, base, act="silu", weight_scale=sw)
    got, = torch.autograd.grad(h, bias, g)
    assert got.dtype == torch.float32
    v, t = base.double().cpu().split(F, 1)
    g64 = g.double().cpu()
    a, da = silu64(t)
    want = torch.cat(((g64 * a).sum(0), (g64 * v * da).sum(0)))
    afp = ACT_ERR * (t.abs() + 1)
    mag = torch.cat(((g64 * a).abs().sum(0), (g64 * v * da).abs().sum(0)))
    bound = torch.cat(((g64 * afp).sum(0), (g64 * v.abs() * afp).sum(0))) + (M + 8) * E * 1.05 * mag
    over = (got.double().cpu() - want).abs() - bound
    assert (over <= 0).all(), float(over.max())
    if M == 1200:  # the mean of silu over a standard normal is 0.207: 0.207 * 400 * 1200 = 99e3
        assert float(want.abs().max()) > 65504


def kept(pre, n):
    """the fp32 bits of p as the backward pass reads them: a plane of the upper 16 bits, one of the next 8"""
    raw = pre.cpu()
    hi, lo = raw[:2 * n].view(torch.int16).long() & 0xffff, raw[2 * n:].long()
    return (hi << 16) | (lo << 8)


@pytest.mark.parametrize("int8", [False, True], ids=["plain", "int8"])
@pytest.mark.parametrize("dt", HALVES, ids=IDS)
@pytest.mark.parametrize("M,F", [(1, 8), (20, 33), (40, 40), (300, 77), (300, 640), (4100, 2560)])
def test_p_is_kept_in_24_bits_to_the_nearest(M, F, dt, int8):
    """half a step of 16 significant bits at most, 2^-16 of the value, and no more below it than above; infinities and NaNs stay what they are"""
    gen = torch.Generator().manual_seed(M + F)
    x, w = torch.zeros(M, 16, dtype=dt, device=DEV), torch.zeros(2 * F, 16, dtype=dt, device=DEV)
    sw = None
    if int8:
        w, sw = ops.int8_quantize(torch.randn(2 * F, 16, generator=gen).to(DEV))
    bits = torch.randint(-2 ** 31, 2 ** 31, (2 * F,), generator=gen, dtype=torch.int64)
    bits[:12] = torch.tensor([0x7f800000, 0xff800000, 0x7fc00000, 0x7fffffff, 0xffffffff, 0x7f800001, 0, 0x80000000, 0x3f800080, 0x3f80007f, 0xbf8000ff, 0x3fffffff])
    bits = bits.remainder(2 ** 32)
    bias = bits.sub((bits >= 2 ** 31).long() * 2 ** 32).to(torch.int32).view(torch.float32)
    h, pre = torch.ops.lycoris_amd._gated_linear_forward(x, w, sw, bias.to(DEV), None, 2, False)
    got = kept(pre, M * 2 * F).view(M, 2 * F)
    assert (got == got[0]).all()  # every row alike, whichever lane and path wrote it
    value = got[0].sub((got[0] >= 2 ** 31).long() * 2 ** 32).to(torch.int32).view(torch.float32)
    nan = bias.isnan()
    assert torch.equal(value.isnan(), nan)
    tiny = bias.abs() < 2.0 ** -126  # below: a product with the scale may flush them
    big = bias.abs() >= 2.0 ** 128 - 2.0 ** 111  # rounds to the power above: infinity
    rest = ~(nan | tiny | big)
    assert torch.equal(value[big], torch.copysign(torch.full_like(value[big], math.inf), bias[big]))
    assert (value[tiny].abs() <= 2.0 ** -126).all()
    b64, v64 = bias[rest].double(), value[rest].double()
    step = 2.0 ** (torch.floor(torch.log2(b64.abs())) - 15)
    off = (v64 - b64) / step
    assert float(off.abs().max()) <= 0.5
    if F >= 640:  # uniform on a step of 1 around 0: standard deviation 0.289 / sqrt(n); truncation would give a mean of -0.5 of the magnitude
        toward = (off * torch.sign(b64)).mean()
        assert abs(float(toward)) < 6 * 0.289 / math.sqrt(off.numel())


def spread(gen, shape, top):
    """fp32 values of all magnitudes in (top / 4, top], every bit of the fraction in use"""
    return ((torch.rand(*shape, generator=gen).double() * 0.75 + 0.25) * top * torch.sign(torch.randn(*shape, generator=gen).double())).float()


@pytest.mark.parametrize("top", [float(torch.finfo(torch.float32).max), 2.0 ** -100, 2.0 ** -112, 2.0 ** -120], ids=["max", "2^-100", "2^-112", "2^-120"])
@pytest.mark.parametrize("M,K,N", [(3, 9, 6), (70, 64, 40), (300, 128, 256)])
def test_32_bit_products_at_both_ends_of_the_range(M, K, N, top):
    """three bf16 planes hold 24 bits where all three are normal numbers.  A term is then off by 3 e of it, the sum by e of the magnitudes for each
    of its 3 n or 6 n products.  A plane below 2^-126 may be lost: 2^-125 of the other factor at most; so may a sum of one matrix instruction
    (32 terms) below 2^-126"""
    gen = torch.Generator().manual_seed(M)
    flush = 2.0 ** -125
    # dx of an 8-bit layer: g is staged; small scales keep the other columns finite
    q = torch.randint(-127, 128, (N, K), generator=gen, dtype=torch.int8)
    q[:, 1], q[0, :] = 0, 0
    q[0, 1] = 1  # column 1 is g's column 0 itself
    s = torch.full((N,), 2.0 ** -8 / max(N, 64))
    s[0] = 1.0
    g = spread(gen, (M, N), top)
    g[0, 0] = top
    x = torch.zeros(M, K, device=DEV, requires_grad=True)
    y = ops.int8_linear(x, q.to(DEV), s.to(DEV))
    dx, = torch.autograd.grad(y, x, g.to(DEV))
    w64 = q.double() * s.double()[:, None]
    want, mag = g.double() @ w64, g.double().abs() @ w64.abs()
    off = (dx.double().cpu() - want).abs()
    assert torch.isfinite(dx).all() and (off <= (3 * N + 8) * E * mag + E * want.abs() + flush * q.double().abs().sum(0) + (3 * N / 32 + 1) * 2.0 ** -126).all(), float((off / mag.clamp_min(1e-300)).max())
    # the gated forward: x is staged against a weight of 2^-10 / K; the gate half is the bias alone, act(1)
    F = N // 2
    w = spread(gen, (2 * F, K), 2.0 ** -10 / K)
    w[F:] = 0
    bias = torch.cat((torch.zeros(F), torch.ones(F)))
    a = spread(gen, (M, K), top)
    a[0, 0] = top
    h = ops.gated_linear(a.to(DEV), w.to(DEV), bias.to(DEV), act="silu")
    one = float(silu64(torch.ones((), dtype=torch.float64))[0])
    p, mag = a.double() @ w[:F].double().t(), a.double().abs() @ w[:F].double().abs().t()
    off = (h.double().cpu() - p * one).abs()
    assert torch.isfinite(h).all()
    assert (off <= (6 * K + 16) * E * mag + (2 * ACT_ERR + E) * p.abs() + 2 * flush * w[:F].double().abs().sum(1) + (6 * K / 32 + 1) * 2.0 ** -126).all(), float((off / mag.clamp_min(1e-300)).max())


def held(gen, N, K):
    w = torch.randn(N, K, generator=gen) / math.sqrt(K) * torch.exp(0.3 * torch.randn(N, 1, generator=gen))
    return ops.int8_quantize(w.to(DEV))


# terms of dx = (g sw) wq: in fp16 with a power of two a row, one rounding (eps / 2 = 2^-11: 11 significant bits) beside bf16 gradients; two planes (2^-22) beside fp16 ones.  Below 2^-14
# of what fp16 holds the step is fixed: 2^-39 of the row's largest (half a step).  Sums: n e of the magnitudes.
TERM = {torch.bfloat16: torch.finfo(torch.float16).eps / 2, torch.float16: 2.0 ** -22}


def check_dx(dx, g, wq, sw, dt):
    w64 = wq.double().cpu() * sw.double().cpu()[:, None]
    g64 = g.double().cpu()
    N = g64.shape[-1]
    want, mag = g64 @ w64, g64.abs() @ w64.abs()
    top = (g64 * sw.double().cpu()).abs().amax(-1, keepdim=True)
    planes = 1 if dt == torch.bfloat16 else 2
    bound = (TERM[dt] + 2 * E + (planes * N + 4) * E) * mag * 1.01 + 2.0 ** -39 * top * wq.double().cpu().abs().sum(0)
    u, f = torch.finfo(dt).eps / 2, torch.finfo(dt)
    bound = bound + u * (want.abs() + bound) + f.smallest_normal * f.eps / 2
    over = (dx.double().cpu() - want).abs() - bound
    assert torch.isfinite(dx).all() and (over <= 0).all(), float(over.max())
    return float((dx.double().cpu() - want).norm() / want.norm()), float((want.to(dt).double() - want).norm() / want.norm())


@pytest.mark.parametrize("dt", HALVES, ids=IDS)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 640, 1280), (5, 200, 17), (33, 64, 600), (130, 136, 1100), (300, 77, 1600), (40, 96, 3000), (257, 320, 5000), (64, 80, 8000),
                                   (20, 64, 8200), (2100, 1284, 1032)])
def test_dx_over_an_8_bit_weight_is_rounded_once(M, K, N, dt):
    """the operands keep more bits than the gradient's type: the error of dx is that of its own rounding"""
    gen = torch.Generator().manual_seed(M + K + N)
    wq, sw = held(gen, N, K)
    g = (torch.randn(M, N, generator=gen) / math.sqrt(N)).to(dt).to(DEV)
    x = torch.zeros(M, K, dtype=dt, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(ops.int8_linear(x, wq, sw), x, g)
    here, once = check_dx(dx, g, wq, sw, dt)
    if M * K > 10000:
        assert here < 1.03 * once, (here, once)


@pytest.mark.parametrize("dt", HALVES, ids=IDS)
def test_dx_of_rows_of_every_magnitude(dt):
    """rows as small as the type has them and as large, rows of zeros, one entry that outweighs the others by all that fp16 can hold and more"""
    gen = torch.Generator().manual_seed(31)
    M, K, N = 48, 72, 200
    wq, sw = held(gen, N, K)
    wq = wq.clone()
    wq[7, :40] = 0
    sw[7] = 1.0
    g = torch.randn(M, N, generator=gen)
    small = 2.0 ** -30 if dt == torch.bfloat16 else 2.0 ** -12
    g[:16] *= 2.0 ** torch.linspace(-20 if dt == torch.float16 else -130, 8 if dt == torch.float16 else 100, 16)[:, None]
    g[16:32] *= small * 2.0 ** -torch.arange(16.0)[:, None]
    g[16:32, 7] = 1.0  # columns below 40 see the small entries alone
    g[32] = 0
    g = g.to(dt).to(DEV)
    x = torch.zeros(M, K, dtype=dt, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(ops.int8_linear(x, wq, sw), x, g)
    check_dx(dx, g, wq, sw, dt)
    assert (dx[32] == 0).all()
    bad = g.clone()
    bad[40, 3], bad[41, 199] = float("nan"), float("inf")
    x2 = x.detach().clone().requires_grad_(True)
    d2, = torch.autograd.grad(ops.int8_linear(x2, wq, sw), x2, bad)
    rest = [m for m in range(M) if m not in (40, 41)]
    assert torch.equal(d2[rest], dx[rest]) and torch.isnan(d2[40]).all() and not torch.isfinite(d2[41]).any()


def gated64(x, w64, wmag, bias, base, act_grad, g, dt, c, p=None):
    """dp in 64 bits, and what an element of it may be off by before it is an operand: p in 24 bits, the activation, the sums of p"""
    K, F = x.shape[-1], w64.shape[0] // 2
    x64, g64 = x.double().cpu(), g.double().cpu()
    Sp = x64.abs() @ wmag.t()
    p = x64 @ w64.t() if p is None else p
    for t in (bias, base):
        if t is not None:
            p, Sp = p + t.double().cpu(), Sp + t.double().cpu().abs()
    ep = 2.0 ** -16 * p.abs() + (K + 8) * E * Sp
    v, t = p.split(F, 1)
    ev, et = ep.split(F, 1)
    a, da = act_grad(t)
    afp = ACT_ERR * (t.abs() + 1)
    dv, d = g64 * a, g64 * v * da
    edv = g64.abs() * (1.2 * et + afp + E * a.abs())
    ed = g64.abs() * ((da.abs() + afp) * ev + (v.abs() + ev) * (et + afp) + 3 * E * (v * da).abs())
    return torch.cat((dv, d), 1), torch.cat((edv, ed), 1)


def check_gated(got, x, w64, dp, edp, c, dt, rows=None):
    """dx and dw against dp in 64 bits: dp takes one rounding as an operand (TERM of it; c: an 8-bit weight's scales), 2^-39 of its row's largest at least;
    the other operands are exact down to 2^-39 of their largest"""
    u, f = torch.finfo(dt).eps / 2, torch.finfo(dt)
    planes = 1 if dt == torch.bfloat16 else 2
    x64, N, M = x.double().cpu(), dp.shape[1], dp.shape[0]
    top = (dp * c).abs().amax(1, keepdim=True)
    step = 2.0 ** -39
    e = edp + (TERM[dt] + 2 * E) * (dp.abs() + edp) + step * top / c
    stats = {}
    wmax = w64.abs().max()
    want, mag = dp @ w64, dp.abs() @ w64.abs()
    bound = {"dx": e @ w64.abs() * 1.01 + (planes * N + 4) * E * mag * 1.01 + step * wmax * dp.abs().sum(1, keepdim=True)}
    wants = {"dx": want}
    if "dw" in got:
        wants["dw"], mag = dp.t() @ x64, dp.abs().t() @ x64.abs()
        lost = step * 2 * top.max() * x64.abs().max() * (dp.abs() / top.clamp_min(1e-300)).sum(0)[:, None]
        bound["dw"] = e.t() @ x64.abs() * 1.01 + (planes * M + 4) * E * mag * 1.01 + lost
    for n, want in wants.items():
        b = bound[n] + u * (want.abs() + bound[n]) + f.smallest_normal * f.eps / 2
        off = (got[n].double().cpu() - want).abs()
        assert torch.isfinite(got[n]).all() and (off <= b).all(), (n, float((off - b).max()), float((off / b).max()))
        stats[n] = float(off.norm() / want.norm()), float((want.to(dt).double() - want).norm() / want.norm())
    return stats


@pytest.mark.parametrize("int8", [False, True], ids=["plain", "int8"])
@pytest.mark.parametrize("dt", HALVES, ids=IDS)
@pytest.mark.parametrize("M,K,F", [(1, 16, 8), (3, 33, 5), (70, 64, 200), (300, 136, 512), (257, 72, 513), (130, 320, 1280), (64, 40, 2560), (50, 24, 8192), (33, 17, 8201), (9, 24, 16384),
                                   (7, 16, 16392), (5, 9, 20003), (2100, 640, 264)])
def test_gated_gradients_are_rounded_once(M, K, F, dt, int8):
    gen = torch.Generator().manual_seed(M + K + F)
    x = torch.randn(M, K, generator=gen).to(dt).to(DEV)
    bias = (0.2 * torch.randn(2 * F, generator=gen)).to(dt).to(DEV)
    g = (torch.randn(M, F, generator=gen) / math.sqrt(F)).to(dt).to(DEV)
    sw, c, p = None, 1.0, None
    if int8:
        w, sw = held(gen, 2 * F, K)
        c = sw.double().cpu()
        w64 = w.double().cpu() * c[:, None]
        q, s = ops.int8_quantize(x)
        p = (q.double().cpu() @ w.double().cpu().t()) * s.double().cpu()[:, None] * c
    else:
        w = (torch.randn(2 * F, K, generator=gen) / math.sqrt(K)).to(dt).to(DEV)
        w64 = w.double().cpu()
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(not int8), bias.clone().requires_grad_(True)]
    h = ops.gated_linear(*leaves, act="silu", weight_scale=sw)
    names = ["dx", "dbias"] if int8 else ["dx", "dw", "dbias"]
    got = dict(zip(names, torch.autograd.grad(h, [t for t in leaves if t.requires_grad], g)))
    dp, edp = gated64(x, w64, w64.abs(), bias, None, silu64, g, dt, c, p)
    stats = check_gated(got, x, w64, dp, edp, c, dt)
    if M * K > 5000 and M > 100:
        assert all(here < 1.03 * once for here, once in stats.values()), stats
    u = torch.finfo(dt).eps / 2
    eb = edp.sum(0) + (M + 8) * E * dp.abs().sum(0)
    assert ((got["dbias"].double().cpu() - dp.sum(0)).abs() <= eb + u * (dp.sum(0).abs() + eb) + 2.0 ** -25).all()
    for which in range(2 - int8):  # each gradient by itself: the same bits
        one = [t.detach().clone().requires_grad_(i == which) for i, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(ops.gated_linear(*one, act="silu", weight_scale=sw), one[which], g)[0], got[names[which]])


@pytest.mark.parametrize("F", [40, 700, 17000], ids=["wave", "workgroup", "twice"])
@pytest.mark.parametrize("dt", HALVES, ids=IDS)
def test_gated_gradients_of_rows_of_every_magnitude(dt, F):
    """gradients from the type's smallest to large ones, rows and weight rows of zeros, rows that are not finite"""
    gen = torch.Generator().manual_seed(17)
    M, K = 64, 24
    x, w = torch.randn(M, K, generator=gen).to(dt), (torch.randn(2 * F, K, generator=gen) / math.sqrt(K)).to(dt)
    w[3], w[F + 5] = 0, 0  # dw of a zero row is not zero
    g = torch.randn(M, F, generator=gen)
    lo, hi = (-14, 4) if dt == torch.float16 else (-100, 60)
    g *= 2.0 ** torch.linspace(lo, hi, M)[torch.randperm(M, generator=gen)][:, None]
    g[11] = 0
    x, w, g = x.to(DEV), w.to(DEV), g.to(dt).to(DEV)

    def grads(x, g):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        return dict(zip(("dx", "dw"), torch.autograd.grad(ops.gated_linear(xl, wl, act="silu"), [xl, wl], g)))

    got = grads(x, g)
    dp, edp = gated64(x, w.double().cpu(), w.double().cpu().abs(), None, None, silu64, g, dt, 1.0)
    check_gated(got, x, w.double().cpu(), dp, edp, 1.0, dt)
    assert (got["dx"][11] == 0).all()
    bad = g.clone()
    bad[20, 7], bad[21, 0] = float("nan"), float("inf")
    d = grads(x, bad)
    rest = [m for m in range(M) if m not in (20, 21)]
    assert torch.equal(d["dx"][rest], got["dx"][rest]) and torch.isnan(d["dx"][20]).all() and not torch.isfinite(d["dx"][21]).any()
    clean = [o for o in range(2 * F) if o not in (7, F + 7, 0, F)]  # the other rows of dw see the finite entries alone
    assert torch.isfinite(d["dw"][clean]).all() and ((d["dw"][clean].double() - got["dw"][clean].double()).norm() <= 2.0 ** -6 * got["dw"][clean].double().norm())
    zero = torch.zeros_like(g)
    assert all((t == 0).all() for t in grads(x, zero).values())
