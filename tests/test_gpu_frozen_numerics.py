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
