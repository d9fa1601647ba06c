"""Cases for the operators of a frozen layer held in 8 bits and of the gated projection of a feed-forward block: what is
measured, on which inputs, and what the answers are.

Operators (``lycoris_amd.ops``):

``int8_quantize(x)``          rows to 8-bit integers: scale = max|x| / 127 of the row, q = round-half-even(127 x / max|x|)
``int8_matmul(aq, sa, bq, sb, bias, dtype)``   (sa[m] sb[n]) sum_k aq[m, k] bq[n, k] + bias[n]
``int8_linear(x, wq, sw, bias, base)``         the same with x quantised inside, plus `base`; backward: dx = g (sw wq)
``gated_linear(x, w, bias, base, act, gate_first, weight_scale)``   p = x w^T + bias + base [.., 2 F]; value * act(gate) of
                              its two halves, in one kernel; w in 16 / 32 bits (trainable) or in 8 bits with weight_scale
                              (x is then quantised inside); backward to x, base, and to a trainable w and bias
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # activations of a self-attention block of the SDXL layer table, four images of 4096 tokens
        dict(name="quantize_tokens", op="quantize", M=16384, K=640, dtype="bf16"),
        # rows of no particular length, in 32 bits (a weight that is laid out, five prompts of 77 tokens)
        dict(name="quantize_ragged_fp32", op="quantize", M=385, K=1001, dtype="fp32"),
        # the time embedding of one image: one row, latency counts
        dict(name="int8_one_row", op="linear", M=1, K=1280, N=1280, dtype="bf16", bias=True, base=False, train=False),
        # a batch of single tokens through a large square layer: the weight is what is read
        dict(name="int8_sixteen_rows", op="linear", M=16, K=4096, N=4096, dtype="fp16", bias=False, base=False, train=False),
        # text context (four prompts of 77 tokens) into a 640-channel cross-attention
        dict(name="int8_text", op="linear", M=308, K=2048, N=640, dtype="fp16", bias=True, base=True, train=False),
        # a value projection on activations that the query projection has quantised already
        dict(name="int8_shared_input", op="matmul", M=4096, K=1280, N=1280, dtype="bf16", bias=True),
        # one attention projection in a training step of its adapter (`base` is the adapter's output)
        dict(name="int8_train", op="linear", M=4096, K=1280, N=1280, dtype="bf16", bias=True, base=True, train=True),
        # the second projection of a feed-forward block at a large batch, training
        dict(name="int8_train_large", op="linear", M=16384, K=5120, N=1280, dtype="bf16", bias=True, base=True, train=True),
        # a single token through a gated block in 8 bits
        dict(name="gated_int8_one_row", op="gated", M=1, I=1280, F=5120, dtype="bf16", act="silu", gate_first=True, int8=True,
             bias=False, base=False, train=False),
        # the 640-channel gated block with a trainable 16-bit weight, two images of 4096 tokens
        dict(name="gated_train", op="gated", M=8192, I=640, F=2560, dtype="bf16", act="gelu", gate_first=False, int8=False,
             bias=True, base=False, train=True),
        # the 1280-channel gated block frozen in 8 bits under an adapter, training
        dict(name="gated_int8_train", op="gated", M=4096, I=1280, F=5120, dtype="bf16", act="gelu", gate_first=False, int8=True,
             bias=True, base=True, train=True),
        # odd sizes in 32 bits, training
        dict(name="gated_ragged_fp32", op="gated", M=333, I=201, F=505, dtype="fp32", act="gelu_tanh", gate_first=True, int8=False,
             bias=True, base=True, train=True),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm; odd sizes and multiples of 64 both."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if n > 128 and rng.random() < 0.6:
        n = n // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "linear", "linear", "gated", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = dict(op=op, M=_spread(rng, 1, 16384), dtype=dtype)
    if op == "quantize":
        case.update(K=_spread(rng, 16, 8192))
    elif op == "matmul":
        case.update(K=_spread(rng, 16, 8192), N=_spread(rng, 16, 8192), bias=rng.random() < 0.5)
    elif op == "linear":
        train = rng.random() < 0.5
        case.update(K=_spread(rng, 16, 8192), N=_spread(rng, 16, 8192), bias=rng.random() < 0.5, base=rng.random() < 0.5, train=train)
    else:
        case.update(I=_spread(rng, 16, 4096), F=_spread(rng, 16, 8192), act=rng.choice(["gelu", "gelu_tanh", "silu"]),
                    gate_first=rng.random() < 0.5, int8=rng.random() < 0.5, bias=rng.random() < 0.5, base=rng.random() < 0.5,
                    train=rng.random() < 0.5)
    top = [work(c) for c in listed()]
    flops = max(t["flops"] for t in top) / (4 if dtype == "fp32" else 1)
    while case["M"] > 1 and (work(case)["flops"] > flops or work(case)["bytes"] > max(t["bytes"] for t in top)):
        case["M"] //= 2
    return case


def _rows(gen, M, K, dtype):
    """Activations behind a normalisation: unit rows, a few channels of larger values."""
    x = torch.randn(M, K, generator=gen, device="cuda")
    x *= 1.0 + 5.0 * (torch.rand(K, generator=gen, device="cuda") < 0.01)
    return x.to(dtype)


def _weight(gen, N, K):
    w = torch.randn(N, K, generator=gen, device="cuda") / math.sqrt(K)
    return w * torch.exp(0.3 * torch.randn(N, 1, generator=gen, device="cuda"))


def _held(w):
    """A weight as a program keeps it in 8 bits: rows at a pitch that is a multiple of 128 bytes, one scale a row."""
    amax = w.abs().amax(1, keepdim=True).double()
    N, K = w.shape
    held = torch.zeros(N, (K + 127) // 128 * 128, dtype=torch.int8, device=w.device)[:, :K]
    held.copy_(torch.round(127.0 * w.double() / amax).to(torch.int8))
    return held, (amax[:, 0] / 127.0).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = dict(case)
    M = case["M"]
    if case["op"] == "quantize":
        s["x"] = _rows(gen, M, case["K"], dt)
        return s
    K, N = (case["I"], 2 * case["F"]) if case["op"] == "gated" else (case["K"], case["N"])
    x = _rows(gen, M, K, dt)
    w = _weight(gen, N, K)
    s["bias"] = (0.1 * torch.randn(N, generator=gen, device="cuda")).to(dt) if case["bias"] else None
    if case["op"] == "matmul":
        (s["aq"], s["sa"]), (s["wq"], s["sw"]) = _held(x.float()), _held(w)
        return s
    s["x"] = x
    s["base"] = (0.3 * torch.randn(M, N, generator=gen, device="cuda")).to(dt) if case["base"] else None
    if case["op"] == "linear" or case["int8"]:
        s["wq"], s["sw"] = _held(w)
    else:
        s["w"] = w.to(dt)
    out = case["F"] if case["op"] == "gated" else N
    s["g"] = (torch.randn(M, out, generator=gen, device="cuda") / math.sqrt(out)).to(dt) if case["train"] else None
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _quantize(x):
    """Rows to 8-bit integers.  The quotient is formed in 64 bits: the values next to a half have to fall on their own side."""
    amax = x.abs().amax(-1, keepdim=True).double()
    q = torch.round(127.0 * x.double() / torch.where(amax > 0, amax, 1.0))
    return q.float(), (amax / 127.0).float()


def _act(name, t):
    """act(t) and its derivative"""
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-t))
        return t * s, s * (1.0 + t * (1.0 - s))
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(t * math.sqrt(0.5)))
        return t * cdf, cdf + t * torch.exp(-0.5 * t * t) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (t + 0.044715 * t * t * t))
    return 0.5 * t * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * t * (1.0 - th * th) * c * (1.0 + 3.0 * 0.044715 * t * t)


def _add(p, bias, base):
    if bias is not None:
        p = p + bias.float()
    return p if base is None else p + base.float()


def _plain(s):
    dt = _DT[s["dtype"]]
    if s["op"] == "quantize":
        q, scale = _quantize(s["x"])
        return {"values": q * scale, "scale": scale[:, 0]}
    if s["op"] == "matmul":
        p = (s["aq"].float() @ s["wq"].float().t()) * s["sa"][:, None] * s["sw"]
        return {"y": _add(p, s["bias"], None).to(dt)}
    held = "wq" in s
    if held:
        q, scale = _quantize(s["x"])
        p = (q @ s["wq"].float().t()) * scale * s["sw"]
    else:
        p = s["x"].float() @ s["w"].float().t()
    p = _add(p, s["bias"], s["base"])
    if s["op"] == "linear":
        out = {"y": p.to(dt)}
        dp = s["g"].float() if s["train"] else None
    else:
        F = s["F"]
        value, gate = (p[:, F:], p[:, :F]) if s["gate_first"] else (p[:, :F], p[:, F:])
        a, da = _act(s["act"], gate)
        out = {"y": (value * a).to(dt)}
        if s["train"]:
            g = s["g"].float()
            dv, dg = g * a, g * value * da
            dp = torch.cat((dg, dv) if s["gate_first"] else (dv, dg), 1)
    if s["train"]:
        w = s["wq"].float() * s["sw"][:, None] if held else s["w"].float()
        out["dx"] = (dp @ w).to(dt)
        if s["op"] == "gated" and s["base"] is not None:
            out["dbase"] = dp.to(dt)
        if not held:
            out["dw"] = (dp.t() @ s["x"].float()).to(dt)
            if s["bias"] is not None:
                out["dbias"] = dp.sum(0).to(dt)
    return out


# ---- the framework's operators -----------------------------------------------------------------------------------------
def _own(s):
    from lycoris_amd import ops
    if s["op"] == "quantize":
        q, scale = ops.int8_quantize(s["x"])
        return {"values": q.float() * scale[:, None], "scale": scale}
    if s["op"] == "matmul":
        return {"y": ops.int8_matmul(s["aq"], s["sa"], s["wq"], s["sw"], s["bias"], dtype=_DT[s["dtype"]])}
    held, train = "wq" in s, s["train"]
    x, base, bias = s["x"], s["base"], s["bias"]
    leaf = lambda t: t.detach().requires_grad_(True)  # noqa: E731
    wanted = {}
    if train:
        wanted["dx"] = x = leaf(x)
        if s["op"] == "gated" and base is not None:
            wanted["dbase"] = base = leaf(base)
    if s["op"] == "linear":
        y = ops.int8_linear(x, s["wq"], s["sw"], bias, base)
    else:
        w = s["wq"] if held else s["w"]
        if train and not held:
            wanted["dw"] = w = leaf(w)
            if bias is not None:
                wanted["dbias"] = bias = leaf(bias)
        y = ops.gated_linear(x, w, bias, base, act=s["act"], gate_first=s["gate_first"], weight_scale=s["sw"] if held else None)
    out = {"y": y.detach()}
    if train:
        out.update(zip(wanted, torch.autograd.grad(y, list(wanted.values()), s["g"])))
    return out


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    """Each input read once, each output written once; the products of the operator's formulas."""
    M, b = case["M"], _BYTES[case["dtype"]]
    if case["op"] == "quantize":
        return {"bytes": M * case["K"] * (b + 1) + 4 * M, "flops": 2 * M * case["K"]}
    if case["op"] == "matmul":
        K, N = case["K"], case["N"]
        return {"bytes": (M + N) * K + 4 * (M + N) + M * N * b + (N * b if case["bias"] else 0), "flops": 2 * M * N * K}
    gated = case["op"] == "gated"
    K, N = (case["I"], 2 * case["F"]) if gated else (case["K"], case["N"])
    out = case["F"] if gated else N
    held = not gated or case["int8"]
    wbytes = N * K + 4 * N if held else N * K * b
    bytes_ = M * K * b + wbytes + M * out * b + (N * b if case["bias"] else 0) + (M * N * b if case["base"] else 0)
    flops = 2 * M * N * K
    if case["train"]:
        bytes_ += M * out * b + M * K * b + (M * N * b if gated and case["base"] else 0)
        flops *= 2 if held else 3
        if not held:
            bytes_ += N * K * b + (N * b if case["bias"] else 0)
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    """The definition in 64 bits, the derivative by the chain rule on sigma, Phi and tanh written out once more."""
    s = prepare(case, seed)
    up = lambda t: None if t is None else t.to(torch.float64)  # noqa: E731
    if case["op"] == "quantize" or (case["op"] != "matmul" and "wq" in s):
        x = up(s["x"])
        top = x.abs().max(dim=1).values
        unit = torch.where(top > 0, top, torch.ones_like(top))
        whole = (x * 127.0).div_(unit.unsqueeze(1)).round_()
        step = top / 127.0
        if case["op"] == "quantize":
            return {"values": whole * step.unsqueeze(1), "scale": step}
        p = torch.mm(whole, up(s["wq"]).t().contiguous())
        p.mul_(step.unsqueeze(1)).mul_(up(s["sw"]).unsqueeze(0))
        w = up(s["wq"]).mul_(up(s["sw"]).unsqueeze(1)) if case["train"] else None
    elif case["op"] == "matmul":
        p = torch.mm(up(s["aq"]), up(s["wq"]).t().contiguous())
        p.mul_(up(s["sa"]).unsqueeze(1)).mul_(up(s["sw"]).unsqueeze(0))
        return {"y": p if s["bias"] is None else p.add_(up(s["bias"]))}
    else:
        w = up(s["w"])
        p = torch.mm(up(s["x"]), w.t().contiguous())
    for extra in ("bias", "base"):
        if s[extra] is not None:
            p = p + up(s[extra])
    if case["op"] == "linear":
        out = {"y": p}
        if case["train"]:
            out["dx"] = torch.mm(up(s["g"]), w)
        return out
    first, second = p.split(case["F"], dim=1)
    gate, value = (first, second) if case["gate_first"] else (second, first)
    if case["act"] == "silu":
        sig = torch.reciprocal(torch.exp(-gate) + 1.0)
        a = gate * sig
        slope = sig + a * (1.0 - sig)
    elif case["act"] == "gelu":
        phi = torch.erfc(gate * -(0.5 ** 0.5)) * 0.5
        a = gate * phi
        slope = phi + gate * torch.exp(gate * gate * -0.5) / (2.0 * math.pi) ** 0.5
    else:
        inner = (2.0 / math.pi) ** 0.5 * (gate + 0.044715 * gate ** 3)
        half = torch.reciprocal(torch.exp(-2.0 * inner) + 1.0)
        a = gate * half
        slope = half + 2.0 * gate * half * (1.0 - half) * (2.0 / math.pi) ** 0.5 * (1.0 + 0.134145 * gate ** 2)
    out = {"y": value * a}
    if not case["train"]:
        return out
    g = up(s["g"])
    d_gate, d_value = g * value * slope, g * a
    dp = torch.cat([d_gate, d_value] if case["gate_first"] else [d_value, d_gate], dim=1)
    out["dx"] = torch.mm(dp, w)
    if s["base"] is not None:
        out["dbase"] = dp
    if not case["int8"]:
        out["dw"] = torch.mm(dp.t().contiguous(), up(s["x"]))
        if s["bias"] is not None:
            out["dbias"] = dp.sum(dim=0)
    return out
