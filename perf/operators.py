"""Measured cases of the microscaled 4-bit operators (unoq_dsp.mx), with their plain forms.

An MX4 matrix holds e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) in blocks of 32
along a row; each block has a power-of-two scale, stored as a biased 8-bit exponent (255: not a
number). Its stored form is two byte matrices: codes (rows, ceil(k/2)), the even element in the low
nibble, and scales (rows, ceil(k/32)). Four kinds of case:

* ``round``   quantise a matrix and read its values back: weights or activations moved to 4 bits.
* ``mm4``     activations quantised in the call, times 4-bit weights: y = q(x) w^T.
* ``mm16``    16-bit activations times 4-bit weights: y = x w^T, nothing rounded on the way in.
* ``experts`` a mixture-of-experts layer for a few tokens: router, selection, gate / up and down
  products of 4-bit expert weights, weighted sum.
"""
import math
import sys

import torch

own = False

BLOCK = 32
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's activations: nothing but latency
        {"name": "round one row", "kind": "round", "m": 1, "k": 4096, "pad": 0, "type": "bf16"},
        # odd sizes in 32 bits, rows of a wider buffer
        {"name": "round odd f32", "kind": "round", "m": 997, "k": 1447, "pad": 9, "type": "f32"},
        # a large weight matrix moved to 4 bits
        {"name": "round weights", "kind": "round", "m": 8192, "k": 8192, "pad": 0, "type": "bf16"},
        # a decoding batch through a 4-bit layer
        {"name": "mm4 16 tokens", "kind": "mm4", "m": 16, "n": 4096, "k": 4096, "pad": 0, "type": "bf16", "out": "bf16"},
        # ragged everything, 32-bit logits out
        {"name": "mm4 odd", "kind": "mm4", "m": 333, "n": 1999, "k": 1447, "pad": 1, "type": "f16", "out": "f32"},
        # a long prompt through a wide layer: bound by the tensor cores
        {"name": "mm4 prompt", "kind": "mm4", "m": 4096, "n": 8192, "k": 4096, "pad": 0, "type": "bf16", "out": "bf16"},
        # one token through a large layer: bound by reading its weights
        {"name": "mm16 one token", "kind": "mm16", "m": 1, "n": 8192, "k": 8192, "pad": 0, "type": "bf16", "out": "bf16"},
        # an uneven batch in half precision
        {"name": "mm16 odd f16", "kind": "mm16", "m": 45, "n": 5003, "k": 2085, "pad": 3, "type": "f16", "out": "f16"},
        # a prompt with 16-bit activations
        {"name": "mm16 prompt", "kind": "mm16", "m": 2048, "n": 4096, "k": 4096, "pad": 0, "type": "bf16", "out": "bf16"},
        # one token through a small layer of experts: latency
        {"name": "experts one token", "kind": "experts", "m": 1, "d": 2048, "f": 1024, "e": 32, "top": 4, "norm": True, "type": "bf16"},
        # a few tokens, odd widths, weights of the softmax over all experts
        {"name": "experts odd f16", "kind": "experts", "m": 7, "d": 1447, "f": 999, "e": 60, "top": 3, "norm": False, "type": "f16"},
        # the largest batch such a layer takes: nearly every expert is read
        {"name": "experts 64 tokens", "kind": "experts", "m": 64, "d": 2048, "f": 1024, "e": 128, "top": 8, "norm": True, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("round", "mm4", "mm16", "experts"))
    if kind == "round":
        k = _log(rng, 33, 8192)
        return {"kind": kind, "m": _log(rng, 1, 8192), "k": k, "pad": rng.choice((0, 0, 1, 8)), "type": rng.choice(sorted(TYPES))}
    if kind == "experts":
        e = _log(rng, 8, 128)
        return {"kind": kind, "m": _log(rng, 1, 64), "d": _log(rng, 256, 2048), "f": _log(rng, 256, 1024), "e": e,
                "top": rng.randint(1, min(8, e)), "norm": rng.random() < 0.5, "type": rng.choice(("bf16", "f16"))}
    m = _log(rng, 1, 2048)
    n, k = _log(rng, 256, 8192), _log(rng, 128, 4096)
    kind_type = rng.choice(("bf16", "f16"))
    return {"kind": kind, "m": m, "n": n, "k": k, "pad": rng.choice((0, 0, 1, 8)), "type": kind_type,
            "out": rng.choice((kind_type, "f32"))}


def work(case):
    c = dict(case)
    if c["kind"] == "round":
        return {"bytes": 2.0 * c["m"] * c["k"] * SIZE[c["type"]], "flops": 0.0}
    if c["kind"] == "experts":
        # experts that m tokens select, each choosing `top` of `e` at random
        read = c["e"] * (1.0 - (1.0 - c["top"] / c["e"]) ** c["m"])
        return {"bytes": read * 3.0 * c["d"] * c["f"] * 17 / 32 + 2.0 * c["e"] * c["d"] + 4.0 * c["m"] * c["d"],
                "flops": 2.0 * c["m"] * (c["top"] * 3.0 * c["d"] * c["f"] + c["e"] * c["d"])}
    m, n, k = c["m"], c["n"], c["k"]
    return {"bytes": 2.0 * m * k + n * k * 17 / 32 + 1.0 * m * n * SIZE[c["out"]], "flops": 2.0 * m * n * k}


# ---- plain forms ---------------------------------------------------------------------------------

def _power(e):
    """2^e of whole numbers, exactly, in 64 bits (a device's exp2 need not be)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored(x):
    """Stored form of x's rows: per block, scale 2^(floor(log2 of the largest) - 2), values to the
    nearest e2m1 (ties to the even code), at most 6; a block holding a NaN or an infinity is NaN."""
    x = x.float()
    rows, k = x.shape
    kb = -(-k // BLOCK)
    x = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).reshape(rows, kb, BLOCK)
    top = x.abs().amax(-1)
    exponent = torch.frexp(top).exponent.clamp(min=-124) + 124        # frexp: top = f * 2^exponent, f in [0.5, 1)
    exponent = torch.where(top == 0, torch.zeros_like(exponent), exponent)
    finite = torch.isfinite(top)
    scale = torch.where(finite, exponent, torch.full_like(exponent, 255))
    v = x.double() * _power(127 - scale)[..., None]
    a = torch.where(finite[..., None], v.abs(), torch.zeros_like(v))
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (torch.signbit(x) & finite[..., None])).to(torch.uint8).reshape(rows, kb * BLOCK)
    code = torch.nn.functional.pad(code[:, :k], (0, k % 2))
    return code[:, 0::2] | (code[:, 1::2] << 4), scale.to(torch.uint8)


def _values(codes, scales, k):
    """The values of a stored matrix, in 32 bits: (..., k)."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)[..., :k]
    s = _power(scales.int() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s).float()
    return v * s.repeat_interleave(BLOCK, -1)[..., :k]


def _select(logits, top, norm):
    """Chosen experts (ties to the lowest index) and their weights, from 64-bit logits."""
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
    if norm:
        return order, torch.softmax(logits.gather(1, order), -1)
    return order, torch.softmax(logits, -1).gather(1, order)


def _plain_experts(s):
    x = s["x"].float()
    d, f = s["d"], s["f"]
    logits = s["x"].double() @ s["router"].double().t()
    order, weight = _select(logits, s["top"], s["norm"])
    share = torch.zeros_like(logits).scatter(1, order, weight).float()          # (m, e)
    gu = torch.matmul(x, _values(*s["gate_up"], d).transpose(1, 2))             # (e, m, 2f)
    g, u = gu[..., :f], gu[..., f:]
    h = g / (1 + torch.exp(-g)) * u
    y = torch.matmul(h, _values(*s["down"], f).transpose(1, 2))                 # (e, m, d)
    return (y * share.t()[..., None]).sum(0).to(s["x"].dtype)


# ---- the tools' functions ------------------------------------------------------------------------

def _mx():
    if "unoq-dsp_b200" not in sys.path:
        sys.path.insert(1, "unoq-dsp_b200")
    from unoq_dsp import mx
    return mx


def _matrix(g, rows, k, pad, kind):
    """Activations as a network has them: normal values, a few channels much larger than the rest."""
    wide = torch.randn(rows, k + pad, generator=g, device="cuda")
    loud = 1 + 15 * (torch.rand(k + pad, generator=g, device="cuda") < 0.01).float()
    return (wide * loud).to(TYPES[kind])[:, :k]


def _weights(g, *shape):
    """Stored 4-bit weights with the spread that a trained layer of that width has."""
    rows, k = math.prod(shape[:-1]), shape[-1]
    codes, scales = _stored(torch.randn(rows, k, generator=g, device="cuda") / math.sqrt(k))
    return codes.reshape(*shape[:-1], -1), scales.reshape(*shape[:-1], -1)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if c["kind"] == "experts":
        d, f, e = c["d"], c["f"], c["e"]
        dtype = TYPES[c["type"]]
        s = dict(c, x=torch.randn(c["m"], d, generator=g, device="cuda").to(dtype),
                 router=(torch.randn(e, d, generator=g, device="cuda") / math.sqrt(d)).to(dtype))
        parts = [_weights(g, 2 * f, d) for _ in range(e)]
        s["gate_up"] = tuple(torch.stack(p) for p in zip(*parts))
        parts = [_weights(g, d, f) for _ in range(e)]
        s["down"] = tuple(torch.stack(p) for p in zip(*parts))
        if own:  # the layer that a program keeps: its weights in the kernels' layout
            s["layer"] = _mx().Experts(s["router"], s["gate_up"], s["down"], top_k=c["top"], normalize=c["norm"])
        return s
    s = dict(c, x=_matrix(g, c["m"], c["k"], c["pad"], c["type"]))
    if c["kind"] != "round":
        s["w"] = _weights(g, c["n"], c["k"])
        if own:  # the weight that a program keeps, in the kernels' layout
            s["weight"] = _mx().pack(*s["w"], k=c["k"])
    return s


def run(state):
    s = state
    if own:
        mx = _mx()
        if s["kind"] == "round":
            return mx.quantize(s["x"]).dequantize(s["x"].dtype)
        if s["kind"] == "experts":
            return s["layer"](s["x"])
        x = mx.quantize(s["x"]) if s["kind"] == "mm4" else s["x"]
        return mx.matmul(x, s["weight"], dtype=TYPES[s["out"]])
    if s["kind"] == "experts":
        return _plain_experts(s)
    x = _values(*_stored(s["x"]), s["k"]) if s["kind"] != "mm16" else s["x"].float()
    if s["kind"] == "round":
        return x.to(s["x"].dtype)
    return (x @ _values(*s["w"], s["k"]).t()).to(TYPES[s["out"]])


# ---- the definition in 64 bits, written apart ------------------------------------------------------

def _round64(x):
    """x's rows rounded to MX4, by the grid spacing of each value's binade, in 64 bits."""
    rows, k = x.shape
    out = torch.empty(rows, k, dtype=torch.float64, device=x.device)
    for at in range(0, k, BLOCK):
        b = x[:, at:at + BLOCK].double()
        top = b.abs().max(1, keepdim=True).values
        binade = (top.view(torch.int64) >> 52) - 1023
        unit = ((binade.clamp(min=-125) - 2 + 1023) << 52).view(torch.float64)
        v = b / unit
        size = v.abs()
        step = 0.5 + 0.5 * (size >= 2) + 1.0 * (size >= 4)
        out[:, at:at + BLOCK] = (torch.round(v / step) * step).clamp(-6, 6) * unit
    return out


def _read64(codes, scales, k):
    """A stored matrix's values from the bits of their codes, in 64 bits."""
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int32, device=codes.device)
    c[..., 0::2] = codes.int() % 16
    c[..., 1::2] = codes.int() // 16
    c = c[..., :k]
    mantissa, power, sign = c % 2, (c // 2) % 4, c // 8
    v = torch.where(power == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * (1 << power) / 2).double() * (1 - 2 * sign)
    block = torch.arange(k, device=codes.device) // BLOCK
    return v * ((scales.long()[..., block] - 127 + 1023) << 52).view(torch.float64)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if s["kind"] == "round":
        return _round64(s["x"])
    if s["kind"] != "experts":
        x = _round64(s["x"]) if s["kind"] == "mm4" else s["x"].double()
        return x @ _read64(*s["w"], s["k"]).t()
    x = s["x"].double()
    score = x @ s["router"].double().t()
    y = torch.zeros_like(x)
    whole = torch.exp(score - score.max(1, keepdim=True).values)
    left, chosen = score.clone(), torch.zeros_like(score)
    for _ in range(s["top"]):
        best = left.argmax(1, keepdim=True)
        chosen.scatter_(1, best, 1.0)
        left.scatter_(1, best, -math.inf)
    part = whole * chosen / (whole * (chosen if s["norm"] else 1)).sum(1, keepdim=True)
    for j in range(s["e"]):
        t = torch.nonzero(chosen[:, j])[:, 0]
        if len(t):
            gu = x[t] @ _read64(s["gate_up"][0][j], s["gate_up"][1][j], s["d"]).t()
            g, u = gu[:, :s["f"]], gu[:, s["f"]:]
            h = g * torch.sigmoid(g) * u
            y[t] += part[t, j:j + 1] * (h @ _read64(s["down"][0][j], s["down"][1][j], s["f"]).t())
    return y
