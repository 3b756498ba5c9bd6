"""The MX4 formats and operators (include/unoq_mx.h) restated in 64 bits on the CPU: the oracle of
test_mx_host.py and test_gpu_mx.py."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def stored(x):
    """Codes (rows, ceil(k/2)) and scales (rows, ceil(k/32)) of x, element by element from the definition:
    the nearest grid value, of two equally near the one with the even code."""
    x = x.cpu().double()
    rows, k = x.shape
    blocks = -(-k // 32)
    wide = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    wide[:, :k] = x
    b = wide.reshape(rows, blocks, 32)
    top = b.abs().amax(-1)
    _, e = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top)))
    s = torch.where(top > 0, (e - 1 - 2 + 127).clamp(min=0), torch.zeros_like(e))
    s = torch.where(torch.isfinite(top), s, torch.full_like(s, 255))
    unit = torch.ldexp(torch.ones_like(top), torch.where(s == 255, torch.zeros_like(s), s - 127))
    v = torch.where(torch.isfinite(top)[..., None], b, torch.zeros_like(b)) / unit[..., None]
    far = (v.abs().clamp(max=6.0)[..., None] - GRID).abs()
    near = far == far.amin(-1, keepdim=True)
    index = torch.arange(8)
    code = torch.where(near & (index % 2 == 0), index, 99).amin(-1)
    code = torch.where(code == 99, torch.where(near, index, 99).amin(-1), code)
    code = code + 8 * (torch.signbit(b) & torch.isfinite(top)[..., None])
    code = code.reshape(rows, blocks * 32)
    code[:, k:] = 0
    code = code[:, :2 * ((k + 1) // 2)].to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), s.to(torch.uint8)


def values(codes, scales, k):
    """(..., k) float64 values of a stored matrix."""
    codes, scales = codes.cpu(), scales.cpu()
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :k].long()
    v = GRID[c & 7] * (1 - 2 * (c >> 3)).double()
    s = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales.int() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return v * s.repeat_interleave(32, -1)[..., :k]


def operand(codes, scales, k, paired=False):
    """The operand layout of one stored matrix, placed byte by byte."""
    n = codes.shape[0]
    if paired:
        half = n // 2
        tiles = -(-half // 64)
        order = []
        for t in range(tiles):
            for part in range(2):
                order += [part * half + t * 64 + i if t * 64 + i < half else -1 for i in range(64)]
    else:
        order = [r if r < n else -1 for r in range(-(-n // 128) * 128)]
    kt = -(-k // 256) * 2
    out_c = torch.zeros(len(order) // 128 * kt * 8192, dtype=torch.uint8)
    out_s = torch.zeros(len(order) // 128 * kt * 512, dtype=torch.uint8)
    wide = torch.zeros(n, kt * 64, dtype=torch.uint8)
    wide[:, :codes.shape[1]] = codes.cpu()
    if k % 2:
        wide[:, k // 2] &= 15
    ws = torch.zeros(n, kt * 4, dtype=torch.uint8)
    ws[:, :scales.shape[1]] = scales.cpu()
    for to, r in enumerate(order):
        if r < 0:
            continue
        for t in range(kt):
            at = (to // 128 * kt + t)
            out_c[at // 2 * 16384 + to % 128 * 128 + t % 2 * 64:][:64] = wide[r, t * 64:t * 64 + 64]
            out_s[at * 512 + to % 32 * 16 + to % 128 // 32 * 4:][:4] = ws[r, t * 4:t * 4 + 4]
    return out_c, out_s


def select(logits, top, normalize):
    """Chosen experts (falling logits, ties to the lowest index) and their weights."""
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :top]
    p = torch.softmax(logits.gather(1, order), -1) if normalize else torch.softmax(logits, -1).gather(1, order)
    return order, p


def experts(x, router, gate_up, down, top, normalize, bias=None):
    """(y, chosen, weights, bound): the layer in 64 bits, and how far each value of y may be off before
    its last rounding, from the roundings that the operator documents (see `_sum_error`)."""
    x, router = x.cpu().double(), router.cpu().double()
    d, f = x.shape[1], gate_up[0].shape[1] // 2
    logits = x @ router.t() + (0 if bias is None else bias.cpu().double())
    order, p = select(logits, top, normalize)
    logit_off = _sum_error(d) * (x.abs() @ router.abs().t()).amax(1) + 2.0 ** -23 * logits.abs().amax(1)
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(top):
            e = int(order[t, j])
            gu = values(gate_up[0][e], gate_up[1][e], d)
            dn = values(down[0][e], down[1][e], f)
            g, u = gu[:f] @ x[t], gu[f:] @ x[t]
            off = _sum_error(d) * (gu.abs() @ x[t].abs())
            h = g * torch.sigmoid(g) * u
            # |silu'| <= 1.1; 2^-20: expf, a division and two products; 2^-13: half a step of 12 bits;
            # and the floor of a block's small values, 2^-21 of its largest
            top_h = h.abs().max() if f else 0
            dh = 1.1 * off[:f] * (u.abs() + off[f:]) + (g * torch.sigmoid(g)).abs() * off[f:]
            dh = dh + h.abs() * (2.0 ** -20 + 2.0 ** -13) + 2.0 ** -21 * top_h
            part = dn @ h
            size = dn.abs() @ (h.abs() + dh)
            y[t] += p[t, j] * part
            # the weights move by at most e^(2 off) - 1 < 3 off (their own sums: 2^-20)
            bound[t] += p[t, j] * (dn.abs() @ dh + _sum_error(f) * size + (3 * logit_off[t] + 2.0 ** -20) * part.abs())
    return y, order, p, bound


def _sum_error(k):
    """Relative to the sum of magnitudes: k additions in 32 bits, each cut off (not rounded) at worst."""
    return (k + 8) * 2.0 ** -23


def product_bound(a, w, y, dtype):
    """How far a product in 32 bits, rounded once to dtype, may be from y = a w^T in 64 bits."""
    return _sum_error(a.shape[1]) * (a.abs() @ w.abs().t()) + half_step(y, dtype)


def half_step(y, dtype):
    """Half a step of dtype at |y|, and below its normal range half a step of the subnormals."""
    info = torch.finfo(dtype)
    return (info.eps / 2) * y.abs() * (1 + info.eps) + info.smallest_normal * info.eps / 2


# ---- expert layers whose gate and up sums are exact in 32 bits ----------------------------------------

NONZERO = 4   # values of a row of `down` in the layers of `whole_layer`


def whole_layer(d, f, e, seed):
    """(x maker, gate_up, down): activations are whole numbers -2..2 and the codes' scales two neighbouring powers of
    two, so every gate and up sum is a multiple of half the smaller scale below 2^24 of them (48 d of them at most).
    Its spread is about 2, where SiLU is neither linear nor zero. A row of `down` has NONZERO values, all others
    zero, so that its sum has next to no error of its own."""
    g = torch.Generator().manual_seed(seed)
    low = 127 - round(math.log2(2.5 * math.sqrt(d)))
    code = torch.randint(0, 256, (e, 2 * f, (d + 1) // 2), generator=g, dtype=torch.uint8)
    scale = torch.randint(low, low + 2, (e, 2 * f, (d + 31) // 32), generator=g, dtype=torch.uint8)
    wide = torch.zeros(e, d, f + f % 2, dtype=torch.uint8)
    at = torch.randint(0, f, (e, d, NONZERO), generator=g)
    wide.scatter_(2, at, torch.randint(1, 8, at.shape, generator=g, dtype=torch.uint8) + 8 * (at % 2).to(torch.uint8))
    down = wide[..., 0::2] | wide[..., 1::2] << 4
    dscale = torch.randint(126, 129, (e, d, (f + 31) // 32), generator=g, dtype=torch.uint8)
    return (lambda t: torch.randint(-2, 3, (t, d), generator=g).double()), (code, scale), (down, dscale)


def hidden64(x, gate_up, e, f):
    """silu(gate) * up of every row of x through expert e, in 64 bits."""
    gu = x @ values(gate_up[0][e], gate_up[1][e], x.shape[1]).t()
    return gu[:, :f] * torch.sigmoid(gu[:, :f]) * gu[:, f:]


def whole_experts(x, order, gate_up, down):
    """(y, bound before the last rounding) of a `whole_layer` whose tokens give every one of the experts in `order`
    (a power of two of them) the same weight, which then is exact. The bound, for each value of y:
    * h = g / (1 + exp(-g)) * u in 32 bits: exp off by 2^-22 (2 units), sum, quotient and product by 2^-24 each: 2^-21
    * h is held to 2^-19 of itself, or 2^-29 of the largest of its block of 32 where that is more
    * the NONZERO products of a row and the pieces of each (_sum_error); the sum over the experts: 2^-24 for each."""
    f, top = gate_up[0].shape[1] // 2, order.shape[1]
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    for e in order.unique().tolist():
        t = (order == e).any(1).nonzero().flatten()
        h, dn = hidden64(x[t], gate_up, e, f), values(down[0][e], down[1][e], f)
        block = torch.nn.functional.pad(h.abs(), (0, -f % 32)).reshape(len(t), -1, 32).amax(-1)
        dh = h.abs() * (2.0 ** -21 + 2.0 ** -19) + 2.0 ** -29 * block.repeat_interleave(32, -1)[:, :f]
        y[t] += h @ dn.t() / top
        bound[t] += (dh + (_sum_error(NONZERO) + top * 2.0 ** -24) * h.abs()) @ dn.abs().t() / top
    return y, bound


def rounding_off(got, want, bound, dtype):
    """How far `got` of type dtype is outside of rounding `want` +- bound to dtype, in half steps (0: inside). The step
    is the one at the nearest end of the interval, so a value one step off is seen unless the interval holds the border."""
    info = torch.finfo(dtype)
    near = want.abs() - bound
    _, e = torch.frexp(near.clamp(min=info.smallest_normal))
    half = torch.ldexp(torch.full_like(want, info.eps / 2), (e - 1))
    # a value just under a power of two may round up to it, and one at its upper end has the step above it
    up = torch.ldexp(torch.ones_like(want), e) - near <= half + 2 * bound
    half = torch.where(up, 2 * half, half)
    return (((got.cpu().double() - want).abs() - bound) / half - 1).clamp(min=0)
