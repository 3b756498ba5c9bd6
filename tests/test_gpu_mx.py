"""The MX4 operators on the GPU against their definition in 64 bits (mxref.py): formats and rounding bit for
bit, products exactly where every partial sum is a 24-bit number and within the bound of 32-bit sums
elsewhere, the expert layer within the bound that follows from its documented roundings."""
import ctypes as C
import functools
import math

import pytest
import torch

import mxref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mx():
    from unoq_dsp import mx
    return mx


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def matrix(rows, k, dtype, seed, pad=0, offset=0):
    """Values of several magnitudes in a view whose rows are k + pad apart, `offset` elements into it."""
    g = gen(seed)
    flat = torch.randn(rows * (k + pad) + offset, generator=g, device="cuda")
    flat = flat * torch.exp(2 * torch.randn(flat.shape, generator=g, device="cuda"))
    return flat.to(dtype)[offset:].view(rows, k + pad)[:, :k]


def on_gpu(pair):
    return tuple(t.cuda() for t in pair)


@functools.lru_cache(maxsize=16)
def weights(n, k, seed, batch=None):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((batch or 1) * n, k, generator=g) / math.sqrt(k)
    c, s = mxref.stored(w)
    if batch:
        return c.view(batch, n, -1), s.view(batch, n, -1)
    return c, s


def assert_within(got, want, bound, what=""):
    got, want = got.cpu().double(), want.double()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    off = (got - want).abs()[~nan]
    over = off > bound.double()[~nan]
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} outside, worst {float((off / bound[~nan].clamp(min=1e-300)).max()):.3g} of its bound"


SIZES = [(1, 1), (1, 2), (3, 31), (2, 32), (5, 33), (1, 127), (130, 128), (4, 129), (257, 77), (64, 1024), (33, 4099)]


# ---- formats -------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantize_is_the_definition(mx, rows, k, name):
    for pad, offset in ((0, 0), (1, 0), (8, 8), (5, 3)):
        x = matrix(rows, k, mxref.TYPES[name], rows * k, pad, offset)
        c, s = mxref.stored(x)
        q = mx.quantize(x, layout="stored")
        assert torch.equal(q.scales.cpu(), s) and torch.equal(q.codes.cpu(), c)
        o = mx.quantize(x)
        for dtype in mxref.TYPES.values():
            want = mxref.values(c, s, k).to(dtype)
            assert torch.equal(q.dequantize(dtype).cpu(), want) and torch.equal(o.dequantize(dtype).cpu(), want)


def test_quantize_operand_bytes(mx):
    for rows, k in ((128, 128), (256, 384), (128, 200)):
        x = matrix(rows, k, torch.bfloat16, k)
        want = mxref.operand(*mxref.stored(x), k)
        q = mx.quantize(x)
        assert torch.equal(q.codes.cpu(), want[0]) and torch.equal(q.scales.cpu(), want[1])


def test_quantize_borders_and_extremes(mx):
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 0.0, -0.0])
    ties = torch.cat((ties, -ties, torch.nextafter(ties, torch.tensor(9.0))))
    x = torch.zeros(12, 64)
    x[:, :36] = ties
    x[:, 40] = 7.0
    x = x * torch.ldexp(torch.ones(12, 1), torch.tensor([[0], [5], [-20], [120], [-120], [-130], [-140], [125], [-149], [1], [-1], [-126]]))
    x[3] = 0
    q = mx.quantize(x.cuda(), layout="stored")
    c, s = mxref.stored(x)
    assert torch.equal(q.scales.cpu(), s) and torch.equal(q.codes.cpu(), c)
    assert torch.equal(q.dequantize(torch.float32).cpu().double(), mxref.values(c, s, 64).float().double())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_nonfinite_value_makes_its_block_nan(mx, bad):
    x = matrix(6, 96, torch.float32, 1)
    x[1, 40] = bad
    x[4, 95] = bad
    for layout in ("stored", "operand"):
        v = mx.quantize(x, layout=layout).dequantize(torch.float32).cpu()
        want = mxref.values(*mxref.stored(x), 96)
        assert torch.equal(torch.isnan(v), torch.isnan(want)) and int(torch.isnan(v).sum()) == 64
        assert torch.equal(v[~torch.isnan(v)].double(), want[~torch.isnan(want)])


@pytest.mark.parametrize("n,k", [(1, 1), (2, 33), (130, 77), (256, 128), (129, 4099)])
def test_pack_is_the_operand_layout(mx, n, k):
    c, s = weights(n, k, n + k)
    if k % 2:
        c = c.clone()
        c[:, -1] |= 0xF0  # what files hold in the nibble past the last value is not read
    p = mx.pack(c.cuda(), s.cuda(), k=k)
    want = mxref.operand(c, s, k)
    assert torch.equal(p.codes.cpu(), want[0]) and torch.equal(p.scales.cpu(), want[1])
    assert torch.equal(p.dequantize(torch.float32).cpu().double(), mxref.values(c, s, k))


def test_pack_of_paired_matrices(mx):
    for f, d in ((1, 5), (128, 64), (200, 130)):
        c, s = weights(2 * f, d, f, batch=3)
        layer = mx.Experts(torch.zeros(3, d, dtype=torch.bfloat16, device="cuda"), (c.cuda(), s.cuda()),
                           on_gpu(weights(d, f, 1, batch=3)), 2)
        parts = [mxref.operand(c[e], s[e], d, paired=True) for e in range(3)]
        assert torch.equal(layer.gate_up[0].cpu(), torch.cat([p[0] for p in parts]))
        assert torch.equal(layer.gate_up[1].cpu(), torch.cat([p[1] for p in parts]))


def test_dequantize_leaves_the_rest_of_a_wide_output(mx):
    x = matrix(5, 70, torch.bfloat16, 3)
    wide = torch.full((6, 90), 7.0, device="cuda", dtype=torch.float16)
    mx.quantize(x).dequantize(torch.float16, out=wide[:5, :70])
    assert (wide[5] == 7).all() and (wide[:, 70:] == 7).all()
    assert torch.equal(wide[:5, :70].cpu(), mxref.values(*mxref.stored(x), 70).to(torch.float16))


# ---- products ------------------------------------------------------------------------------------

PRODUCTS = [(1, 1, 1), (1, 8, 32), (2, 3, 33), (7, 129, 127), (8, 128, 128), (9, 300, 700), (10, 140, 1500), (11, 130, 260), (16, 256, 512), (16, 1200, 2049), (17, 200, 1000), (65, 130, 257),
            (128, 256, 384), (129, 384, 640), (200, 1000, 96), (257, 515, 1023), (300, 129, 4100), (1, 4096, 4096),
            (3, 2049, 8192), (40, 4097, 2080), (600, 700, 300),
            # many tokens: pairs of CTAs, odd numbers of row tiles and ragged last tiles among them
            (1100, 2400, 300), (700, 2433, 1000), (330, 2433, 129), (2000, 2700, 640), (1025, 4800, 65), (2048, 2304, 520),
            (513, 8200, 70)]


def whole(rows, k, seed, narrow):
    """MX4 values whose products and sums are exact in 32 bits: scales 1 and 2 (or 1)."""
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, 256, (rows, (k + 1) // 2), generator=g, dtype=torch.uint8)
    if k % 2:
        c[:, -1] &= 15
    s = torch.randint(127, 128 if narrow else 129, (rows, (k + 31) // 32), generator=g, dtype=torch.uint8)
    return c, s


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_exact(mx, m, n, k):
    a, w = whole(m, k, m + k, True), whole(n, k, n * 3 + k, False)
    want = mxref.values(*a, k) @ mxref.values(*w, k).t()   # multiples of 1/4 below 2^22: exact in 32 bits
    A, W = mx.pack(*on_gpu(a), k=k), mx.pack(*on_gpu(w), k=k)
    assert torch.equal(mx.matmul(A, W, dtype=torch.float32).cpu().double(), want)
    for dtype in (torch.float16, torch.bfloat16):
        assert torch.equal(mx.matmul(A, W, dtype=dtype).cpu(), want.to(torch.float32).to(dtype))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_x16_exact(mx, m, n, k, name):
    # whole activations up to 255: eight bits, exact in both types, and within 2^-12 of their blocks' largest
    g = torch.Generator().manual_seed(m + n + k)
    x = torch.randint(-255, 256, (m, k), generator=g).to(mxref.TYPES[name])
    c, s = whole(n, k, n + k, True)
    # products are multiples of 1/2; the sum of magnitudes stays below 2^23 halves
    want = x.double() @ mxref.values(c, s, k).t()
    W = mx.pack(c.cuda(), s.cuda(), k=k)
    bound = torch.zeros_like(want) if float((x.double().abs() @ mxref.values(c, s, k).abs().t()).max()) < 2 ** 22 else \
        mxref.product_bound(x.double(), mxref.values(c, s, k), want, torch.float32)
    assert_within(mx.matmul(x.cuda(), W, dtype=torch.float32), want, bound)


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_of_quantised_activations(mx, m, n, k):
    x = matrix(m, k, torch.bfloat16, m * n)
    c, s = weights(n, k, m)
    a, w = mxref.values(*mxref.stored(x), k), mxref.values(c, s, k)
    W = mx.pack(c.cuda(), s.cuda(), k=k)
    for dtype in mxref.TYPES.values():
        assert_within(mx.matmul(mx.quantize(x), W, dtype=dtype), a @ w.t(), mxref.product_bound(a, w, a @ w.t(), dtype), str(dtype))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul_x16(mx, m, n, k, name):
    x = torch.randn(m, k + 3, generator=gen(m + n), device="cuda")
    x = (x * torch.exp(torch.randn(x.shape, generator=gen(n), device="cuda"))).to(mxref.TYPES[name])[:, :k]
    c, s = weights(n, k, n)
    a, w = x.cpu().double(), mxref.values(c, s, k)
    pieces = (a.abs().amax(1, keepdim=True) * 2.0 ** -21) @ w.abs().sum(1)[None]  # the documented floor of small values
    W = mx.pack(c.cuda(), s.cuda(), k=k)
    for dtype in mxref.TYPES.values():
        assert_within(mx.matmul(x, W, dtype=dtype), a @ w.t(), mxref.product_bound(a, w, a @ w.t(), dtype) + pieces, str(dtype))


def test_matmul_x16_wide_range_in_a_block(mx):
    """Values far below their block's largest: exact down to 2^-12 of it, within 2^-21 of it below."""
    k = 64
    c, s = whole(16, k, 5, True)
    w = mxref.values(c, s, k)
    for dtype in (torch.bfloat16, torch.float16):
        for shift in range(0, 24):
            x = torch.zeros(1, k)
            x[0, 0] = 96.0
            x[0, 7] = 1.8359375 * 2.0 ** (6 - shift)   # eight significant bits
            x[0, 33] = -3.0
            x = x.to(dtype)
            want = x.double() @ w.t()
            got = mx.matmul(x.cuda(), mx.pack(c.cuda(), s.cuda(), k=k), dtype=torch.float32).cpu().double()
            floor = 0.0 if shift <= 12 else 6 * 96 * 2.0 ** -21
            # the sum itself: three products in 32 bits
            bound = floor + 4 * 2.0 ** -23 * (x.double().abs() @ w.abs().t())
            assert ((got - want).abs() <= bound).all(), (dtype, shift)


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -120, 2.0 ** 100])
def test_matmul_x16_far_magnitudes(mx, scale):
    x = (torch.randn(3, 256, generator=gen(1), device="cuda") * scale).to(torch.bfloat16)
    c, s = weights(40, 256, 3)
    a, w = x.cpu().double(), mxref.values(c, s, 256)
    # below 2^-108 the last piece's scale byte stops at 0: its grid is 2^-127 * 2^-9, half of that per value
    low = 2.0 ** -137 * w.abs().sum(1)[None]
    got = mx.matmul(x, mx.pack(c.cuda(), s.cuda()), dtype=torch.float32)
    pieces = (a.abs().amax(1, keepdim=True) * 2.0 ** -21) @ w.abs().sum(1)[None]
    assert_within(got, a @ w.t(), mxref.product_bound(a, w, a @ w.t(), torch.float32) + pieces + low)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite_rows_stay_apart(mx, bad):
    x = torch.randn(20, 300, generator=gen(2), device="cuda").to(torch.bfloat16)
    x[3, 299] = bad
    x[17, 0] = bad
    c, s = weights(140, 300, 2)
    W = mx.pack(c.cuda(), s.cuda())
    for a in (x, mx.quantize(x)):
        y = mx.matmul(a, W)
        rows = torch.isnan(y).all(1)
        assert rows.nonzero().flatten().tolist() == [3, 17] and not torch.isnan(y[~rows]).any()
    s2 = s.clone()
    s2[9, 1] = 255  # a weight block that is not a number: one column
    y = mx.matmul(x[:3], mx.pack(c.cuda(), s2.cuda()))
    assert torch.isnan(y).all(0).nonzero().flatten().tolist() == [9] and not torch.isnan(y[:, :9]).any()


def test_zero_rows_and_columns(mx):
    W = mx.pack(*on_gpu(weights(16, 64, 1)))
    assert mx.matmul(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16), W).shape == (0, 16)
    q = mx.quantize(torch.empty(0, 64, device="cuda"))
    assert q.shape == (0, 64) and q.dequantize().shape == (0, 64) and mx.matmul(q, W).shape == (0, 16)
    none = mx.quantize(torch.empty(0, 64, device="cuda"))
    assert mx.matmul(torch.ones(3, 64, device="cuda", dtype=torch.float16), none).shape == (3, 0)


def test_matmul_shapes_and_outputs(mx):
    x = torch.randn(2, 3, 96, generator=gen(4), device="cuda").to(torch.float16)
    W = mx.pack(*on_gpu(weights(50, 96, 4)))
    y = mx.matmul(x, W)
    assert y.shape == (2, 3, 50) and y.dtype == torch.float16
    assert torch.equal(mx.matmul(x.view(6, 96), W).view(2, 3, 50), y)
    assert torch.equal(mx.matmul(x[0, 1], W), y[0, 1])
    t = x.view(6, 96).t().contiguous().t()  # values of a row apart: copied first
    assert torch.equal(mx.matmul(t, W).view(2, 3, 50), y)
    one = x[:1, :1].expand(1, 4, 96)        # rows that are one row
    assert torch.equal(mx.matmul(one, W)[0, 3], y[0, 0])
    wide = torch.full((8, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    mx.matmul(x.view(6, 96), W, dtype=torch.bfloat16, out=wide[:6, 5:55])
    assert torch.equal(wide[:6, 5:55], mx.matmul(x.view(6, 96), W, dtype=torch.bfloat16))
    rest = torch.ones_like(wide, dtype=torch.bool)
    rest[:6, 5:55] = False
    assert (wide[rest] == 3).all()


def test_quantised_weights_with_ragged_rows(mx):
    """A quantised weight is a packed one up to the rows that pad its last tile, which no output shows."""
    for n, k in ((1, 40), (130, 300), (257, 513), (2433, 64)):
        w = torch.randn(n, k, generator=gen(n), device="cuda")
        q, p = mx.quantize(w), mx.pack(*on_gpu(mxref.stored(w)), k=k)
        for m in (1, 5, 40, 700):
            x = torch.randn(m, k, generator=gen(m), device="cuda").to(torch.bfloat16)
            assert torch.equal(mx.matmul(x, q), mx.matmul(x, p))
            assert torch.equal(mx.matmul(mx.quantize(x), q), mx.matmul(mx.quantize(x), p))


def test_an_operand_from_its_bytes(mx):
    q = mx.quantize(torch.randn(70, 300, generator=gen(1), device="cuda"))
    again = mx.MX4(q.codes.clone(), q.scales.clone(), 70, 300)
    x = torch.randn(3, 300, generator=gen(2), device="cuda").to(torch.float16)
    assert torch.equal(mx.matmul(x, q), mx.matmul(x, again)) and torch.equal(q.dequantize(), again.dequantize())
    s = mx.quantize(torch.randn(70, 300, generator=gen(1), device="cuda"), layout="stored")
    assert s.codes.shape == (70, 150) and s.scales.shape == (70, 10)
    assert torch.equal(mx.pack(s.codes, s.scales).dequantize(), q.dequantize())


def test_python_refusals(mx):
    x = torch.randn(4, 64, device="cuda").to(torch.bfloat16)
    W = mx.pack(*on_gpu(weights(16, 64, 1)))
    with pytest.raises(ValueError, match="float64"):
        mx.quantize(x.double())
    with pytest.raises(ValueError, match="gradient"):
        mx.quantize(x.float().requires_grad_())
    with torch.no_grad():
        mx.quantize(x.float().requires_grad_())
    with pytest.raises(ValueError, match="at least one"):
        mx.quantize(x[:, :0])
    with pytest.raises(ValueError, match="layout"):
        mx.quantize(x, layout="rows")
    with pytest.raises(ValueError, match="operand"):
        mx.matmul(x, mx.quantize(x, layout="stored"))
    with pytest.raises(ValueError, match="rows of 32"):
        mx.matmul(x[:, :32], W)
    with pytest.raises(ValueError):
        mx.matmul(x.float(), W)
    with pytest.raises(ValueError, match="dtype"):
        mx.matmul(x, W, dtype=torch.float64)
    with pytest.raises(ValueError, match="shape"):
        mx.matmul(x, W, out=torch.empty(4, 17, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="overlap"):
        mx.matmul(x[:, :64], W, out=x[:, :16])
    with pytest.raises(ValueError, match="contiguous rows"):
        mx.matmul(x, W, out=torch.empty(16, 4, device="cuda", dtype=torch.bfloat16).t())
    with pytest.raises(ValueError, match="bytes"):
        mx.MX4(W.codes[:-1], W.scales, 16, 64)
    with pytest.raises(ValueError, match="code and"):
        mx.pack(torch.zeros(4, 32, dtype=torch.uint8, device="cuda"), torch.zeros(4, 2, dtype=torch.uint8, device="cuda"), k=66)


def test_abi_refuses_host_pointers(native):
    d = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    h = torch.zeros(1 << 16, dtype=torch.uint8)
    at = (h.data_ptr() + 255) // 256 * 256
    assert native.ug_mx4_quantize(at, 0, 1, 32, 32, 0, d.data_ptr(), d.data_ptr() + 4096, None) == 22
    assert native.ug_mx4_matmul(d.data_ptr(), d.data_ptr(), 1, d.data_ptr(), at, 8, 32, d.data_ptr() + 32768, 0, 8, None) == 22
    assert native.ug_mx4_check(99) == 2002
    assert native.ug_mx4_check(0) == 0


# ---- the expert layer ------------------------------------------------------------------------------

EXPERTS = [  # tokens, d, f, experts, top_k, normalize, type, bias
    (1, 1, 1, 1, 1, True, "bf16", False), (1, 64, 64, 4, 2, True, "bf16", False), (1, 512, 256, 32, 4, True, "bf16", True),
    (3, 130, 70, 5, 5, False, "f16", False), (7, 333, 129, 60, 3, False, "f16", True), (2, 1024, 384, 8, 1, True, "f16", False),
    (16, 256, 512, 16, 2, True, "bf16", False), (33, 257, 200, 4, 3, True, "bf16", False), (64, 384, 128, 128, 8, True, "bf16", False),
    (64, 128, 256, 2, 2, False, "f16", False), (128, 200, 136, 256, 16, True, "bf16", True), (128, 256, 128, 3, 1, True, "f16", False),
    (5, 1447, 999, 12, 4, True, "bf16", False),
    # long rows: their scales, and so K, spread over a cluster
    (3, 16384, 64, 2, 2, True, "bf16", False), (2, 40, 16384, 2, 1, True, "f16", False), (128, 4200, 70, 2, 2, True, "bf16", False),
    (20, 300, 4300, 3, 2, False, "bf16", False),
    # at most 32 pairs, and just more: the parts are added in the product, or after it
    (16, 260, 130, 20, 2, True, "bf16", False), (11, 260, 130, 20, 3, True, "bf16", False)]


def layer_parts(d, f, e, name, bias, seed):
    g = torch.Generator().manual_seed(seed)
    router = (torch.randn(e, d, generator=g) / math.sqrt(d)).to(mxref.TYPES[name])
    return router, weights(2 * f, d, seed + 1, batch=e), weights(d, f, seed + 2, batch=e), \
        torch.randn(e, generator=g) if bias else None


def distinct(x, router, bias, top):
    """Rows of x whose choice does not hang on the last bits of the logits."""
    logits = x.cpu().double() @ router.double().t() + (0 if bias is None else bias.double())
    if logits.shape[1] == top:
        gap = torch.ones(logits.shape[0])
    else:
        s = logits.sort(-1, descending=True).values
        gap = s[:, top - 1] - s[:, top]
    order = logits.sort(-1, descending=True).values[:, :top]
    inner = (order[:, :-1] - order[:, 1:]).amin(-1) if top > 1 else torch.ones(logits.shape[0])
    return (torch.minimum(gap, inner) > 1e-4).cpu()


@pytest.mark.parametrize("t,d,f,e,top,norm,name,with_bias", EXPERTS)
def test_experts(mx, t, d, f, e, top, norm, name, with_bias):
    router, gate_up, down, bias = layer_parts(d, f, e, name, with_bias, t + d)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), top, norm, None if bias is None else bias.cuda())
    x = torch.randn(t, d + 5, generator=gen(d), device="cuda").to(mxref.TYPES[name])[:, :d]
    y, chosen, p = layer(x, return_choice=True)
    ok = distinct(x, router, bias, top)
    assert ok.sum() >= t / 2
    want, order, weight, bound = mxref.experts(x, router, gate_up, down, top, norm, bias)
    assert torch.equal(chosen.cpu().long()[ok], order[ok])
    # softmax weights: 3 times what the logits are off by, and 2^-20 for expf and the division
    logit_off = (mxref._sum_error(d) + 2.0 ** -22) * (x.cpu().double().abs() @ router.double().abs().t() + 3).amax(1, keepdim=True)
    assert ((p.cpu().double() - weight).abs()[ok] <= ((3 * logit_off + 2.0 ** -20) * weight)[ok]).all()
    assert_within(y[ok.cuda()], want[ok], (bound + mxref.half_step(want, x.dtype))[ok])
    assert torch.equal(layer(x), y)  # same answer every time


def test_experts_ties_go_to_the_lowest_index(mx):
    router, gate_up, down, _ = layer_parts(64, 64, 40, "bf16", False, 3)
    router[:] = router[0]
    router[7] = router[0] * 2
    x = torch.randn(9, 64, generator=gen(1), device="cuda").to(torch.bfloat16)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 4)
    _, chosen, _ = layer(x, return_choice=True)
    sign = (x.cpu().double() @ router[0].double()) > 0
    for row, up in zip(chosen.tolist(), sign.tolist()):
        assert row == ([7, 0, 1, 2] if up else [0, 1, 2, 3])


def test_experts_masked_by_the_bias(mx):
    """Experts of a bias of minus infinity: chosen last, with no weight; none else is read as a number."""
    router, gate_up, down, _ = layer_parts(128, 70, 9, "bf16", False, 4)
    bias = torch.full((9,), -math.inf)
    bias[[2, 6]] = 0.5
    x = torch.randn(7, 128, generator=gen(5), device="cuda").to(torch.bfloat16)
    parts = (router.cuda(), on_gpu(gate_up), on_gpu(down))
    for norm in (True, False):
        y, chosen, p = mx.Experts(*parts, 4, norm, bias.cuda())(x, return_choice=True)
        assert {2, 6} == set(chosen[:, :2].flatten().tolist()) and chosen[:, 2:].tolist() == [[0, 1]] * 7
        assert (p[:, 2:] == 0).all() and torch.allclose(p.sum(1), torch.ones(7, device="cuda"), atol=2 ** -20)
        assert torch.equal(y, mx.Experts(*parts, 2, norm, bias.cuda())(x))


def test_experts_every_token_to_one_expert(mx):
    """The most uneven load: all tokens choose the same two experts of many."""
    router, gate_up, down, _ = layer_parts(256, 200, 24, "bf16", False, 9)
    bias = torch.full((24,), -50.0)
    bias[[3, 20]] = 50.0
    x = torch.randn(128, 256, generator=gen(6), device="cuda").to(torch.bfloat16)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2, bias=bias.cuda())
    y, chosen, _ = layer(x, return_choice=True)
    assert set(chosen.flatten().tolist()) == {3, 20}
    ok = distinct(x, router, bias, 2)
    want, _, _, bound = mxref.experts(x, router, gate_up, down, 2, True, bias)
    assert_within(y[ok.cuda()], want[ok], (bound + mxref.half_step(want, x.dtype))[ok])


def test_experts_nonfinite_token(mx):
    router, gate_up, down, _ = layer_parts(96, 64, 8, "bf16", False, 5)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2)
    x = torch.randn(6, 96, generator=gen(3), device="cuda").to(torch.bfloat16)
    clean = layer(x)
    for bad in (math.nan, math.inf):
        x2 = x.clone()
        x2[4, 50] = bad
        y, chosen, _ = layer(x2, return_choice=True)
        assert torch.isnan(y[4]).all() and torch.equal(y[:4], clean[:4]) and torch.equal(y[5], clean[5])
        assert ((chosen >= 0) & (chosen < 8)).all()


def test_experts_outputs_and_refusals(mx):
    router, gate_up, down, _ = layer_parts(64, 64, 4, "f16", False, 5)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2)
    x = torch.randn(2, 3, 64, generator=gen(3), device="cuda").to(torch.float16)
    y = layer(x)
    assert y.shape == (2, 3, 64) and layer(x[:0]).shape == (0, 3, 64)
    wide = torch.full((7, 80), 3.0, device="cuda", dtype=torch.float16)
    layer(x.view(6, 64), out=wide[:6, 1:65])
    assert torch.equal(wide[:6, 1:65], y.view(6, 64)) and (wide[6] == 3).all() and (wide[:, 65:] == 3).all() and (wide[:, 0] == 3).all()
    with pytest.raises(ValueError):
        layer(x.to(torch.bfloat16))
    with pytest.raises(ValueError):
        layer(x[..., :32])
    with pytest.raises(ValueError, match="at most 128"):
        layer(torch.zeros(129, 64, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="top_k"):
        mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 5)
    with pytest.raises(ValueError, match="down"):
        mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(gate_up), 2)
    with pytest.raises(ValueError, match="bias"):
        mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2, bias=torch.zeros(5, device="cuda"))


# ---- offsets past 32 bits ----------------------------------------------------------------------------

def test_quantize_past_32_bits(mx):
    """A matrix of more than 2^32 bytes and 2^31 values: its last rows, and rows a long way apart."""
    rows, k = 36000, 65536
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, k, generator=gen(1), device="cuda").to(torch.bfloat16)
    x[:2] = torch.randn(2, k, generator=gen(2), device="cuda").to(torch.bfloat16)
    x[2:-3] = 1.5
    q = mx.quantize(x)
    for part in (slice(0, 2), slice(rows - 3, rows)):
        want = mxref.values(*mxref.stored(x[part]), k)
        y = q.dequantize(torch.bfloat16)
        assert torch.equal(y[part].cpu(), want.to(torch.bfloat16)) and bool((y[3:-3:997] == 1.5).all())
        del y
    far = torch.empty_strided((2, 64), (2 ** 31 + 8, 1), dtype=torch.bfloat16, device="cuda")
    far.copy_(torch.randn(2, 64, generator=gen(3), device="cuda"))
    assert torch.equal(mx.quantize(far).dequantize().cpu(), mxref.values(*mxref.stored(far), 64).to(torch.bfloat16))


def test_products_past_32_bits(mx):
    """Outputs of more than 2^32 bytes, from either activations; the corners against the definition."""
    m, n, k = 60000, 40000, 64
    c, s = weights(n // 100, k, 3)
    w = mx.pack(c.repeat(100, 1).cuda(), s.repeat(100, 1).cuda())
    x = torch.randn(m, k, generator=gen(4), device="cuda").to(torch.bfloat16)
    wv = mxref.values(c, s, k)[-8:]
    for four in (True, False):
        y = mx.matmul(mx.quantize(x) if four else x, w)
        for rows in (slice(0, 4), slice(m - 4, m)):
            a = mxref.values(*mxref.stored(x[rows]), k) if four else x[rows].cpu().double()
            want = a @ wv.t()
            assert_within(y[rows, n - 8:], want, mxref.product_bound(a, wv, want, torch.bfloat16) + 1e-6)
        del y


# ---- streams, graphs, a run of them together -------------------------------------------------------

def block(mx, x, w_in, w_mid, layer):
    """A small network's step: a 16-bit product, a 4-bit product, the expert layer."""
    h = mx.matmul(x, w_in)
    h = mx.matmul(mx.quantize(h), w_mid, dtype=x.dtype)
    return layer(h)


def network(mx):
    router, gate_up, down, _ = layer_parts(160, 96, 12, "bf16", False, 8)
    return (mx.pack(*on_gpu(weights(192, 128, 1))), mx.pack(*on_gpu(weights(160, 192, 2))),
            mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 3))


def test_a_run_of_them_together(mx):
    parts = network(mx)
    x = torch.randn(10, 128, generator=gen(7), device="cuda").to(torch.bfloat16)
    w1, w2 = weights(192, 128, 1), weights(160, 192, 2)
    h1 = mx.matmul(x, parts[0])
    a = mxref.values(*mxref.stored(h1), 192)
    want = a @ mxref.values(*w2, 192).t()
    h2 = mx.matmul(mx.quantize(h1), parts[1], dtype=x.dtype)
    assert_within(h2, want, mxref.product_bound(a, mxref.values(*w2, 192), want, x.dtype))
    assert_within(h1, x.cpu().double() @ mxref.values(*w1, 128).t(),
                  mxref.product_bound(x.cpu().double(), mxref.values(*w1, 128), x.cpu().double() @ mxref.values(*w1, 128).t(), x.dtype) + 1e-5)
    assert torch.equal(block(mx, x, *parts), parts[2](h2))
    mx.check()


def test_captured_graphs_replay_on_new_inputs(mx):
    parts = network(mx)
    x = torch.randn(10, 128, generator=gen(7), device="cuda").to(torch.bfloat16)
    x2 = torch.randn(10, 128, generator=gen(8), device="cuda").to(torch.bfloat16)
    want = [block(mx, v, *parts).clone() for v in (x, x2)]
    graphs = []
    for _ in range(2):  # two graphs, to be replayed at the same time
        static = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(mx, static, *parts)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = block(mx, static, *parts)
        graphs.append((g, static, y))
    graphs[1][1].copy_(x2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, _, y), w in zip(graphs, want):
        assert torch.equal(y, w)
    mx.check()


def test_calls_on_two_streams_at_once(mx):
    parts = network(mx)
    xs = [torch.randn(12, 128, generator=gen(20 + i), device="cuda").to(torch.bfloat16) for i in range(4)]
    want = [block(mx, x, *parts).clone() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(block(mx, xs[i], *parts))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(v, w) for v in g)


def test_calls_from_two_threads(mx):
    import threading
    parts = network(mx)
    x = torch.randn(12, 128, generator=gen(30), device="cuda").to(torch.bfloat16)
    want = block(mx, x, *parts)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                if not torch.equal(block(mx, x, *parts), want):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_experts_workspace_contents_do_not_matter(mx, native):
    router, gate_up, down, _ = layer_parts(200, 136, 6, "bf16", False, 2)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 3)
    x = torch.randn(5, 200, generator=gen(2), device="cuda").to(torch.bfloat16)
    want = layer(x)
    need = native.ug_mx4_experts_workspace(C.byref(layer._layer), 5)
    for fill in (0, 255, 127):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device="cuda")
        y = torch.empty_like(x)
        torch.cuda.synchronize()
        rc = native.ug_mx4_experts(C.byref(layer._layer), x.data_ptr(), 200, 5, y.data_ptr(), 200, None, None, ws.data_ptr(),
                                   need, None)
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(y, want) and (ws[need:] == fill).all()


def test_product_workspace_contents_do_not_matter(mx, native):
    W = mx.pack(*on_gpu(weights(130, 200, 2)))
    x = torch.randn(25, 200, generator=gen(2), device="cuda").to(torch.float16)
    want = mx.matmul(x, W)
    need = native.ug_mx4_matmul_x16_workspace(25, 200, 1)
    assert need
    for fill in (0, 255, 127):
        ws = torch.full((need + 4096,), fill, dtype=torch.uint8, device="cuda")
        y = torch.empty(25, 130, device="cuda", dtype=torch.float16)
        torch.cuda.synchronize()
        rc = native.ug_mx4_matmul_x16(x.data_ptr(), 1, 200, 25, W.codes.data_ptr(), W.scales.data_ptr(), 130, 200, y.data_ptr(), 1,
                                      130, ws.data_ptr(), need, None)
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(y, want) and (ws[need:] == fill).all()


def test_more_rows_or_values_than_32_bits_count_are_refused(mx):
    one = torch.ones(1, device="cuda", dtype=torch.bfloat16)
    W = mx.quantize(one.view(1, 1))
    for tall in (one.expand(2 ** 32 + 1, 1), one.expand(1, 2 ** 32 + 32), one.expand(2 ** 31, 1)):
        with pytest.raises(ValueError, match="at most"):
            mx.quantize(tall, layout="stored")
        with pytest.raises(ValueError, match="at most"):
            mx.matmul(tall, W)
    byte = torch.zeros(1, device="cuda", dtype=torch.uint8)
    with pytest.raises(ValueError, match="at most"):
        mx.MX4(byte, byte, 2 ** 32 + 1, 1, layout="stored")
    with pytest.raises(ValueError, match="at most"):
        mx.pack(byte.expand(2 ** 32 + 1, 1), byte.expand(2 ** 32 + 1, 1), k=1)


def test_copies_have_bytes_of_their_own(mx):
    import copy
    import pickle
    x = torch.randn(5, 96, generator=gen(1), device="cuda").to(torch.bfloat16)
    W = mx.quantize(torch.randn(70, 96, generator=gen(2), device="cuda"))
    router, gate_up, down, bias = layer_parts(96, 64, 8, "bf16", True, 5)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2, normalize=False, bias=bias.cuda())
    want = mx.matmul(x, W), layer(x)
    copies = [(copy.deepcopy(W), copy.deepcopy(layer)), pickle.loads(pickle.dumps((W, layer))), (copy.copy(W), copy.copy(layer))]
    for w, other in copies[:2]:
        assert w._codes != W._codes and other._layer.down_codes != layer._layer.down_codes
    del W, layer, w, other
    filler = [torch.full((1 << 16,), 255, device="cuda", dtype=torch.uint8) for _ in range(64)]   # what was freed is written over
    for w, other in copies:
        assert torch.equal(mx.matmul(x, w), want[0]) and torch.equal(other(x), want[1])
    del filler


def test_an_experts_layer_keeps_its_tensors(mx):
    router, gate_up, down, _ = layer_parts(96, 64, 8, "bf16", False, 5)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2)
    x = torch.randn(5, 96, generator=gen(1), device="cuda").to(torch.bfloat16)
    want = layer(x)
    layer.router = layer.gate_up = layer.down = None
    filler = [torch.full((1 << 16,), 255, device="cuda", dtype=torch.uint8) for _ in range(64)]
    assert torch.equal(layer(x), want)
    del filler


def test_split_products_on_many_streams(mx):
    """Short products over clusters whose CTAs share SMs: every one of them gets its tensor memory."""
    cases = []
    for i, (m, n, k, four) in enumerate([(1, 8192, 512, False), (16, 4096, 1024, True), (9, 2048, 1024, False), (32, 1024, 2048, True),
                                         (3, 8192, 768, False), (20, 8192, 1024, True)]):
        W = mx.pack(*on_gpu(weights(n, k, 40 + i)))
        x = torch.randn(m, k, generator=gen(40 + i), device="cuda").to(torch.bfloat16)
        a = mx.quantize(x) if four else x
        cases.append((a, W, mx.matmul(a, W)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(12)]
    got = []
    for _ in range(20):
        for i, s in enumerate(streams):
            a, W, want = cases[i % len(cases)]
            with torch.cuda.stream(s):
                got.append((mx.matmul(a, W), want))
    torch.cuda.synchronize()
    mx.check()
    assert all(torch.equal(y, want) for y, want in got)


@pytest.mark.parametrize("t,d,f,e,top,norm,name,with_bias", [
    # of gate and up
    (8, 130, 1000, 20, 4, True, "bf16", False), (1, 100, 1300, 16, 16, False, "f16", True), (90, 256, 4500, 6, 2, True, "bf16", True),
    # of down: added there, and after it
    (8, 2000, 130, 20, 4, True, "bf16", False), (40, 2600, 70, 16, 3, True, "f16", False),
    # of both
    (128, 640, 420, 64, 4, False, "bf16", False)])
def test_experts_with_more_tiles_than_ctas(mx, t, d, f, e, top, norm, name, with_bias):
    """Every CTA takes several tiles, and goes on from one expert to the next."""
    test_experts(mx, t, d, f, e, top, norm, name, with_bias)


WHOLE = [  # tokens, d, f, experts, experts of every token, type
    (1, 64, 70, 4, 1, "f16"), (1, 2048, 1024, 8, 4, "bf16"), (7, 1447, 999, 12, 2, "f16"), (5, 300, 1500, 3, 1, "bf16"), (40, 520, 260, 2, 2, "f16"),
    (128, 200, 136, 4, 2, "bf16"), (100, 333, 40, 2, 1, "f16"), (64, 640, 420, 64, 16, "bf16"),
    # long rows: K spread over a cluster
    (3, 16384, 64, 2, 2, "bf16"), (2, 40, 16384, 2, 1, "f16"), (33, 4200, 70, 2, 1, "f16"), (9, 300, 4300, 2, 2, "bf16"),
    # several tiles to a CTA, from one expert on to the next
    (8, 130, 1000, 20, 16, "bf16"), (90, 256, 4500, 2, 1, "f16"), (40, 2600, 70, 16, 16, "f16"),
    # 24 tokens of an expert to a CTA: one to a tile, several tiles, dealt out
    (44, 520, 260, 2, 1, "f16"), (48, 1447, 999, 4, 2, "bf16"), (128, 130, 1000, 6, 1, "f16"), (72, 2000, 4000, 4, 1, "bf16")]


@pytest.mark.parametrize("t,d,f,e,top,name", WHOLE)
def test_experts_of_exact_gate_and_up_sums(mx, t, d, f, e, top, name):
    """Nothing but SiLU, the pieces of the hidden vector and the last rounding is off: a lost stage, a share of a cluster's
    or a piece too few would show (test_the_bound_of_whole_layers_sees_faults)."""
    make, gate_up, down = mxref.whole_layer(d, f, e, t + d + f)
    x, dtype = make(t), mxref.TYPES[name]
    layer = mx.Experts(torch.zeros(e, d, device="cuda", dtype=dtype), on_gpu(gate_up), on_gpu(down), top)
    y, chosen, p = layer(x.to(dtype).cuda(), return_choice=True)
    assert (chosen.cpu() == torch.arange(top)).all() and (p == 1 / top).all()   # equal logits: the lowest, alike
    want, bound = mxref.whole_experts(x, chosen.cpu().long(), gate_up, down)
    off = mxref.rounding_off(y, want, bound, dtype)
    assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.numel()}, worst {float(off.max()):.3g} half steps"
    mx.check()


@pytest.mark.parametrize("t,d,f,e,name", [(50, 700, 333, 9, "f16"), (128, 1000, 200, 40, "bf16"), (9, 2048, 1024, 32, "bf16")])
def test_experts_of_exact_sums_each_token_its_own(mx, t, d, f, e, name):
    """One expert to a token, whichever its router takes: its weight is 1."""
    make, gate_up, down = mxref.whole_layer(d, f, e, t + d + f)
    x, dtype = make(t), mxref.TYPES[name]
    router = (torch.randn(e, d, generator=gen(t), device="cuda") / math.sqrt(d)).to(dtype)
    y, chosen, p = mx.Experts(router, on_gpu(gate_up), on_gpu(down), 1)(x.to(dtype).cuda(), return_choice=True)
    assert (p == 1).all() and len(chosen.unique()) > 4
    want, bound = mxref.whole_experts(x, chosen.cpu().long(), gate_up, down)
    assert not (mxref.rounding_off(y, want, bound, dtype) > 0).any()


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("e,top,bad", [(9, 2, (5,)), (200, 16, (0, 33, 199)), (3, 3, (1,)), (40, 1, (39, 7))])
def test_a_nan_logit_is_chosen_and_makes_the_output_nan(mx, e, top, bad, name, norm):
    """As torch.sort orders them: a NaN before every number, equal ones by index. A damaged router shows in both modes."""
    router, gate_up, down, bias = layer_parts(96, 64, e, name, True, 5)
    x = torch.randn(6, 96, generator=gen(3), device="cuda").to(mxref.TYPES[name])
    clean = x.cpu().double() @ router.double().t() + bias.double()
    for broken in ("router", "bias"):
        r, b = router.clone(), bias.clone()
        if broken == "router":
            r[list(bad), 50] = math.nan
        else:
            b[list(bad)] = math.nan
        y, chosen, p = mx.Experts(r.cuda(), on_gpu(gate_up), on_gpu(down), top, norm, b.cuda())(x, return_choice=True)
        assert torch.isnan(y).all() and torch.isnan(p).all()
        order, _ = mxref.select(torch.where(torch.isin(torch.arange(e), torch.tensor(bad)), math.nan, clean), top, norm)
        first = min(len(bad), top)
        assert chosen[:, :first].tolist() == [sorted(bad)[:first]] * 6
        ok = distinct(x, router, bias, e)   # all of its logits apart
        assert torch.equal(chosen.cpu().long()[ok], order[ok]) and (ok.any() or e > 100)
        assert all(len(set(row)) == top and 0 <= min(row) and max(row) < e for row in chosen.tolist())


def test_forward_mode_tangents_are_refused(mx):
    from torch.autograd import forward_ad
    x = torch.randn(4, 96, generator=gen(1), device="cuda").to(torch.bfloat16)
    W = mx.quantize(torch.randn(70, 96, generator=gen(2), device="cuda"))
    router, gate_up, down, bias = layer_parts(96, 64, 8, "bf16", True, 5)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2)
    want = mx.matmul(x, W), layer(x), mx.quantize(x).dequantize()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        out = forward_ad.make_dual(torch.empty(4, 70, device="cuda", dtype=x.dtype), torch.ones(4, 70, device="cuda", dtype=x.dtype))
        for call in (lambda: mx.quantize(dual), lambda: mx.matmul(dual, W), lambda: layer(dual), lambda: mx.matmul(x, W, out=out),
                     lambda: mx.Experts(forward_ad.make_dual(router.cuda(), router.cuda()), on_gpu(gate_up), on_gpu(down), 2),
                     lambda: mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2, bias=forward_ad.make_dual(bias.cuda(), bias.cuda()))):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        for got, v in zip((mx.matmul(x, W), layer(x), mx.quantize(x).dequantize()), want):   # no tangent: as ever
            assert torch.equal(got, v)
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda v: mx.matmul(v, W), (x,), (x,))
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.vmap(lambda v: mx.matmul(v, W))(x)


def test_a_product_of_the_most_4_bit_rows(mx):
    """2^21 rows of 32,768 values, 34 GB of codes, of which the first and the last tile are looked at."""
    m, n, k = 2 ** 21, 40, 32768
    codes = torch.zeros(m // 2 * k, dtype=torch.uint8, device="cuda")
    scales = torch.full((m * k // 32,), 127, dtype=torch.uint8, device="cuda")
    a, w = whole(128, k, 1, True), whole(n, k, 2, False)
    tile = mx.pack(*on_gpu(a))
    for part in (slice(0, len(tile.codes)), slice(-len(tile.codes), None)):
        codes[part] = tile.codes
    for part in (slice(0, len(tile.scales)), slice(-len(tile.scales), None)):
        scales[part] = tile.scales
    y = mx.matmul(mx.MX4(codes, scales, m, k), mx.pack(*on_gpu(w)), dtype=torch.float32)
    want = mxref.values(*a, k) @ mxref.values(*w, k).t()   # multiples of 1/4 below 2^22
    assert torch.equal(y[:128].cpu().double(), want) and torch.equal(y[-128:].cpu().double(), want)
    assert not y[128:-128].any()
    del codes, scales, y
    big = torch.empty(1, dtype=torch.bfloat16, device="cuda")
    for rows, k in ((2 ** 21 + 1, 40), (2 ** 21 - 1, 65536)):   # refused before the rows would be copied (275 GB)
        with pytest.raises(ValueError, match="at most"):
            mx.matmul(big.expand(rows, k), mx.quantize(torch.zeros(1, k, device="cuda")))
    with pytest.raises(ValueError, match="65536"):
        mx.matmul(mx.quantize(torch.zeros(1, 65537, device="cuda")), mx.quantize(torch.zeros(1, 65537, device="cuda")))


def test_outputs_in_the_buffer_of_their_input(mx):
    W = mx.pack(*on_gpu(weights(50, 96, 4)))
    router, gate_up, down, _ = layer_parts(64, 64, 4, "f16", False, 5)
    layer = mx.Experts(router.cuda(), on_gpu(gate_up), on_gpu(down), 2)
    for m in (1, 6, 40, 300):
        buf = torch.randn(m, 200, generator=gen(m), device="cuda").to(torch.float16)
        was = buf.clone()
        mx.matmul(buf[:, 3:99], W, out=buf[:, 120:170])
        assert torch.equal(buf[:, 120:170], mx.matmul(was[:, 3:99], W))
        buf[:, 120:170] = was[:, 120:170]
        assert torch.equal(buf, was)
        if m <= 40:
            layer(buf[:, :64], out=buf[:, 64:128])
            assert torch.equal(buf[:, 64:128], layer(was[:, :64]))
            buf[:, 64:128] = was[:, 64:128]
            assert torch.equal(buf, was)
        with pytest.raises(ValueError, match="overlap"):
            mx.matmul(buf[:, 3:99], W, out=buf[:, 98:148])


@pytest.mark.parametrize("name,floor", [("bf16", 2.0 ** -21), ("f16", 2.0 ** -25)])
@pytest.mark.parametrize("m,n,k", [(1, 300, 256), (10, 130, 1000), (40, 200, 520), (1100, 2400, 256)])
def test_matmul_x16_beside_loud_values(mx, m, n, k, name, floor):
    """One value of 2^14 in every block, facing weights of zero: what the others keep is what the header says, for
    f16 2^-25 of the largest (its three pieces). The sum's own error is that of the pieces' magnitudes, which exceed the
    values' by half of the first piece's least step, 2^-17 of the largest, and less for each next one."""
    g = torch.Generator().manual_seed(m + k)
    x = 0.02 * torch.randn(m, k, generator=g)
    c, s = weights(n, k, n)
    w = mxref.values(c, s, k)
    loud = torch.arange(k) % 32 == 5
    x[:, loud] = 2.0 ** 14
    x = x.to(mxref.TYPES[name])
    codes = torch.stack((c & 15, c >> 4), -1).flatten(-2)[:, :k]
    codes[:, loud] = 0
    codes = torch.nn.functional.pad(codes, (0, k % 2))
    w = w * ~loud
    W = mx.pack((codes[:, 0::2] | codes[:, 1::2] << 4).cuda(), s.cuda(), k=k)
    a = x.double() * ~loud
    largest = 2.0 ** 14 * (torch.arange(k) // 32 * 32 + 5 < k)
    want = a @ w.t()
    held = largest[None].double() @ w.abs().t()
    bound = floor * held + mxref._sum_error(k) * (a.abs() @ w.abs().t() + 2.0 ** -16 * held)
    for dtype in (torch.float32, mxref.TYPES[name]):
        assert_within(mx.matmul(x.cuda(), W, dtype=dtype), want, bound + mxref.half_step(want.abs() + bound, dtype), str(dtype))


def test_experts_past_32_bits(mx):
    """256 experts of 8.6 GB of gate and up codes: the first and the last two, chosen by the bias."""
    d, f, e = 8192, 4096, 256
    make, gate_up, down = mxref.whole_layer(d, f, 3, 1)
    at = [0, 254, 255]
    parts = []
    for small in (gate_up, down):
        wide = tuple(torch.zeros(e, *t.shape[1:], dtype=torch.uint8, device="cuda") for t in small)
        for to, t in zip(wide, small):
            to[at] = t.cuda()
        parts.append(wide)
    bias = torch.full((e,), -math.inf)
    router = torch.zeros(e, d, dtype=torch.bfloat16, device="cuda")
    x = make(9)
    for chosen in ((0, 2), (1, 2)):
        b = bias.clone()
        b[[at[i] for i in chosen]] = 1.0
        layer = mx.Experts(router, *parts, 2, bias=b.cuda())
        y, got, _ = layer(x.to(torch.bfloat16).cuda(), return_choice=True)
        assert got.tolist() == [[at[i] for i in chosen]] * 9
        want, bound = mxref.whole_experts(x, torch.tensor([chosen] * 9), gate_up, down)
        assert not (mxref.rounding_off(y, want, bound, torch.bfloat16) > 0).any()
        del layer


def test_captured_forks_copies_and_joins(mx):
    """A graph whose branches meet in a call, with copies and fills as the nodes before the kernels."""
    parts = network(mx)
    router, gate_up, down, _ = layer_parts(160, 96, 12, "bf16", False, 8)
    other = mx.Experts(router.cuda().flip(0), on_gpu(gate_up), on_gpu(down), 2)
    x = torch.randn(10, 128, generator=gen(7), device="cuda").to(torch.bfloat16)

    def run(v, side):
        a = v.clone()                      # a copy before a product
        h = mx.matmul(a, parts[0])
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):      # one branch
            q = mx.quantize(h)
            one = mx.matmul(q, parts[1], dtype=v.dtype)
            left = parts[2](one)
        two = torch.zeros(10, 160, device="cuda", dtype=v.dtype)
        mx.matmul(h, parts[1], out=two)    # the other, after a fill
        right = other(two)
        here.wait_stream(side)
        both = torch.empty(20, 160, device="cuda", dtype=v.dtype)
        mx.matmul(h, parts[1], out=both[:10])
        both[10:] = left + right
        return other(both), left, right

    want = [t.clone() for t in run(x, torch.cuda.Stream())]
    torch.cuda.synchronize()
    static, side, g = x.clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(static, side)
    for _ in range(20):
        [t.fill_(math.nan) for t in got]
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    mx.check()


def test_the_first_calls_of_a_process_may_be_captured(mx):
    """No call needs one before it: a fresh process whose first calls are captured."""
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = %r
import torch
from unoq_dsp import mx
w = torch.randn(192, 128, device="cuda")
x = torch.randn(24, 128, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
def run():
    q = mx.quantize(w)
    return mx.matmul(x, q), mx.matmul(mx.quantize(x), q), mx.matmul(x[:3], q), q.dequantize()
with torch.cuda.graph(g):
    got = run()
g.replay()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
mx.check()
print("captured")
""" % [p for p in sys.path if p]
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=200)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 130, 65536), (2, 300, 40000), (4, 200, 8193), (5, 200, 8193), (9, 130, 5000), (6, 2100, 16384), (3, 1, 30000)])
def test_matmul_x16_few_tokens_of_long_rows(mx, m, n, k, name):
    """Around the change from pieces made in the product to those made before it."""
    test_matmul_x16_exact(mx, m, n, k, name)
    test_matmul_x16(mx, m, n, k, name)
