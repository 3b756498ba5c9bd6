"""CPU: the MX4 operators' host side (include/unoq_mx.h, unoq_dsp.mx): sizes, refusals in their order
before any device is touched, and the oracle's own format checks."""
import ctypes as C

import pytest
import torch

import mxref

P = 1 << 20  # a well-aligned address that is never followed: every call here is refused first


def test_sizes(native):
    assert native.ug_mx4_codes_bytes(0, 5, 33) == 5 * 17 and native.ug_mx4_scales_bytes(0, 5, 33) == 10
    assert native.ug_mx4_codes_bytes(1, 129, 257) == 4 * 16384 and native.ug_mx4_scales_bytes(1, 129, 257) == 8 * 512
    assert native.ug_mx4_codes_bytes(1, 128, 1) == 16384 and native.ug_mx4_scales_bytes(1, 1, 256) == 1024
    assert native.ug_mx4_codes_bytes(2, 5, 33) == 0 and native.ug_mx4_scales_bytes(-1, 5, 33) == 0
    assert native.ug_mx4_codes_bytes(1, 2 ** 32 - 1, 128) == 2 ** 25 * 16384  # past 32 bits
    assert native.ug_mx4_pack_rows(3, 130, 0) == 3 * 256 and native.ug_mx4_pack_rows(3, 130, 1) == 3 * 256
    assert native.ug_mx4_pack_rows(2, 260, 1) == 2 * 384 and native.ug_mx4_pack_rows(2, 128, 1) == 256
    assert native.ug_mx4_pack_rows(2 ** 31, 130, 0) == 0  # does not fit
    assert native.ug_mx4_matmul_x16_workspace(3, 100, 0) == 0
    assert native.ug_mx4_matmul_x16_workspace(40, 100, 2) >= 80 * 128 + 512
    assert native.ug_mx4_matmul_x16_workspace(16, 100, 2) == 0 and native.ug_mx4_matmul_x16_workspace(17, 100, 2) > 0
    assert native.ug_mx4_matmul_x16_workspace(10, 100, 1) == 0 and native.ug_mx4_matmul_x16_workspace(11, 100, 1) > 0


def test_quantize_refusals(native):
    q = native.ug_mx4_quantize
    assert q(P, 3, 1, 32, 32, 0, P, P, None) == 18       # type
    assert q(P, 0, 1, 32, 32, 2, P, P, None) == 18       # layout
    assert q(P, 0, 1, 0, 32, 0, P, P, None) == 18        # k
    assert q(P, 0, 1, 32, 31, 0, P, P, None) == 18       # rows overlap
    assert q(P, 0, 2 ** 31, 256, 256, 1, P, P, None) == 18
    assert q(None, 0, 1, 32, 32, 0, P, P, None) == 22
    assert q(P, 0, 1, 32, 32, 0, None, P, None) == 22
    assert q(P + 2, 0, 1, 32, 32, 0, P, P, None) == 22   # x misaligned for its type
    assert q(P, 0, 1, 32, 32, 1, P + 64, P, None) == 22  # operand codes misaligned
    assert q(P, 0, 1, 32, 32, 1, P, P + 8, None) == 22
    assert q(None, 0, 0, 32, 32, 0, None, None, None) == 0  # zero rows do nothing
    assert native.ug_last_error()


def test_dequantize_and_pack_refusals(native):
    dq, pk = native.ug_mx4_dequantize, native.ug_mx4_pack
    assert dq(P, P, 5, 1, 32, P, 0, 32, None) == 18
    assert dq(P, P, 0, 1, 32, P, 9, 32, None) == 18
    assert dq(P, P, 0, 1, 32, P, 0, 5, None) == 18
    assert dq(P, None, 0, 1, 32, P, 0, 32, None) == 22
    assert dq(P, P, 0, 1, 32, P + 1, 1, 32, None) == 22
    assert dq(None, None, 0, 0, 32, None, 0, 32, None) == 0
    assert pk(P, P, 1, 3, 32, 1, P, P, None) == 18   # odd rows do not pair
    assert pk(P, P, 1, 4, 32, 2, P, P, None) == 18
    assert pk(P, P, 1, 4, 0, 0, P, P, None) == 18
    assert pk(P, P, 2 ** 31, 130, 32, 0, P, P, None) == 18
    assert pk(P, None, 1, 4, 32, 0, P, P, None) == 22
    assert pk(P, P, 1, 4, 32, 0, P + 16, P, None) == 22
    assert pk(None, None, 0, 4, 32, 0, None, None, None) == 0


def test_product_refusals(native):
    mm, mx = native.ug_mx4_matmul, native.ug_mx4_matmul_x16
    assert mm(P, P, 1, P, P, 8, 32, P, 4, 8, None) == 18
    assert mm(P, P, 1, P, P, 8, 0, P, 0, 8, None) == 18
    assert mm(P, P, 1, P, P, 8, 65537, P, 0, 8, None) == 18
    assert mm(P, P, 1, P, P, 8, 32, P, 0, 7, None) == 18
    assert mm(None, P, 1, P, P, 8, 32, P, 0, 8, None) == 22
    assert mm(P, P, 1, None, P, 8, 32, P, 0, 8, None) == 22
    assert mm(P, P, 1, P + 8, P, 8, 32, P, 0, 8, None) == 22
    assert mm(P, P, 1, P, P, 8, 32, P + 2, 0, 8, None) == 22
    assert mm(None, None, 0, None, None, 8, 32, None, 0, 8, None) == 0
    need = native.ug_mx4_matmul_x16_workspace(64, 32, 2)
    assert mx(P, 0, 32, 64, P, P, 8, 32, P, 0, 8, P, need, None) == 18   # 32-bit x
    assert mx(P, 2, 31, 64, P, P, 8, 32, P, 0, 8, P, need, None) == 18
    assert mx(P, 2, 32, 64, P, P, 8, 32, P, 0, 8, P, need - 1, None) == 22
    assert mx(P, 2, 32, 64, P, P, 8, 32, P, 0, 8, P + 16, need, None) == 22
    assert mx(P, 2, 32, 64, P, P, 8, 32, P, 0, 8, None, need, None) == 22
    assert mx(P + 1, 2, 32, 64, P, P, 8, 32, P, 0, 8, P, need, None) == 22
    assert mx(P + 1, 2, 32, 1, P, P, 8, 32, P, 0, 8, None, 0, None) == 22
    assert mx(None, 2, 32, 0, None, None, 8, 32, None, 0, 8, None, 0, None) == 0


def _layer(**other):
    from unoq_dsp.mx import UgMx4Experts
    fields = dict(experts=8, top_k=2, d=64, f=64, normalize=1, type=2, router=P, bias=None, gate_up_codes=P,
                  gate_up_scales=P, down_codes=P, down_scales=P)
    fields.update(other)
    return UgMx4Experts(**fields)


def test_experts_refusals(native):
    size, run = native.ug_mx4_experts_workspace, native.ug_mx4_experts

    def call(layer, x=P, xs=64, t=1, y=P, ys=64, ws=P, n=1 << 30):
        return run(C.byref(layer), x, xs, t, y, ys, None, None, ws, n, None)

    assert size(C.byref(_layer()), 4) > 0
    for bad in (dict(experts=0), dict(experts=257), dict(top_k=0), dict(top_k=9), dict(experts=32, top_k=17), dict(d=0),
                dict(d=16385), dict(f=0), dict(f=16385), dict(type=0)):
        assert size(C.byref(_layer(**bad)), 4) == 0 and call(_layer(**bad)) == 18, bad
    assert size(C.byref(_layer()), 129) == 0 and call(_layer(), t=129) == 18
    assert call(_layer(), xs=63) == 18 and call(_layer(), ys=63) == 18
    assert call(_layer(), x=None) == 22 and call(_layer(), y=None) == 22 and call(_layer(), ws=None) == 22
    assert call(_layer(router=None)) == 22 and call(_layer(down_scales=None)) == 22
    assert call(_layer(bias=P + 2)) == 22 and call(_layer(gate_up_codes=P + 64)) == 22 and call(_layer(), x=P + 1) == 22
    assert call(_layer(), ws=P + 128) == 22
    need = size(C.byref(_layer()), 1)
    assert call(_layer(), n=need - 1) == 22
    assert call(_layer(), t=0, x=None) == 0
    assert run(None, P, 64, 1, P, 64, None, None, P, 1 << 30, None) == 22


def test_no_device_is_an_error(native):
    if torch.cuda.is_available():
        pytest.skip("a device is here")
    assert native.ug_mx4_quantize(P, 0, 1, 32, 32, 0, P, P, None) == 2002
    assert native.ug_mx4_check(0) == 2002


def test_python_refuses_host_tensors():
    from unoq_dsp import mx
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        mx.quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        mx.pack(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="MX4"):
        mx.matmul(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        mx.Experts(torch.zeros(4, 64, dtype=torch.bfloat16), (x, x), (x, x), 2)


@pytest.mark.parametrize("k", [1, 31, 32, 33, 77])
def test_oracle_stored_form(k):
    """The oracle's values are the nearest grid points: off by at most half the spacing of their binade."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(9, k, generator=g) * torch.exp(3 * torch.randn(9, 1, generator=g))
    x[0] = 0
    v = mxref.values(*mxref.stored(x), k)
    for at in range(0, k, 32):
        b, w = x[:, at:at + 32].double(), v[:, at:at + 32]
        top = b.abs().amax(1, keepdim=True)
        assert ((w - b).abs() <= top / 4 + 1e-300).all()       # top is in [4, 8) scales: off by 1, or by 2 past 6
        small = b.abs() <= top / 4
        assert ((w - b).abs()[small] <= (top / 16).expand_as(b)[small]).all()  # under 2 scales: off by a quarter


def _held(h, pieces):
    """h as so many e4m3 pieces hold it, by its definition: a scale per 32, each piece 16 times finer than the one before."""
    rows, f = h.shape
    b = torch.nn.functional.pad(h, (0, -f % 32)).reshape(rows, -1, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    left = torch.ldexp(b, 8 - e)
    total, unit = torch.zeros_like(left), 1.0
    for _ in range(pieces):
        piece = left.float().to(torch.float8_e4m3fn).double()
        total += piece * unit
        left, unit = (left - piece) * 16, unit / 16
    return torch.ldexp(total, e - 8).reshape(rows, -1)[:, :f]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,f", [(64, 70), (300, 1500), (4200, 64), (16384, 64)])
def test_the_bound_of_whole_layers_sees_faults(d, f, dtype):
    """What a kernel could do wrong falls outside of the bound; the layer as it is documented does not."""
    make, gate_up, down = mxref.whole_layer(d, f, 2, d + f)
    x = make(9)
    order = torch.tensor([[0, 1]]).expand(9, 2)
    want, bound = mxref.whole_experts(x, order, gate_up, down)

    def layer(change_h=lambda h: h, change_x=lambda x: x):
        parts = [change_h(mxref.hidden64(change_x(x), gate_up, e, f)) @ mxref.values(down[0][e], down[1][e], f).t() for e in (0, 1)]
        return (sum(parts) / 2).to(dtype)

    def outside(y):
        return int((mxref.rounding_off(y, want, bound, dtype) > 0).sum())

    def without(step):   # 128 values of K, as a lost stage
        def cut(x):
            x = x.clone()
            x[:, step * 128:step * 128 + 128] = 0
            return x
        return cut

    assert outside(layer()) == 0 and outside(layer(lambda h: _held(h, 4))) == 0
    assert outside(layer(lambda h: _held(h, 3))) > 0          # 14 bits
    assert outside(layer(lambda h: _held(h, 2))) > want.numel() / 16
    assert outside(torch.zeros_like(want)) > want.numel() * 0.9
    assert outside(layer(change_x=without((d - 1) // 128))) > want.numel() * 0.5
    assert outside(layer(lambda h: torch.cat((h[:, :-32], torch.zeros_like(h[:, -32:])), 1))) > 0   # a lost block


def test_the_bound_of_whole_layers_rests_on_exact_sums():
    for d in (1, 64, 16384):
        make, gate_up, _ = mxref.whole_layer(d, 4, 1, d)
        unit = 2.0 ** (int(gate_up[1].min()) - 128)
        size = make(8).abs() @ mxref.values(gate_up[0][0], gate_up[1][0], d).abs().t() / unit
        assert (size == size.round()).all() and float(size.max()) < 2 ** 24
    h = torch.randn(50, 320, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    h = h * torch.exp(2 * torch.randn(h.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64))
    top = h.abs().reshape(50, 10, 32).amax(-1).repeat_interleave(32, -1)
    for pieces in (1, 2, 3, 4, 5):
        off = (_held(h, pieces) - h).abs()
        assert (off <= torch.maximum(h.abs() * 2.0 ** (1 - 5 * pieces), top * 2.0 ** (-13 - 4 * pieces))).all()


def test_python_refuses_gradients_and_tangents():
    from torch.autograd import forward_ad

    from unoq_dsp import mx
    x = torch.ones(2, 3)
    mx._refuse_gradient(x, "x")
    with pytest.raises(ValueError, match="x needs a gradient"):
        mx._refuse_gradient(x.clone().requires_grad_(), "x")
    with torch.no_grad():
        mx._refuse_gradient(x.clone().requires_grad_(), "x")
    with forward_ad.dual_level():
        mx._refuse_gradient(x, "x")
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="x carries a tangent"):
                mx._refuse_gradient(dual, "x")
        mx._refuse_gradient(forward_ad.unpack_dual(dual).primal, "x")
    seen = []

    def inside(v):
        with pytest.raises(ValueError, match="tangent"):
            mx._refuse_gradient(v, "x")
        seen.append(1)
        return v

    torch.func.jvp(inside, (x,), (x,))
    assert seen == [1]


def test_a_layer_is_on_the_device_of_its_tensors(native):
    """As loading with tensors mapped to another device leaves it: the state names the old one, the tensors are elsewhere."""
    import copy

    from unoq_dsp import mx
    layer = mx.Experts.__new__(mx.Experts)
    state = dict(router=torch.zeros(2, 64, dtype=torch.bfloat16), bias=None, top_k=1, d=64, f=64, experts=2, normalize=True,
                 device=torch.device("cuda", 1), gate_up=[torch.zeros(1, dtype=torch.uint8)] * 2,
                 down=[torch.zeros(1, dtype=torch.uint8)] * 2)
    layer.__setstate__(state)
    assert layer.device == torch.device("cpu") and copy.copy(layer).device == layer.device
    with pytest.raises(ValueError, match="CUDA"):
        layer(torch.zeros(1, 64, dtype=torch.bfloat16))


def _edge(fits, lo, hi):
    """The largest size in [lo, hi) that fits, hi not fitting."""
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if fits(mid) else (lo, mid)
    return lo


def test_the_documented_limits_and_no_nearer_ones(native):
    """Both sides of every joint limit, in C (18: too large; 22: the null pointer that is looked at next) and in Python."""
    from unoq_dsp import mx

    def python_takes(call, *args):
        try:
            call(*args)
            return True
        except ValueError as e:
            assert "at most" in str(e)
            return False

    for k in (1, 256, 257, 5000, 65536, 2 ** 30):
        tiles = 2 * -(-k // 256)
        rows = (2 ** 31 - 1) // tiles
        for fit, r in ((True, rows), (False, rows + 1)):
            want = 22 if fit else 18
            assert native.ug_mx4_quantize(None, 0, r, k, k, 0, None, None, None) == want
            assert native.ug_mx4_dequantize(None, None, 1, r, k, None, 0, k, None) == want
            assert python_takes(mx._fits, r, k, "x") == fit
        assert native.ug_mx4_quantize(None, 0, 1, 2 ** 30 + 1, 2 ** 30 + 1, 0, None, None, None) == 18
        whole = rows // 128 * 128   # pack counts whole tiles
        if whole:
            assert native.ug_mx4_pack(None, None, 1, whole, k, 0, None, None, None) == 22
        assert native.ug_mx4_pack(None, None, 1, whole + 1, k, 0, None, None, None) == 18
    for k in (1, 256, 5000, 32768, 65536):
        tiles = 2 * -(-k // 256)
        most = (2 ** 31 - 1) // tiles
        for pieces, m in ((False, min(most - 255, 2 ** 21)), (True, min((most - 256) // 4, 2 ** 21))):
            for fit, rows, cols in ((True, m, most - 127), (False, m + 1, 1), (False, 1, most - 126)):
                want = 22 if fit else 18
                if pieces:
                    got = native.ug_mx4_matmul_x16(P, 2, k, rows, None, None, cols, k, None, 0, cols, P, 1 << 62, None)
                else:
                    got = native.ug_mx4_matmul(P, P, rows, None, None, cols, k, None, 0, cols, None)
                assert got == want, (k, rows, cols)
                assert python_takes(mx._product_fits, rows, cols, k, pieces) == fit
    assert native.ug_mx4_matmul(P, P, 2 ** 21, P, P, 8, 65537, P, 0, 8, None) == 18
    # what the Python calls look at first lets nothing past
    for k in (1, 100, 256, 257, 65536, 2 ** 30):
        assert _edge(lambda r: python_takes(mx._fits, r, k, "x"), 0, 2 ** 40) >= (2 ** 38 - 1) // (k + 255)
    for m, n in ((0, 2 ** 21 - 1), (2 ** 19 - 1, 3)):
        assert 4 * m + n < 2 ** 21 and python_takes(mx._product_fits, m, n, 65536, True)


def test_outputs_beside_inputs_in_one_buffer():
    """An output overlaps an input where they share a byte, not where only their extents cross."""
    from unoq_dsp import mx
    buf = torch.zeros(12, 40, dtype=torch.bfloat16)
    flat = buf.view(-1)

    def takes(out, x):
        shared = {out.data_ptr() + 2 * (i * out.stride(0) + j) for i in range(out.shape[0]) for j in range(out.shape[1])} & \
            {x.data_ptr() + 2 * (i * x.stride(0) + j) for i in range(x.shape[0]) for j in range(x.shape[1])}
        try:
            mx._output(out, out.shape, out.dtype, out.device, (x,))
            return True, not shared
        except ValueError as e:
            assert "overlap" in str(e)
            return False, not shared

    for lo, hi in ((0, 20), (20, 40), (21, 40), (19, 40), (5, 6), (39, 40), (0, 40)):
        for rows in (slice(0, 12), slice(1, 12), slice(3, 4)):
            took, apart = takes(buf[rows, lo:hi], buf[:, :20])
            assert took == apart, (lo, hi, rows)
    assert takes(buf[0::2], buf[1::2]) == (True, True) and takes(buf[0::2], buf[2::2]) == (False, False)
    assert takes(buf[3:4, 20:], buf[:, :20]) == (True, True) and takes(buf[:, 20:], buf[5:6, :20]) == (True, True)
    assert takes(buf[3:4], buf[4:5]) == (True, True)
    # a row that reaches round the end of the other's: the last one's, and the next one's first
    assert takes(flat[20:20 + 11 * 40].view(11, 40)[:, :30], buf[:, :20]) == (False, False)
    other = torch.as_strided(flat, (8, 4), (50, 1), 20)   # rows of another distance: their extents decide
    assert takes(other, buf[:, :20])[0] is False
    for x in (flat[:40], buf[:1, :20]):
        assert takes(buf[1:], x.view(1, -1)) == (True, True)


def test_workspaces_of_few_rows(native):
    """Few rows are split into pieces inside the product and need none; the longer the rows, the fewer."""
    need = native.ug_mx4_matmul_x16_workspace
    for x_type, pieces in ((2, 2), (1, 3)):
        for k, columns in ((1, 32), (4096, 32), (4097, 15), (8192, 8), (16384, 4), (30000, 2), (65536, 1)):
            m = columns // pieces
            assert need(m, k, x_type) == 0 and need(m + 1, k, x_type) > 0
