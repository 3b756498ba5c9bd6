"""Microscaled 4-bit (MX4) operators on PyTorch tensors: quantise, product, expert layer.

The functions check their tensors, allocate the results (and a workspace of the call's own) with
PyTorch's allocator and launch the kernels of include/unoq_mx.h on the current stream of the
tensors' device, without waiting for it; all of them may be captured into a CUDA graph. They are
for inference: an input that needs a gradient is refused while gradients are recorded, and one that carries a
forward-mode tangent always. PyTorch is imported here only; the rest of the package does not need it.

    w = mx.quantize(weight)                      # (n, k) -> MX4, once
    y = mx.matmul(x, w)                          # 16-bit x, 4-bit weights (what x keeps: see matmul)
    y = mx.matmul(mx.quantize(x), w)             # both in 4 bits
    layer = mx.Experts(router, gate_up, down, top_k=4)
    y = layer(x)                                 # a few tokens through a mixture of experts
"""
import ctypes as C

import torch
from torch.autograd import forward_ad

from .errors import DSPError
from .native import last_error, load_library

STORED, OPERAND = 0, 1
MAX_TOKENS = 128
MAX_K = 65536            # of a product
MAX_ROWS = 2 ** 21       # of a product's activations
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_HALF = {t: _TYPES[t] for t in (torch.float16, torch.bfloat16)}


class UgMx4Experts(C.Structure):
    """include/unoq_mx.h UgMx4Experts."""
    _fields_ = [("experts", C.c_uint32), ("top_k", C.c_uint32), ("d", C.c_uint32), ("f", C.c_uint32),
                ("normalize", C.c_int), ("type", C.c_int), ("router", C.c_void_p), ("bias", C.c_void_p),
                ("gate_up_codes", C.c_void_p), ("gate_up_scales", C.c_void_p), ("down_codes", C.c_void_p),
                ("down_scales", C.c_void_p)]


_lib = None
_need = {}   # (m, k, type): workspace bytes of a product with 16-bit activations


def _library():
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


def _check(lib, rc, what):
    if rc:
        raise DSPError(f"{what} failed: {rc & 0xFFFFFFFF:#010x} {last_error(lib)}; no CPU fallback".rstrip())


def _stream(device):
    # the current stream's handle without building a Stream object (which costs as much as a launch)
    return torch._C._cuda_getCurrentRawStream(device.index)


def _input(x, what, types):
    """Refuse what the kernels do not take: other types and devices, gradients."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if x.dtype not in types:
        raise ValueError(f"{what} must be one of {', '.join(str(t) for t in types)}, not {x.dtype}")
    _refuse_gradient(x, what)
    return x


def _refuse_gradient(x, what):
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} needs a gradient; the MX4 operators are for inference (use torch.no_grad())")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:   # torch.no_grad() keeps these
        raise ValueError(f"{what} carries a tangent; the MX4 operators are for inference (use forward_ad.unpack_dual)")


def _rows(x, what, types, n=-1):
    """(x as rows of contiguous values, rows, k, row stride, type code); copied only where it has to be, and not
    before the limits of a product with n rows of weights."""
    code = types.get(x.dtype) if isinstance(x, torch.Tensor) and x.is_cuda else None
    if code is None or x.requires_grad or forward_ad._current_level >= 0:
        code = types[_input(x, what, types).dtype]
    if x.dim() != 2:
        if x.dim() < 1 or x.shape[-1] < 1:
            raise ValueError(f"{what} needs at least one value in its last axis")
        x = x.reshape(-1, x.shape[-1])
    rows, k = x.shape
    if rows * (k + 255) >= 2 ** 38 or k > 2 ** 30:   # no limit is nearer: the exact ones are looked at only then
        _fits(rows, k, what)
    if n >= 0 and (k > MAX_K or 4 * rows + n >= 2 ** 21):
        _product_fits(rows, n, k, True)
    row, step = x.stride()
    if rows < 2:
        row = k
    if step != 1 or row < k or not k:
        if not k:
            raise ValueError(f"{what} needs at least one value in its last axis")
        if k > 1 or row < k:
            x, row = x.contiguous(), k
    return x, rows, k, row, code


def _fits(rows, k, what):
    """Refuse a matrix that the C calls cannot count in 32 bits (the limits of include/unoq_mx.h)."""
    if k > 2 ** 30 or rows * (2 * (k + 255 >> 8)) >= 2 ** 31:
        raise ValueError(f"{what} of {rows} rows of {k}: at most 2^30 values to a row, and rows x 2 ceil(k / 256) below 2^31")


def _product_fits(m, n, k, pieces):
    """Refuse a product past the same limits; `pieces`: its activations are in 16 bits."""
    if k > MAX_K or m > MAX_ROWS:
        raise ValueError(f"a product takes at most {MAX_ROWS} rows of {MAX_K} values, not {m} of {k}")
    tiles = 2 * (k + 255 >> 8)
    if (4 * m + 256 if pieces else m + 255) * tiles >= 2 ** 31 or (n + 127) * tiles >= 2 ** 31:
        raise ValueError(f"a product of {m} and {n} rows of {k}: at most 2^31 / (2 ceil(k / 256)) rows of either, with "
                         "their padding" + (", of 16-bit activations a quarter of that" if pieces else ""))


def _row_stride(x, rows, k):
    return x.stride(0) if rows > 1 else max(k, 1)


def _output(out, shape, dtype, device, inputs):
    """Refuse an `out` that the kernels cannot write."""
    if not isinstance(out, torch.Tensor) or tuple(out.shape) != tuple(shape) or out.device != device:
        raise ValueError(f"out must be a tensor of shape {tuple(shape)} on {device}")
    if out.dtype != dtype:
        raise ValueError(f"out must be {dtype}")
    _refuse_gradient(out, "out")
    if out.shape[-1] > 1 and out.stride(-1) != 1 or out.dim() != 2 and not out.is_contiguous() \
            or out.dim() == 2 and out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError("out needs contiguous rows that do not overlap")
    lo = out.data_ptr()
    hi = lo + _extent(out)
    for x in inputs:
        if lo < x.data_ptr() + _extent(x) and x.data_ptr() < hi and not _side_by_side(out, x):
            raise ValueError("out must not overlap an input")


def _side_by_side(a, b):
    """Whether two matrices whose extents cross share no byte: columns of one buffer, or every other of its rows."""
    if a.dim() != 2 or b.dim() != 2:
        return False
    pitches = {x.stride(0) * x.element_size() for x in (a, b) if x.shape[0] > 1}
    if len(pitches) != 1:
        return False
    pitch = pitches.pop()
    at = (b.data_ptr() - a.data_ptr()) % pitch   # of b's rows behind those of a
    return a.shape[1] * a.element_size() <= at <= pitch - b.shape[1] * b.element_size()


def _extent(x):
    """Bytes from x's first to its last element."""
    if x.numel() == 0:
        return 0
    return (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) * x.element_size()


def _sizes(operand, rows, k):
    """Bytes of the codes and of the scales (ug_mx4_codes_bytes, ug_mx4_scales_bytes)."""
    if operand:
        tiles = (rows + 127 >> 7) * (k + 255 >> 8)
        return tiles << 14, tiles << 10
    return rows * ((k + 1) // 2), rows * ((k + 31) // 32)


class MX4:
    """A matrix of ``rows`` x ``k`` 4-bit values with a scale per 32: ``codes`` and ``scales`` (uint8)
    in the ``layout`` ``"operand"`` (what :func:`matmul` reads) or ``"stored"`` (row-major, the form of
    files: (rows, ceil(k/2)) and (rows, ceil(k/32)))."""

    __slots__ = ("rows", "k", "layout", "device", "_data", "_any", "_codes", "_scales")

    def __init__(self, codes, scales, rows, k, layout="operand"):
        if rows < 0 or k < 1:
            raise ValueError("rows must be 0 or more and k 1 or more")
        _fits(rows, k, "a matrix")
        for x, want, name in zip((codes, scales), _sizes(_layout(layout), rows, k), ("codes", "scales")):
            _input(x, name, (torch.uint8,))
            if not x.is_contiguous() or x.numel() != want:
                raise ValueError(f"{name} must be {want} contiguous bytes")
        if codes.device != scales.device:
            raise ValueError("codes and scales are on two devices")
        self.rows, self.k, self.layout, self.device = rows, k, layout, codes.device
        self._data, self._any = (codes, scales), codes   # _any: a tensor to allocate beside
        self._codes, self._scales = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _new(cls, rows, k, layout, beside):
        """An unwritten one on the device of `beside`: both arrays in one allocation, the codes first."""
        self = cls.__new__(cls)
        code_bytes, scale_bytes = _sizes(layout == "operand", rows, k)
        at = (code_bytes + 15) & ~15
        self._data = self._any = data = beside.new_empty(at + scale_bytes, dtype=torch.uint8)
        self.rows, self.k, self.layout, self.device = rows, k, layout, data.device
        self._codes = codes = data.data_ptr()
        self._scales = codes + at
        return self

    def __reduce__(self):   # copies and pickles carry the bytes, not this one's addresses
        return MX4, (self.codes, self.scales, self.rows, self.k, self.layout)

    def _views(self):
        if not isinstance(self._data, tuple):
            code_bytes, scale_bytes = _sizes(self.layout == "operand", self.rows, self.k)
            data = self._data
            codes, scales = data[:code_bytes], data[data.numel() - scale_bytes:]
            if self.layout == "stored":
                codes, scales = codes.view(self.rows, (self.k + 1) // 2), scales.view(self.rows, (self.k + 31) // 32)
            self._data = (codes, scales)
        return self._data

    @property
    def codes(self):
        return self._views()[0]

    @property
    def scales(self):
        return self._views()[1]

    @property
    def shape(self):
        return (self.rows, self.k)

    def dequantize(self, dtype=torch.bfloat16, out=None):
        """The values, (rows, k), rounded to ``dtype`` once."""
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be one of {', '.join(str(t) for t in _TYPES)}")
        lib, rows, k, device = _lib or _library(), self.rows, self.k, self.device
        stride = k
        if out is None:
            out = self._any.new_empty((rows, k), dtype=dtype)
        else:
            _output(out, (rows, k), dtype, device, (self.codes, self.scales))
            stride = _row_stride(out, rows, k)
        rc = lib.ug_mx4_dequantize(self._codes, self._scales, self.layout == "operand", rows, k, out.data_ptr(),
                                   _TYPES[dtype], stride, _stream(device))
        if rc:
            _check(lib, rc, "MX4 dequantise")
        return out


def _layout(name):
    if name not in ("stored", "operand"):
        raise ValueError("layout must be stored or operand")
    return OPERAND if name == "operand" else STORED


def quantize(x, layout="operand"):
    """(..., k) values in 32 or 16 bits -> :class:`MX4` of their rows. Each block of 32 gets the scale
    2^(floor(log2 of its largest magnitude) - 2); values go to the nearest e2m1 (ties to even), at
    most 6 scales; a block holding a NaN or an infinity becomes NaN."""
    x, rows, k, stride, code = _rows(x, "x", _TYPES)
    lib, operand = _lib or _library(), _layout(layout)
    q = MX4._new(rows, k, layout, x)
    rc = lib.ug_mx4_quantize(x.data_ptr(), code, rows, k, stride, operand, q._codes, q._scales, _stream(q.device))
    if rc:
        _check(lib, rc, "MX4 quantise")
    return q


def _stored_pair(codes, scales, k, what):
    for x, name in ((codes, f"{what} codes"), (scales, f"{what} scales")):
        _input(x, name, (torch.uint8,))
    if codes.dim() < 2 or scales.shape[:-1] != codes.shape[:-1] or codes.device != scales.device:
        raise ValueError(f"{what}: codes and scales need the same leading shape and device")
    if k < 1 or codes.shape[-1] != (k + 1) // 2 or scales.shape[-1] != (k + 31) // 32:
        raise ValueError(f"{what}: {k} values a row need {(k + 1) // 2} code and {(k + 31) // 32} scale bytes")
    return codes.contiguous(), scales.contiguous()


def _pack(codes, scales, count, rows, k, paired):
    _fits(count * (rows + 127 & ~127), k, "a matrix in whole tiles")
    lib = _library()
    padded = lib.ug_mx4_pack_rows(count, rows, paired)
    out = [torch.empty(size, dtype=torch.uint8, device=codes.device) for size in _sizes(OPERAND, padded, k)]
    _check(lib, lib.ug_mx4_pack(codes.data_ptr(), scales.data_ptr(), count, rows, k, paired, out[0].data_ptr(),
                                out[1].data_ptr(), _stream(codes.device)), "MX4 pack")
    return out


def pack(codes, scales, k=None):
    """A stored matrix, (n, ceil(k/2)) and (n, ceil(k/32)) bytes, in the operand layout: once per weight.
    ``k`` defaults to twice the code bytes of a row."""
    k = 2 * codes.shape[-1] if k is None else k
    codes, scales = _stored_pair(codes, scales, k, "pack")
    if codes.dim() != 2:
        raise ValueError("pack takes one matrix")
    n = codes.shape[0]
    return MX4(*_pack(codes, scales, 1, n, k, 0), n, k)


def matmul(a, w, dtype=None, out=None):
    """y = a w^T for 4-bit weights ``w`` (n x k): ``a`` is an :class:`MX4` (m x k), or 16-bit values (..., k)
    which are kept exactly down to 2^-12 of the largest of their block of 32, and below that to within 2^-21 of
    that largest (float16: 2^-25): what is far smaller than a loud neighbour loses bits. Sums are held in 32 bits
    and rounded once to ``dtype`` (default: a's, bfloat16 for an MX4). A NaN or an infinity in a block of ``a``
    makes its row NaN."""
    if not isinstance(w, MX4) or w.layout != "operand":
        raise ValueError("w must be an MX4 in operand layout (quantize or pack)")
    lib, n, device = _lib or _library(), w.rows, w.device
    four = isinstance(a, MX4)
    if four:
        if a.layout != "operand":
            raise ValueError("a must be in operand layout")
        m, k, dtype = a.rows, a.k, dtype or torch.bfloat16
        shape = (m, n)
    else:
        values = a
        a, m, k, a_stride, x_type = _rows(a, "a", _HALF, n)
        dtype = dtype or a.dtype
        shape = (m, n) if values is a else (*values.shape[:-1], n)
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be one of {', '.join(str(t) for t in _TYPES)}")
    if k != w.k or a.device != device:
        raise ValueError(f"a has rows of {k} on {a.device}, w of {w.k} on {device}")
    if four and (k > MAX_K or 4 * m + n >= 2 ** 21):
        _product_fits(m, n, k, False)
    stride = n
    if out is None:
        out = w._any.new_empty(shape, dtype=dtype)
    else:
        _output(out, shape, dtype, device, ((a.codes, a.scales) if four else (a,)) + (w.codes, w.scales))
        if out.dim() == 2:
            stride = _row_stride(out, m, n)
    if four:
        rc = lib.ug_mx4_matmul(a._codes, a._scales, m, w._codes, w._scales, n, k, out.data_ptr(), _TYPES[dtype], stride,
                               _stream(device))
    else:
        need = _need.get((m, k, x_type))
        if need is None:
            if len(_need) > 4096:
                _need.clear()
            need = _need[m, k, x_type] = lib.ug_mx4_matmul_x16_workspace(m, k, x_type)
        ws = w._any.new_empty(need) if need else None   # bytes
        rc = lib.ug_mx4_matmul_x16(a.data_ptr(), x_type, a_stride, m, w._codes, w._scales, n, k, out.data_ptr(),
                                   _TYPES[dtype], stride, ws.data_ptr() if need else None, need, _stream(device))
    if rc:
        _check(lib, rc, "MX4 product")
    return out


class Experts:
    """A mixture-of-experts layer for a few tokens (at most 128), its expert weights in 4 bits.

    ``router``: (experts, d) in 16 bits; ``bias``: (experts,) float32 added to the logits, or None.
    ``gate_up``: stored codes and scales of (experts, 2f, d), the gate's rows before the up rows;
    ``down``: those of (experts, d, f). ``normalize``: softmax over the chosen logits, else over all.
    Ties go to the lowest index; a NaN logit comes before every number and makes its token's output NaN.
    The weights are packed once, here; the stored ones are not kept."""

    def __init__(self, router, gate_up, down, top_k, normalize=True, bias=None):
        _input(router, "router", _HALF)
        if router.dim() != 2 or min(router.shape) < 1:
            raise ValueError("router must be (experts, d)")
        e, d = router.shape
        if not 1 <= e <= 256 or not 1 <= top_k <= min(16, e):
            raise ValueError("experts must be 1..256 and top_k 1..16, at most the experts")
        (gc, gs), (dc, ds) = gate_up, down
        if not isinstance(gc, torch.Tensor) or gc.dim() != 3 or gc.shape[0] != e or gc.shape[1] < 2 or gc.shape[1] % 2:
            raise ValueError("gate_up must be codes and scales of (experts, 2f, d)")
        f = gc.shape[1] // 2
        if not isinstance(dc, torch.Tensor) or dc.dim() != 3 or dc.shape[:2] != (e, d):
            raise ValueError("down must be codes and scales of (experts, d, f)")
        if max(d, f) > 16384:
            raise ValueError("widths must be at most 16384")
        gc, gs = _stored_pair(gc, gs, d, "gate_up")
        dc, ds = _stored_pair(dc, ds, f, "down")
        if bias is not None:
            _input(bias, "bias", (torch.float32,))
            if bias.shape != (e,):
                raise ValueError("bias must be (experts,)")
            bias = bias.contiguous()
        for x in (gc, dc) + (() if bias is None else (bias,)):
            if x.device != router.device:
                raise ValueError("the layer's tensors are on two devices")
        self.router, self.bias, self.top_k, self.d, self.f, self.experts = router.contiguous(), bias, top_k, d, f, e
        self.normalize = bool(normalize)
        self.gate_up = _pack(gc, gs, e, 2 * f, d, 1)
        self.down = _pack(dc, ds, e, d, f, 0)
        self._bind()

    def _bind(self):
        """The C side's view of the tensors, which it keeps alive whatever becomes of the attributes."""
        code = _TYPES[self.router.dtype]
        self.device = self.router.device   # a loaded layer's tensors may have been mapped to another
        self._kept = kept = (self.router, self.bias, *self.gate_up, *self.down)
        self._layer = UgMx4Experts(self.experts, self.top_k, self.d, self.f, self.normalize, code,
                                   *(None if x is None else x.data_ptr() for x in kept))
        self._lib, self._ref, self._need, self._types = _library(), C.byref(self._layer), {}, {self.router.dtype: code}

    def __getstate__(self):   # copies and pickles carry the tensors, not this one's addresses
        return {name: value for name, value in self.__dict__.items() if name[0] != "_"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    def __call__(self, x, out=None, return_choice=False):
        """(..., d) of the router's type -> the same shape. ``return_choice``: also the chosen experts
        (tokens, top_k) int32, in falling order of their logits, and their float32 weights."""
        d, device, values = self.d, self.device, x
        x, t, k, x_stride, _ = _rows(x, "x", self._types)
        shape = values.shape
        if k != d or x.device != device:
            raise ValueError(f"x must be (..., {d}) on {device}")
        if t > MAX_TOKENS:
            raise ValueError(f"at most {MAX_TOKENS} tokens, not {t}")
        stride = d
        if out is None:
            out = x.new_empty(shape)
        else:
            _output(out, shape, x.dtype, device, (x, *(kept for kept in self._kept if kept is not None)))
            if out.dim() == 2:
                stride = _row_stride(out, t, d)
        chosen = weights = None
        if return_choice:
            chosen = torch.empty((t, self.top_k), dtype=torch.int32, device=device)
            weights = torch.empty((t, self.top_k), dtype=torch.float32, device=device)
        need = self._need.get(t)
        if need is None:
            need = self._need[t] = self._lib.ug_mx4_experts_workspace(self._ref, t)
        ws = self._kept[-1].new_empty(need)   # bytes
        rc = self._lib.ug_mx4_experts(self._ref, x.data_ptr(), x_stride, t, out.data_ptr(), stride,
                                      chosen.data_ptr() if return_choice else None,
                                      weights.data_ptr() if return_choice else None, ws.data_ptr(), need, _stream(device))
        if rc:
            _check(self._lib, rc, "MX4 experts")
        return (out, chosen, weights) if return_choice else out


def check(device=None):
    """Wait for the device; raise DSPError if a kernel failed or ran out of its bounded waits."""
    device = None if device is None else torch.device(device).index
    device = torch.cuda.current_device() if device is None else device
    lib = _library()
    _check(lib, lib.ug_mx4_check(device), "MX4 check")
