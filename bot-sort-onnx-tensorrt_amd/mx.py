"""Microscaled feature rows (csrc/mx.hip): rows in 4 or 8 bits with a scale per 32 elements, the root-mean-square norm that writes
them, and their product -- `cosine_similarity` for galleries that are kept quantised.

Unlike the NumPy-in / NumPy-out functions of `matching`, everything here takes and returns DEVICE tensors and only enqueues work on
torch's current stream of their device (like `DeviceTracker.step`): no copies, no synchronisation, safe to capture in a graph.
Tensors handed in to be filled may not share memory with inputs, except where a call says so; nothing here forms gradients.
"""
from __future__ import annotations

import ctypes

from . import _lib

torch = None                            # imported by the first call: importing the package does not
_DTYPES = {}                            # enum bts_dtype
_raw_stream = None
_forward_ad = _increment_version = None
_FORMATS = {"e2m1": 0, "e4m3": 1}       # enum bts_mx_format
_ROW, _BLOCK = 128, 32                  # elements a row is padded to; elements per scale
_MOST = 0x7fffffff                      # rows and row strides are C ints


def _init():
    global torch, _raw_stream, _forward_ad, _increment_version
    import torch as t
    from torch.autograd import forward_ad
    from torch.autograd.graph import increment_version
    _DTYPES.update({t.float32: 1, t.float16: 2, t.bfloat16: 3})
    # the number of a device's current stream without the Stream object around it (2 us of a 10 us call)
    _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None)
    _forward_ad, _increment_version = forward_ad, increment_version
    torch = t


def _tensor(t, name):
    if torch is None:
        _init()
    if not isinstance(t, torch.Tensor):
        raise _lib.BtsError("%s: a device tensor is expected, got %s" % (name, type(t).__name__))
    return t


def _dtype_code(dtype):
    if torch is None:
        _init()
    code = _DTYPES.get(dtype)
    if code is None:
        raise _lib.BtsError("mx rows: float32, float16 or bfloat16 expected, got %s" % (dtype,))
    return code


def _format_code(fmt):
    code = _FORMATS.get(fmt)
    if code is None:
        raise _lib.BtsError("mx rows: unknown format %r (e2m1, e4m3)" % (fmt,))
    return code


def _width(d):
    """elements of a padded row"""
    d = int(d)
    if not 0 < d <= 1 << 30:
        raise _lib.BtsError("mx rows: d must lie in 1 .. 2^30, got %d" % d)
    return (d + _ROW - 1) // _ROW * _ROW


def _no_gradient(t, name):
    if t.requires_grad and torch.is_grad_enabled():
        raise _lib.BtsError("%s: no gradient is formed here: detach it or call under torch.no_grad()" % name)
    # (unpack_dual takes 0.3 us a tensor: only inside a dual_level)
    if getattr(_forward_ad, "_current_level", 0) >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise _lib.BtsError("%s: no tangent is formed here: unpack the dual tensor" % name)


def _no_negative(t, name):
    # (parts of complex tensors have a stride of 2: they get here as single columns only)
    if t.is_neg():
        raise _lib.BtsError("%s: the imaginary part of a conjugate: call .resolve_neg()" % name)


def _rows2d(t, name, like=None):
    """A device matrix with unit column stride -> (pointer, row stride in elements)."""
    if not _tensor(t, name).is_cuda:
        raise _lib.BtsError("%s: a device tensor is expected" % name)
    if t.dim() != 2:
        raise _lib.BtsError("%s: [rows, d] expected, got %d dimensions" % (name, t.dim()))
    _no_gradient(t, name)
    n, d = t.shape
    ld, unit = t.stride()
    if n <= 1:
        ld = max(d, 1)
    if (unit != 1 and d > 1) or ld < d:
        raise _lib.BtsError("%s: the elements of a row must be adjacent and rows may not overlap (strides %s): call .contiguous()" % (name, t.stride()))
    if unit != 1:
        _no_negative(t, name)
    if n > _MOST or ld > _MOST:
        raise _lib.BtsError("%s: at most 2^31 - 1 rows, and elements between them" % name)
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise _lib.BtsError("%s: shape, type and device of x expected (%s %s %s)" % (name, tuple(like.shape), like.dtype, like.device))
    return t.data_ptr(), ld


def _call(device):
    """(library, context handle, stream) of a device's current stream."""
    index = device.index
    ctx = _lib._default_ctx.get(index) or _lib.default_context(index)
    stream = torch.cuda.current_stream(device).cuda_stream if index is None or _raw_stream is None else _raw_stream(index)
    return _lib.load(), ctx.handle, stream


def mx_row_bytes(fmt: str, d: int) -> "tuple[int, int]":
    """(code bytes, scale bytes) of one row of d elements."""
    c, s = ctypes.c_int64(), ctypes.c_int64()
    _width(d)
    _lib.check(_lib.load().bts_mx_row_bytes(_format_code(fmt), int(d), ctypes.byref(c), ctypes.byref(s)))
    return c.value, s.value


class MxRows:
    """n rows of d values in microscaled form: `codes` uint8 [n, code bytes], `scales` uint8 [n, d rounded up to 128, / 32], `fmt`
    "e2m1" (two elements a byte, the even one in the low nibble) or "e4m3".  Element = code value * 2^(scale - 127); scale 255 = NaN.
    The layout is include/botsort_hip.h's: a consumer may fill the tensors itself."""
    # rows made here lie in one allocation, codes before scales; the two tensors are views made when asked for (an allocation and two views
    # less: 2 us of an 8 us call)
    __slots__ = ("d", "fmt", "device", "_code", "_n", "_room", "_codes", "_scales")

    def __init__(self, codes, scales, d: int, fmt: str):
        _tensor(codes, "codes"), _tensor(scales, "scales")
        self._code = _format_code(fmt)
        d, wide = int(d), _width(d)
        n = codes.shape[0] if codes.dim() == 2 and codes.shape[0] <= _MOST else -1
        if (codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.shape != (n, wide // 2 if fmt == "e2m1" else wide)
                or scales.shape != (n, wide // _BLOCK)):
            raise _lib.BtsError("MxRows: uint8 codes [n, %d] and scales [n, %d] expected for d = %d in %s, got %s %s" % (
                wide // 2 if fmt == "e2m1" else wide, wide // _BLOCK, d, fmt, tuple(codes.shape), tuple(scales.shape)))
        if not codes.is_cuda or codes.device != scales.device:
            raise _lib.BtsError("MxRows: codes and scales on one GPU expected")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise _lib.BtsError("MxRows: contiguous codes and scales expected")
        self.d, self.fmt, self.device, self._n, self._room, self._codes, self._scales = d, fmt, codes.device, n, None, codes, scales

    def _pointers(self):
        if self._room is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        at = self._room.data_ptr()
        return at, at + self._n * self._widths()[0]

    def _widths(self):
        """(code bytes, scale bytes) of a row"""
        wide = (self.d + _ROW - 1) // _ROW * _ROW
        return wide // 2 if self._code == 0 else wide, wide // _BLOCK

    @property
    def codes(self):
        if self._codes is None:
            c, n = self._widths()[0], self._n
            self._codes = self._room[:n * c].view(n, c)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            (c, t), n = self._widths(), self._n
            self._scales = self._room[n * c:].view(n, t)
        return self._scales

    def __len__(self):
        return self._n

    def __repr__(self):
        return "MxRows(%d x %d, %s, %s)" % (self._n, self.d, self.fmt, self.device)

    @classmethod
    def empty(cls, n: int, d: int, fmt: str, device="cuda") -> "MxRows":
        """Room for n rows."""
        if torch is None:
            _init()
        code, wide = _format_code(fmt), _width(d)
        if not 0 <= n <= _MOST:
            raise _lib.BtsError("MxRows: 0 .. 2^31 - 1 rows, got %d" % n)
        self = cls.__new__(cls)
        self.d, self.fmt, self._code, self._n, self._codes, self._scales = int(d), fmt, code, n, None, None
        self._room = torch.empty(n * ((wide // 2 if code == 0 else wide) + wide // _BLOCK), dtype=torch.uint8, device=device)
        self.device = self._room.device
        if not self._room.is_cuda:
            raise _lib.BtsError("MxRows: rows live on a GPU, got %s" % self.device)
        return self

    def dequantize(self, dtype=None):
        """[n, d] of the values held (float32 unless `dtype` says otherwise)."""
        if torch is None:
            _init()
        dtype = torch.float32 if dtype is None else dtype
        code = _dtype_code(dtype)
        n, d = self._n, self.d
        out = torch.empty((n, d), dtype=dtype, device=self.device)
        lib, ctx, stream = _call(self.device)
        pc, ps = self._pointers()
        _lib.check(lib.bts_mx_dequantize(ctx, pc, ps, self._code, n, d, out.data_ptr(), code, d, stream))
        return out


def _written(*given):
    """Matrices and rows that the caller handed in to be filled (or None): autograd's check of saved tensors is to see that they changed."""
    for t in given:
        if t is not None:
            _increment_version(t if not isinstance(t, MxRows) else t._room if t._room is not None else (t._codes, t._scales))


def _room(out, n, d, fmt, device):
    if out is None:
        return MxRows.empty(n, d, fmt, device)
    if not isinstance(out, MxRows):
        raise _lib.BtsError("out: MxRows expected, got %s" % type(out).__name__)
    if out._n != n or out.d != d or out.fmt != fmt or out.device != device:
        raise _lib.BtsError("out: %d x %d rows in %s on %s expected, got %r" % (n, d, fmt, device, out))
    return out


def mx_quantize(x, fmt: str = "e2m1", out: MxRows = None) -> MxRows:
    """x [n, d] (float32, float16 or bfloat16; rows may be strided) -> its rows in 4 (e2m1) or 8 (e4m3) bits; `out`: rows to fill."""
    dt, f = _dtype_code(_tensor(x, "x").dtype), _format_code(fmt)
    p, ld = _rows2d(x, "x")
    n, d = x.shape
    rows = _room(out, n, d, fmt, x.device)
    lib, ctx, stream = _call(x.device)
    pc, ps = rows._pointers()
    _lib.check(lib.bts_mx_quantize(ctx, p, dt, ld, n, d, f, pc, ps, stream))
    if out is not None:
        _written(out)
    return rows


def rms_norm_mx(x, residual=None, weight=None, eps: float = 1e-6, fmt: str = "e4m3", sum_out=None, y_out=None, out: MxRows = None):
    """Root-mean-square norm of the rows of h = x + residual (rounded to x's type; h = x without a residual), times `weight` [d]
    -> (rows in `fmt`, h).  fmt=None: no quantised rows, only `y_out`.

    `sum_out` (may be x or residual themselves: the addition in place) receives h, `y_out` (likewise) the normalised rows in x's type.
    Without a residual h is x itself, or a copy where y_out takes its place."""
    dt = _dtype_code(_tensor(x, "x").dtype)
    px, ldx = _rows2d(x, "x")
    n, d = x.shape
    pr, ldr = _rows2d(residual, "residual", x) if residual is not None else (None, 0)
    if weight is not None:
        if _tensor(weight, "weight").shape != (d,) or weight.dtype != x.dtype or weight.device != x.device or not weight.is_contiguous():
            raise _lib.BtsError("weight: contiguous [%d] of x's type and device expected" % d)
        _no_gradient(weight, "weight")
        if d == 1:
            _no_negative(weight, "weight")
    py, ldy = _rows2d(y_out, "y_out", x) if y_out is not None else (None, 0)
    h = sum_out
    if h is None and (residual is not None or py == px):            # (y in the place of x: h is x as it was)
        h = torch.empty((n, d), dtype=x.dtype, device=x.device)
        ps, lds = h.data_ptr(), d
    else:
        ps, lds = _rows2d(h, "sum_out", x) if h is not None else (None, 0)
    if fmt is None and out is not None:
        raise _lib.BtsError("out: rows to fill need their fmt")
    f = 0 if fmt is None else _format_code(fmt)
    rows = None if fmt is None else _room(out, n, d, fmt, x.device)
    lib, ctx, stream = _call(x.device)
    qc, qs = (None, None) if rows is None else rows._pointers()
    _lib.check(lib.bts_rms_norm(ctx, dt, px, ldx, pr, ldr, None if weight is None else weight.data_ptr(), n, d, float(eps), ps, lds, py, ldy, f,
                                qc, qs, stream))
    _written(sum_out, y_out, out)
    return rows, x if h is None else h


def mx_product(a: MxRows, b: MxRows, alpha: float = 1.0, floor_zero: bool = False, dtype=None, out=None):
    """[len(a), len(b)] of alpha (a float32) * <a_i, b_j>; floor_zero: max(0, .), the similarity of `cosine_similarity` for unit rows.

    `dtype`: float32 (the default) where both are e2m1; float16 / bfloat16 for any (the default with an e4m3 operand is bfloat16).
    `out`: a matrix to fill (its type counts; rows may be strided)."""
    if not isinstance(a, MxRows) or not isinstance(b, MxRows):
        raise _lib.BtsError("mx_product: MxRows expected")
    device = a.device
    if a.d != b.d or b.device != device:
        raise _lib.BtsError("mx_product: rows of one width on one device expected, got %r and %r" % (a, b))
    n, m = a._n, b._n
    made = out is None
    if made:
        if dtype is None:
            dtype = torch.float32 if a.fmt == b.fmt == "e2m1" else torch.bfloat16
        code = _dtype_code(dtype)
        out = torch.empty((n, m), dtype=dtype, device=device)
        po, ld = out.data_ptr(), m
    else:
        code = _dtype_code(_tensor(out, "out").dtype)
        if tuple(out.shape) != (n, m) or out.device != device or dtype not in (None, out.dtype):
            raise _lib.BtsError("out: [%d, %d] on %s%s expected" % (n, m, device, "" if dtype is None else " of %s" % dtype))
        po, ld = _rows2d(out, "out")
    lib, ctx, stream = _call(device)
    (ac, as_), (bc, bs) = a._pointers(), b._pointers()
    _lib.check(lib.bts_mx_product(ctx, ac, as_, a._code, n, bc, bs, b._code, m, a.d, float(alpha), 1 if floor_zero else 0, po, code, ld, stream))
    if not made:
        _written(out)
    return out
