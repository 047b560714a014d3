"""Matrices in 4 bits per value: quantisation, and the products a fit and a layer make with them.

    from linearcorex_amd import mx4

    q = mx4.quantize(w)                    # w (N, K) on the GPU -> 4.25 bits per value, blocks of 32 along K
    y = mx4.linear(x, q)                   # x (..., K) . w^T -> (..., N); differentiable with respect to x
    dx = mx4.linear_grad(dy, q)            # dy (..., N) . w   -> (..., K)
    y = mx4.matmul(mx4.quantize(x), q)     # both operands in 4 bits: 4-bit matrix instructions
    w4 = mx4.dequantize(q)                 # the values that the 4 bits stand for

A value is a 4-bit float (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign); 32 neighbours share one power-of-two scale.  The layout and the
rounding are defined in include/lcx.h (lcx_mx4_*), which these functions call on torch tensors: on the current stream, without
waiting, on the device of the tensors.  Wrong arguments raise ValueError or TypeError before anything is launched, a failing call
`LcxError`; there is no CPU fallback.

`Corex(x_storage="mx4")` keeps the data of a fit in this form.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _abi
from ._abi import LcxError          # noqa: F401  (what a failing call raises)

_DTYPES = {torch.float32: _abi.LCX_F32, torch.float64: _abi.LCX_F64, torch.bfloat16: _abi.LCX_BF16, torch.float16: _abi.LCX_F16}
_PRODUCT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
BLOCK = 32


def _sizes(rows, cols):
    """bytes of the codes and of the scales (include/lcx.h, lcx_mx4_layout)"""
    tiles = (rows + 15) >> 4
    return tiles * ((cols + 255) >> 8) * 2048, tiles * ((cols + 511) >> 9) * 256


class Mx4(object):
    """A matrix in 4 bits per value, made by `quantize`.

    shape   (rows, columns) of the matrix
    axis    the axis along which 32 neighbours share a scale: 1 = along a row, 0 = along a column
    codes, scales   its device buffers (uint8): of the matrix itself for axis 1, of its transpose for axis 0
    `q.t()` is the transposed matrix on the same buffers; `copy.deepcopy` and pickling copy them.  Like any tensor, a matrix that is used on
    another stream than the one it was made on must outlive that use."""

    __slots__ = ("shape", "axis", "index", "_buf", "_codes", "_scales", "_cp", "_sp")

    def __init__(self, shape, axis, codes, scales):
        self.shape, self.axis, self._buf, self._codes, self._scales = tuple(shape), axis, None, codes, scales
        if axis not in (0, 1) or len(self.shape) != 2:
            raise ValueError("a matrix has two dimensions and its blocks run along axis 0 or 1")
        for t, n, what in zip((codes, scales), _sizes(*self._stored()), ("codes", "scales")):
            if t.dtype != torch.uint8 or t.numel() != n or not t.is_contiguous() or t.device != codes.device:
                raise ValueError("%s of a matrix of shape %r must be %d contiguous bytes on one device" % (what, self.shape, n))
        self.index, self._cp, self._sp = codes.get_device(), codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _over(cls, shape, axis, index, buf, cp, sp):
        """on one buffer that holds the codes and, behind them, the scales"""
        q = cls.__new__(cls)
        q.shape, q.axis, q.index, q._buf, q._codes, q._scales, q._cp, q._sp = shape, axis, index, buf, None, None, cp, sp
        return q

    @property
    def codes(self):
        if self._codes is None:
            self._codes = self._buf[:_sizes(*self._stored())[0]]
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._scales = self._buf[_sizes(*self._stored())[0]:]
        return self._scales

    @property
    def device(self):
        return (self._codes if self._buf is None else self._buf).device

    @property
    def nbytes(self):
        return sum(_sizes(*self._stored()))

    def t(self):
        q = Mx4.__new__(Mx4)
        q.shape, q.axis, q.index = (self.shape[1], self.shape[0]), 1 - self.axis, self.index
        q._buf, q._codes, q._scales, q._cp, q._sp = self._buf, self._codes, self._scales, self._cp, self._sp
        return q

    def __reduce__(self):
        # (the addresses are the buffers' own: a copy takes its own)
        return Mx4, (self.shape, self.axis, self.codes, self.scales)

    def _stored(self):
        """(rows, columns) of the buffers: blocks run along the columns"""
        return self.shape if self.axis == 1 else (self.shape[1], self.shape[0])

    def __repr__(self):
        return "Mx4(shape=%r, axis=%d, device=%s)" % (self.shape, self.axis, self.device)


def _on_gpu(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor, not %s" % (what, type(t).__name__))
    if t.layout is not torch.strided:
        raise TypeError("%s must be a dense tensor" % what)
    if not t.is_cuda:
        raise ValueError("%s must be on the GPU, it is on %s (there is no CPU fallback)" % (what, t.device))


def _is_mx4(q, what):
    if not isinstance(q, Mx4):
        raise TypeError("%s must be an Mx4 matrix (mx4.quantize), not %s" % (what, type(q).__name__))


_entry = {}


def _call(index, name, *args):
    """one entry point on the current stream of device `index`"""
    if index < 0:
        raise ValueError("the matrix must be on the GPU (there is no CPU fallback)")
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_abi.load(), name)
    if torch._C._cuda_getDevice() == index:        # (a matrix on the GPU exists: torch has been initialised)
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status != 0:
        _abi.check(status)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(op, dtype, m, n, k):
    b = C.c_int64()
    _abi.check(_abi.load().lcx_mx4_workspace(op, dtype, m, n, k, C.byref(b)))
    return b.value


def quantize(x, axis=1):
    """x (rows, columns) -> `Mx4` of the same shape; blocks of 32 run along `axis`.

    float32, float64, bfloat16 or float16, any strides (a transposed view is read in place).  Per block: scale
    2^(floor(log2 max|x|) - 2), values rounded to nearest (ties to the even code), those above 6 scales saturate; a block that holds an
    infinity or a NaN is NaN.  Not differentiable: the result carries no graph."""
    _on_gpu(x, "x")
    if x.dim() != 2:
        raise ValueError("x must have two dimensions, it has %d" % x.dim())
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float32, float64, bfloat16 or float16, not %s" % x.dtype)
    if isinstance(axis, bool) or axis not in (0, 1, -1, -2):
        raise ValueError("axis must be 0 or 1")
    axis %= 2
    if x.is_neg():                       # (the imaginary part of a conjugated view)
        x = x.resolve_neg()
    (rows, cols), (rs, cs) = x.shape, x.stride()
    shape = (rows, cols)
    if axis == 0:
        rows, cols, rs, cs = cols, rows, cs, rs
    cb, sb = _sizes(rows, cols)
    buf = torch.empty(cb + sb, dtype=torch.uint8, device=x.device)
    index, cp = x.get_device(), buf.data_ptr()
    sp = cp + cb
    if rows and cols:
        _call(index, "lcx_mx4_quantize", x.data_ptr(), _DTYPES[x.dtype], rows, cols, rs, cs, cp, sp)
    return Mx4._over(shape, axis, index, buf, cp, sp)


def dequantize(q, dtype=torch.float32):
    """The values that the 4 bits stand for, as a dense tensor of `q.shape` (exact in float32, float64 and bfloat16)."""
    _is_mx4(q, "q")
    if dtype not in _DTYPES:
        raise TypeError("dtype must be float32, float64, bfloat16 or float16, not %s" % dtype)
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    if out.numel():
        (rows, cols), ld = q._stored(), q.shape[1]
        rs, cs = (ld, 1) if q.axis == 1 else (1, ld)
        _call(q.index, "lcx_mx4_dequantize", q._cp, q._sp, rows, cols, out.data_ptr(), _DTYPES[dtype], rs, cs)
    return out


def matmul(a, b, dtype=torch.float32):
    """a (M, K) . b (N, K)^T of two `Mx4` matrices -> (M, N) in `dtype` (float32, bfloat16, float16): exact products, float32 sums,
    rounded once.  Both hold their blocks along K (axis 1)."""
    _is_mx4(a, "a")
    _is_mx4(b, "b")
    if dtype not in _PRODUCT_DTYPES:
        raise TypeError("dtype must be float32, bfloat16 or float16, not %s" % dtype)
    if a.axis != 1 or b.axis != 1:
        raise ValueError("matmul contracts along the blocks: quantize both operands along their columns (axis 1)")
    if a.shape[1] != b.shape[1]:
        raise ValueError("a has %d columns, b has %d" % (a.shape[1], b.shape[1]))
    if a.index != b.index:
        raise ValueError("a is on %s, b on %s" % (a.device, b.device))
    (m, k), n = a.shape, b.shape[0]
    out = torch.empty((m, n), dtype=dtype, device=a.device)
    if m and n:
        dt = _DTYPES[dtype]
        wb = _workspace_bytes(0, dt, m, n, k)
        w = torch.empty(wb, dtype=torch.uint8, device=a.device) if wb else None
        _call(a.index, "lcx_mx4_matmul", a._cp, a._sp, m, b._cp, b._sp, n, k, out.data_ptr(), dt, n, 1, w.data_ptr() if wb else None, wb)
    return out


def _product(x, q, along):
    """x (..., C) . q: along the blocks (contraction over the stored columns) or across them (over the stored rows)"""
    n, k = q._stored()
    c, o = (k, n) if along else (n, k)
    if x.is_neg():
        x = x.resolve_neg()
    lead = None
    if x.dim() == 2:
        m, x2 = x.size(0), x
    else:
        lead, m = x.shape[:-1], 1
        for d in lead:
            m *= d
        x2 = x.reshape(m, c)
    out = x.new_empty((m, o))
    if m and o:
        dt = _DTYPES[x.dtype]
        wb = _workspace_bytes(1 if along else 2, dt, m, n, k)
        w = torch.empty(wb, dtype=torch.uint8, device=x.device) if wb else None
        rs, cs = x2.stride()
        _call(q.index, "lcx_mx4_linear" if along else "lcx_mx4_linear_grad", x2.data_ptr(), dt, m, rs, cs, q._cp, q._sp, n, k,
              out.data_ptr(), o, 1, w.data_ptr() if wb else None, wb)
    return out if lead is None else out.reshape(lead + (o,))


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, q, along):
        ctx.q, ctx.along = q, along
        return _product(x, q, along)

    @staticmethod
    def backward(ctx, dy):
        # the product is linear in x: its gradient is the other product with the same matrix, itself differentiable
        return _apply(dy, ctx.q, not ctx.along), None, None


def _apply(x, q, along):
    if torch.is_grad_enabled() and x.requires_grad:
        return _Product.apply(x, q, along)
    return _product(x, q, along)


def _checked(x, q, what, contracted):
    _on_gpu(x, what)
    _is_mx4(q, "q")
    if x.dtype not in _PRODUCT_DTYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, not %s" % (what, x.dtype))
    if x.dim() < 1:
        raise ValueError("%s must have a dimension to contract" % what)
    if x.size(-1) != q.shape[contracted]:
        raise ValueError("%s has %d values to contract, q has shape %r" % (what, x.size(-1), q.shape))
    if x.get_device() != q.index:
        raise ValueError("%s is on %s, q on %s" % (what, x.device, q.device))


def linear(x, q):
    """x (..., K) . q (N, K)^T -> (..., N) in x's type (float32, bfloat16, float16): x as it is, the matrix in 4 bits.

    Every product is exact (x enters as a sum of bfloat16 numbers: three for float32, two for float16; what a float32 number holds below
    bfloat16's last place, 2^-133, is rounded to it), the sums are float32, the result is rounded once.  Any strides of x.  Differentiable with respect to x, any number of times; q is a constant.  Blocks of q
    along either axis."""
    _checked(x, q, "x", 1)
    return _apply(x, q, q.axis == 1)


def linear_grad(dy, q):
    """dy (..., N) . q (N, K) -> (..., K): the gradient of `linear` with respect to x, and the product with the matrix itself where
    `linear` multiplies with its transpose.  Same types, rounding and differentiability."""
    _checked(dy, q, "dy", 0)
    return _apply(dy, q, q.axis == 0)
