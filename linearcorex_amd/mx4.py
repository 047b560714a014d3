"""Matrices in 4 bits per value: quantisation, and the products a fit and a layer make with them.

    from linearcorex_amd import mx4

    q = mx4.quantize(w)                    # w (N, K) on the GPU -> 4.25 bits per value, blocks of 32 along K
    y = mx4.linear(x, q)                   # x (..., K) . w^T -> (..., N); differentiable with respect to x
    dx = mx4.linear_grad(dy, q)            # dy (..., N) . w   -> (..., K)
    y = mx4.matmul(mx4.quantize(x), q)     # both operands in 4 bits: 4-bit matrix instructions
    w4 = mx4.dequantize(q)                 # the values that the 4 bits stand for

A value is a 4-bit float (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign); 32 neighbours share one power-of-two scale.  The layout and the
rounding are defined in include/lcx.h (lcx_mx4_*), which these functions call on torch tensors: on the current stream, without
waiting, on the device of the tensors.  Traced, compiled and under dispatch modes they are the operators torch.ops.linearcorex_amd.mx4_*; `linear` and
`linear_grad` have derivatives in both modes and work inside torch.func's transforms.  Wrong arguments raise ValueError or TypeError before anything is launched, a failing call
`LcxError`; there is no CPU fallback.

Import torch, or this module, before the first fit of a process: the library then shares the HIP runtime that torch brings along.  Loaded the other way
round there are two of them, and torch finds no GPU (a warning says so here).

`Corex(x_storage="mx4")` keeps the data of a fit in this form.
"""
from __future__ import annotations

import ctypes as C
import functools
import warnings

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _abi
from ._abi import LcxError          # noqa: F401  (what a failing call raises)

if not _abi.torch_first:
    warnings.warn("linearcorex_amd was used before torch was imported: torch brings a HIP runtime of its own and may find no GPU now; import torch (or "
                  "linearcorex_amd.mx4) first", RuntimeWarning, stacklevel=2)

_DTYPES = {torch.float32: _abi.LCX_F32, torch.float64: _abi.LCX_F64, torch.bfloat16: _abi.LCX_BF16, torch.float16: _abi.LCX_F16}
_PRODUCT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
BLOCK = 32

# who may be looking at the operations (each a tenth of a microsecond a call): torch.compile, dispatch modes, torch.jit.trace, torch.func
_compiling, _watching, _tracing = torch.compiler.is_compiling, torch._C._len_torch_dispatch_stack, torch._C._is_tracing
_transforming, _PLAIN = torch._C._are_functorch_transforms_active, (torch.Tensor, torch.nn.Parameter)
# (looked up once: a call of a few microseconds notices)
_Tensor, _strided, _uint8 = torch.Tensor, torch.strided, torch.uint8
_current, _raw_stream = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)


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

    __slots__ = ("shape", "axis", "index", "_buf", "_codes", "_scales", "_cp", "_sp")       # (_cp, _sp: None while a program is traced)

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

    # (not kept: a view made while a program is traced belongs to that program)
    @property
    def codes(self):
        return self._codes if self._buf is None else self._buf[:_sizes(*self._stored())[0]]

    @property
    def scales(self):
        return self._scales if self._buf is None else self._buf[_sizes(*self._stored())[0]:]

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
    if not isinstance(t, _Tensor):
        raise TypeError("%s must be a torch tensor, not %s" % (what, type(t).__name__))
    if t.layout is not _strided:
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
    if _current() == index:                        # (a matrix on the GPU exists: torch has been initialised)
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
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
    shape = x.shape
    if len(shape) != 2:
        raise ValueError("x must have two dimensions, it has %d" % len(shape))
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float32, float64, bfloat16 or float16, not %s" % x.dtype)
    if type(axis) is not int or not 0 <= axis <= 1:
        if isinstance(axis, bool) or axis not in (0, 1, -1, -2):
            raise ValueError("axis must be 0 or 1")
        axis = int(axis) % 2
    if _compiling() or _watching() or _tracing() or type(x) not in _PLAIN:
        return Mx4._over(tuple(shape), axis, x.get_device(), torch.ops.linearcorex_amd.mx4_quantize(x, axis), None, None)
    return _quantize(x, shape, axis)


def _quantize(x, shape, axis):
    if x.is_neg():                       # (the imaginary part of a conjugated view)
        x = x.resolve_neg()
    (rows, cols), (rs, cs) = shape, x.stride()
    if axis == 0:
        rows, cols, rs, cs = cols, rows, cs, rs
    cb, sb = _sizes(rows, cols)
    buf = x.new_empty(cb + sb, dtype=_uint8)
    index, cp = x.get_device(), buf.data_ptr()
    sp = cp + cb
    if rows and cols:
        _call(index, "lcx_mx4_quantize", x.data_ptr(), _DTYPES[x.dtype], rows, cols, rs, cs, cp, sp)
    return Mx4._over(tuple(shape), axis, index, buf, cp, sp)


def dequantize(q, dtype=torch.float32):
    """The values that the 4 bits stand for, as a dense tensor of `q.shape` (exact in float32, float64 and bfloat16)."""
    _is_mx4(q, "q")
    if dtype not in _DTYPES:
        raise TypeError("dtype must be float32, float64, bfloat16 or float16, not %s" % dtype)
    if q._cp is None or _compiling() or _watching() or _tracing():
        return torch.ops.linearcorex_amd.mx4_dequantize(q.codes, q.scales, *q.shape, q.axis, dtype)
    return _dequantize(q.shape, q.axis, q._buf if q._codes is None else q._codes, q.index, q._cp, q._sp, dtype)


def _dequantize(shape, axis, like, index, cp, sp, dtype):
    out = like.new_empty(shape, dtype=dtype)
    if out.numel():
        ld = shape[1]
        (rows, cols), (rs, cs) = (shape, (ld, 1)) if axis == 1 else (shape[::-1], (1, ld))
        _call(index, "lcx_mx4_dequantize", cp, sp, rows, cols, out.data_ptr(), _DTYPES[dtype], rs, cs)
    return out


def matmul(a, b, dtype=torch.float32):
    """a (M, K) . b (N, K)^T of two `Mx4` matrices -> (M, N) in `dtype` (float32, bfloat16, float16): exact products, float32 sums,
    rounded once.  Both hold their blocks along K (axis 1)."""
    if type(a) is not Mx4 or type(b) is not Mx4:
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
    if a._cp is None or b._cp is None or _compiling() or _watching() or _tracing():
        return torch.ops.linearcorex_amd.mx4_matmul(a.codes, a.scales, m, b.codes, b.scales, n, k, dtype)
    return _matmul(a._buf if a._codes is None else a._codes, a.index, a._cp, a._sp, m, b._cp, b._sp, n, k, dtype)


def _matmul(like, index, ac, asc, m, bc, bsc, n, k, dtype):
    out = like.new_empty((m, n), dtype=dtype)
    if m and n:
        dt = _DTYPES[dtype]
        wb = _workspace_bytes(0, dt, m, n, k)
        w = like.new_empty(wb, dtype=_uint8) if wb else None
        _call(index, "lcx_mx4_matmul", ac, asc, m, bc, bsc, n, k, out.data_ptr(), dt, n, 1, w.data_ptr() if wb else None, wb)
    return out


def _product(x, shape, index, cp, sp, n, k, along):
    """x (..., C) of that shape . the stored (n, k) matrix: along the blocks (contraction over the stored columns) or across them (over the rows)"""
    c, o = (k, n) if along else (n, k)
    if x.is_neg():
        x = x.resolve_neg()
    lead = None
    if len(shape) == 2:
        m, x2 = shape[0], x
    else:
        lead, m = shape[:-1], 1
        for d in lead:
            m *= d
        x2 = x.reshape(m, c)
    out = x.new_empty((m, o))
    if m and o:
        dt, (rs, cs), xp, op = _DTYPES[x.dtype], x2.stride(), x2.data_ptr(), 1 if along else 2
        if m > 16 and dt == 2 and cs == 1 and not (rs | xp >> 1) & 7 and rs < 1 << 23 and not c & (127 if along else 63):
            op += 2                      # read in place (include/lcx.h, lcx_mx4_workspace)
        wb = _workspace_bytes(op, dt, m, n, k)
        w = x.new_empty(wb, dtype=_uint8) if wb else None
        _call(index, "lcx_mx4_linear" if along else "lcx_mx4_linear_grad", xp, dt, m, rs, cs, cp, sp, n, k,
              out.data_ptr(), o, 1, w.data_ptr() if wb else None, wb)
    return out if lead is None else out.reshape(lead + (o,))


# ---- derivatives and traced programs -------------------------------------------------------------------------------------------------
# The functions above hand raw pointers to the library, of which a tracer, a dispatch mode or a tensor subclass sees nothing but the empty output.
# Where one of them is watching, the same work goes through registered operators.
def _buffers(codes, scales, rows, cols, like):
    """addresses of a matrix that an operator was handed as tensors"""
    if like.get_device() != codes.get_device():
        raise ValueError("one operand is on %s, the other on %s" % (like.device, codes.device))
    return Mx4((rows, cols), 1, codes, scales)


@torch.library.custom_op("linearcorex_amd::mx4_quantize", mutates_args=())
def _quantize_op(x: torch.Tensor, axis: int) -> torch.Tensor:
    return _quantize(x, x.shape, axis)._buf


@_quantize_op.register_fake
def _(x, axis):
    return x.new_empty(sum(_sizes(*(x.shape if axis == 1 else x.shape[::-1]))), dtype=torch.uint8)


@torch.library.custom_op("linearcorex_amd::mx4_dequantize", mutates_args=())
def _dequantize_op(codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, axis: int, dtype: torch.dtype) -> torch.Tensor:
    q = _buffers(codes, scales, *((rows, cols) if axis == 1 else (cols, rows)), codes)
    return _dequantize((rows, cols), axis, codes, q.index, q._cp, q._sp, dtype)


@_dequantize_op.register_fake
def _(codes, scales, rows, cols, axis, dtype):
    return codes.new_empty((rows, cols), dtype=dtype)


@torch.library.custom_op("linearcorex_amd::mx4_matmul", mutates_args=())
def _matmul_op(a_codes: torch.Tensor, a_scales: torch.Tensor, m: int, b_codes: torch.Tensor, b_scales: torch.Tensor, n: int, k: int,
               dtype: torch.dtype) -> torch.Tensor:
    a, b = _buffers(a_codes, a_scales, m, k, b_codes), _buffers(b_codes, b_scales, n, k, a_codes)
    return _matmul(a_codes, a.index, a._cp, a._sp, m, b._cp, b._sp, n, k, dtype)


@_matmul_op.register_fake
def _(a_codes, a_scales, m, b_codes, b_scales, n, k, dtype):
    return a_codes.new_empty((m, n), dtype=dtype)


# x . the stored (n, k) matrix, `_product`
@torch.library.custom_op("linearcorex_amd::mx4_product", mutates_args=())
def _product_op(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, n: int, k: int, along: bool) -> torch.Tensor:
    q = _buffers(codes, scales, n, k, x)
    if x.size(-1) != (k if along else n):
        raise ValueError("x has %d values to contract, the matrix is %d x %d" % (x.size(-1), n, k))
    return _product(x, x.shape, q.index, q._cp, q._sp, n, k, along)


@_product_op.register_fake
def _(x, codes, scales, n, k, along):
    return x.new_empty(x.shape[:-1] + (n if along else k,))


def _product_op_setup(ctx, inputs, output):
    _, codes, scales, ctx.n, ctx.k, ctx.along = inputs
    ctx.save_for_backward(codes, scales)


def _product_op_backward(ctx, dy):
    return torch.ops.linearcorex_amd.mx4_product(dy, *ctx.saved_tensors, ctx.n, ctx.k, not ctx.along), None, None, None, None, None


_product_op.register_autograd(_product_op_backward, setup_context=_product_op_setup)


def _forward(x, q, along):
    n, k = q._stored()
    if _watching() or q._cp is None or type(x) not in _PLAIN:
        return torch.ops.linearcorex_amd.mx4_product(x, q.codes, q.scales, n, k, along)
    return _product(x, x.shape, q.index, q._cp, q._sp, n, k, along)


class _Product(torch.autograd.Function):
    """the product is linear in x: its gradient is the other product with the same matrix, its tangent the same product of the tangent"""

    @staticmethod
    def forward(ctx, x, q, along):
        ctx.q, ctx.along = q, along
        return _forward(x, q, along)

    @staticmethod
    def backward(ctx, dy):
        return _apply(dy, ctx.q, not ctx.along), None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        if dx._is_zerotensor():                  # (a tangent that is known to be zero may have no memory)
            dx = dx.new_zeros(dx.shape)
        return _apply(dx, ctx.q, ctx.along)


class _TransformedProduct(torch.autograd.Function):
    """the same for torch.func's transforms (which need setup_context; it costs 10 us a call)"""

    @staticmethod
    def forward(x, q, along):
        return _forward(x, q, along)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, ctx.q, ctx.along = inputs

    backward, jvp = staticmethod(_Product.backward), staticmethod(_Product.jvp)

    @staticmethod
    def vmap(info, in_dims, x, q, along):
        return _apply(x.movedim(in_dims[0], 0), q, along), 0


def _apply(x, q, along):
    if _compiling() or _tracing():
        return torch.ops.linearcorex_amd.mx4_product(x, q.codes, q.scales, *q._stored(), along)
    if _transforming():
        return _TransformedProduct.apply(x, q, along)
    if (x.requires_grad and torch.is_grad_enabled()) or _forward_ad._current_level >= 0:
        return _Product.apply(x, q, along)
    return _forward(x, q, along)


def _call_product(x, q, what, contracted):
    _on_gpu(x, what)
    _is_mx4(q, "q")
    if x.dtype not in _PRODUCT_DTYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, not %s" % (what, x.dtype))
    shape = x.shape
    if not shape:
        raise ValueError("%s must have a dimension to contract" % what)
    if shape[-1] != q.shape[contracted]:
        raise ValueError("%s has %d values to contract, q has shape %r" % (what, shape[-1], q.shape))
    if x.get_device() != q.index:
        raise ValueError("%s is on %s, q on %s" % (what, x.device, q.device))
    along = q.axis == contracted
    if _compiling() or _watching() or _tracing() or _transforming() or _forward_ad._current_level >= 0 or x.requires_grad or type(x) is not _Tensor \
            or q._cp is None:
        return _apply(x, q, along)
    n, k = q._stored()
    return _product(x, shape, q.index, q._cp, q._sp, n, k, along)              # (nobody watches, nothing to differentiate)


def linear(x, q):
    """x (..., K) . q (N, K)^T -> (..., N) in x's type (float32, bfloat16, float16): x as it is, the matrix in 4 bits.

    Every product is exact (x enters as a sum of bfloat16 numbers: three for float32, two for float16; what a float32 number holds below
    bfloat16's last place, 2^-133, is rounded to it), the sums are float32, the result is rounded once.  Any strides of x.  Differentiable with respect to x, any number of times; q is a constant.  Blocks of q
    along either axis."""
    return _call_product(x, q, "x", 1)


def linear_grad(dy, q):
    """dy (..., N) . q (N, K) -> (..., K): the gradient of `linear` with respect to x, and the product with the matrix itself where
    `linear` multiplies with its transpose.  Same types, rounding and differentiability."""
    return _call_product(dy, q, "dy", 0)
