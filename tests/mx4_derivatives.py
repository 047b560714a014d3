"""What the 4-bit products promise to automatic differentiation and to programs that watch operations, as functions of the module and a device:
run on the GPU, and on the host with the library's calls computed by `Emulator` (test infrastructure)."""
import ctypes as C

import numpy as np
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from tests import mx4_reference as R

TYPES = {0: C.c_float, 1: C.c_double}


class Emulator(object):
    """`mx4._call` on host memory (float32, float64), from the definition in include/lcx.h"""

    @staticmethod
    def array(ptr, dtype, rows, cols, rs, cs):
        n = 1 + (rows - 1) * rs + (cols - 1) * cs
        a = np.ctypeslib.as_array((TYPES[dtype] * n).from_address(ptr))
        return np.lib.stride_tricks.as_strided(a, (rows, cols), (rs * a.itemsize, cs * a.itemsize))

    @staticmethod
    def buffers(cp, sp, rows, cols):
        tiles = -(-rows // 16)
        return (np.ctypeslib.as_array((C.c_uint8 * (tiles * -(-cols // 256) * 2048)).from_address(cp)),
                np.ctypeslib.as_array((C.c_uint8 * (tiles * -(-cols // 512) * 256)).from_address(sp)))

    @classmethod
    def values(cls, cp, sp, rows, cols):
        code, byte = R.unpack(*cls.buffers(cp, sp, rows, cols), rows, cols)
        return R.values(code, byte[:, :code.shape[1] // 32])[:rows, :cols]

    def __call__(self, index, name, *a):
        if name == "lcx_mx4_quantize":
            x, dtype, rows, cols, rs, cs, cp, sp = a
            code, byte = R.quantize(self.array(x, dtype, rows, cols, rs, cs).astype(np.float64))
            codes, scales = self.buffers(cp, sp, rows, cols)
            tiles, steps, quads = -(-rows // 16), -(-cols // 256) * 2, -(-cols // 512)
            full, b = np.zeros((tiles * 16, steps * 128), np.uint8), np.full((tiles * 16, quads * 16), 2, np.uint8)
            full[:rows, :cols], b[:rows, :byte.shape[1]] = code, byte
            packed = full[:, 0::2] + 16 * full[:, 1::2]
            codes[:] = packed.reshape(tiles, 16, steps, 4, 16).transpose(0, 2, 3, 1, 4).reshape(-1)
            scales[:] = b.reshape(tiles, 16, quads, 4, 4).transpose(0, 2, 4, 1, 3).reshape(-1)
        elif name == "lcx_mx4_dequantize":
            cp, sp, rows, cols, out, dtype, rs, cs = a
            self.array(out, dtype, rows, cols, rs, cs)[:] = self.values(cp, sp, rows, cols)
        elif name == "lcx_mx4_matmul":
            ac, asc, m, bc, bsc, n, k, out, dtype, rs, cs = a[:11]
            self.array(out, dtype, m, n, rs, cs)[:] = self.values(ac, asc, m, k) @ self.values(bc, bsc, n, k).T
        else:
            x, dtype, m, xrs, xcs, cp, sp, n, k, out, rs, cs = a[:12]
            w = self.values(cp, sp, n, k)
            w = w.T if name == "lcx_mx4_linear" else w
            self.array(out, dtype, m, w.shape[1], rs, cs)[:] = self.array(x, dtype, m, w.shape[0], xrs, xcs) @ w


def data(mx4, dev, axis=1):
    """integers of a size whose products and sums are exact: every check below is to the bit"""
    g = torch.Generator().manual_seed(7)
    w = torch.randint(-2, 3, (24, 70), generator=g).float().to(dev)
    x, t = (torch.randint(-4, 5, (5, 70), generator=g).float().to(dev) for _ in range(2))
    dy, v = (torch.randint(-4, 5, (5, 24), generator=g).float().to(dev) for _ in range(2))
    q = mx4.quantize(w, axis=axis)
    wq = mx4.dequantize(q)
    return x, t, dy, v, q, wq


def forward_mode(mx4, dev):
    for axis in (0, 1):
        x, t, dy, v, q, wq = data(mx4, dev, axis)
        for needs in (False, True):
            with fw.dual_level():
                for op, a, b, want in ((mx4.linear, x, t, t @ wq.t()), (mx4.linear_grad, dy, v, v @ wq)):
                    a = a.detach().requires_grad_(needs)
                    p, tan = fw.unpack_dual(op(fw.make_dual(a, b), q))
                    assert tan is not None and torch.equal(tan, want) and torch.equal(p.detach(), op(a.detach(), q))
                    # a tangent that is known to be zero has no memory; an operand without one has no tangent
                    zero = torch._efficientzerotensor(a.shape, device=a.device)
                    tan = fw.unpack_dual(op(fw.make_dual(a, b) * 0 + fw.make_dual(a, zero), q)).tangent
                    assert tan is None or not tan.any()
                    assert fw.unpack_dual(op(a, q)).tangent is None
        # forward over reverse: the gradient is linear in dy, its tangent the product of dy's
        with fw.dual_level():
            xr = x.detach().requires_grad_(True)
            g, = torch.autograd.grad(mx4.linear(xr, q), xr, fw.make_dual(dy, v))
            assert torch.equal(fw.unpack_dual(g).tangent, v @ wq)
        # under no_grad as well: forward mode is not switched off by it
        with fw.dual_level(), torch.no_grad():
            assert torch.equal(fw.unpack_dual(mx4.linear(fw.make_dual(x, t), q)).tangent, t @ wq.t())


def reverse_mode(mx4, dev):
    x, t, dy, v, q, wq = data(mx4, dev)
    x, dy = x.requires_grad_(True), dy.requires_grad_(True)
    g, = torch.autograd.grad(mx4.linear(x, q), x, dy, create_graph=True)
    gg, = torch.autograd.grad(g, dy, t)
    assert torch.equal(g.detach(), (dy @ wq).detach()) and torch.equal(gg, t @ wq.t())


def transforms(mx4, dev):
    from torch.func import grad, jacrev, jvp, vjp, vmap
    for axis in (0, 1):
        x, t, dy, v, q, wq = data(mx4, dev, axis)
        f = lambda a: mx4.linear(a, q)                                   # noqa: E731
        y, tan = jvp(f, (x,), (t,))
        assert torch.equal(y, x @ wq.t()) and torch.equal(tan, t @ wq.t())
        y, pull = vjp(f, x)
        assert torch.equal(y, x @ wq.t()) and torch.equal(pull(dy)[0], dy @ wq)
        assert torch.equal(grad(lambda a: (f(a) * dy).sum())(x), dy @ wq)
        for d in (0, 1):
            stack = torch.stack((x, t, x + t), dim=d)
            want = torch.stack([f(x), f(t), f(x + t)])
            assert torch.equal(vmap(f, in_dims=d)(stack), want)
            assert torch.equal(vmap(f, in_dims=d, out_dims=2)(stack), want.movedim(0, 2))
        assert torch.equal(vmap(f)(x), f(x))                             # rows one by one
        assert torch.equal(jacrev(f)(x[0]), wq)
        # the transposed matrix, and per-sample gradients
        assert torch.equal(vmap(lambda a: mx4.linear_grad(a, q))(dy), dy @ wq)
        per = vmap(grad(lambda a, b: (f(a) * b).sum()))(x, dy)
        assert torch.equal(per, dy @ wq)
        hv = jvp(lambda a: grad(lambda b: (f(b) ** 2).sum())(a), (x,), (t,))[1]
        assert torch.equal(hv, 2 * (t @ wq.t()) @ wq)


class Watch(TorchDispatchMode):
    """records the operators that run under it"""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def _all(mx4, w, x, dy):
    """every operator once, the matrix made inside"""
    q = mx4.quantize(w)
    return (mx4.linear(x, q), mx4.linear_grad(dy, q), mx4.matmul(mx4.quantize(x), q), mx4.dequantize(mx4.quantize(w, axis=0)),
            mx4.linear(dy, mx4.quantize(w, axis=0).t()))


def traced(mx4, dev):
    x, t, dy, v, q, wq = data(mx4, dev)
    other = (wq.flip(0).contiguous(), t, v)
    first, want = _all(mx4, wq, x, dy), _all(mx4, *other)
    assert not torch.equal(first[0], want[0])

    def same(got, want):
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    # the traced program computes: other inputs give their results
    prog = torch.jit.trace(lambda *a: _all(mx4, *a), (wq, x, dy), check_trace=False)
    same(prog(*other), want)
    same(prog(wq, x, dy), first)
    fx = make_fx(lambda *a: _all(mx4, *a))(wq, x, dy)
    assert sum("mx4_" in str(n.target) for n in fx.graph.nodes) == 9 and not any("empty" in str(n.target) for n in fx.graph.nodes)
    same(fx(*other), want)
    # a matrix from outside is a constant of the program
    prog = torch.jit.trace(lambda a: mx4.linear(a, q), (x,), check_trace=False)
    assert torch.equal(prog(t), mx4.linear(t, q))
    prog = make_fx(lambda a: mx4.linear(a, q))(x)
    assert torch.equal(prog(t), mx4.linear(t, q))
    # ... with its gradient
    leaf = t.detach().requires_grad_(True)
    for p in (prog, torch.jit.trace(lambda a: mx4.linear(a, q), (x,), check_trace=False)):
        g, = torch.autograd.grad(p(leaf), leaf, dy)
        assert torch.equal(g, dy @ wq)
    # a gradient inside the traced program
    prog = make_fx(torch.func.grad(lambda a: (mx4.linear(a, q) * dy).sum()))(x)
    assert torch.equal(prog(t), dy @ wq)
    # under a mode that watches: the operators are seen, results and derivatives are the same
    with Watch() as w:
        same(_all(mx4, wq, x, dy), first)
        leaf = x.detach().requires_grad_(True)
        g, = torch.autograd.grad(mx4.linear(leaf, q), leaf, dy)
        with fw.dual_level():
            tan = fw.unpack_dual(mx4.linear(fw.make_dual(x, t), q)).tangent
    assert torch.equal(g, dy @ wq) and torch.equal(tan, t @ wq.t())
    for name in ("quantize", "dequantize", "matmul", "product"):
        assert any("mx4_" + name in s for s in w.seen), (name, w.seen)
    # a matrix made while something watched is one like any other
    with Watch():
        inside = mx4.quantize(wq)
    assert torch.equal(mx4.linear(x, inside), first[0]) and torch.equal(mx4.dequantize(inside.t()), wq.t())


def shapes_only(mx4, dev):
    """a program on tensors without memory learns the shapes"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        w, x, dy = torch.empty(24, 70, device=dev), torch.empty(2, 5, 70, device=dev, dtype=torch.bfloat16), torch.empty(24, device=dev)
        q = mx4.quantize(w)
        assert mx4.linear(x, q).shape == (2, 5, 24) and mx4.linear(x, q).dtype == torch.bfloat16
        assert mx4.linear_grad(dy, q).shape == (70,) and mx4.dequantize(q, torch.float16).dtype == torch.float16
        assert mx4.matmul(mx4.quantize(w), q, torch.bfloat16).shape == (24, 24) and q.codes.numel() + q.scales.numel() == q.nbytes


CHECKS = [forward_mode, reverse_mode, transforms, traced, shapes_only]


def compiled(mx4, dev):
    """torch.compile takes whole programs, without breaks"""
    x, t, dy, v, q, wq = data(mx4, dev)
    want = _all(mx4, wq, x, dy)
    for backend in ("eager", "aot_eager"):
        torch._dynamo.reset()
        f = torch.compile(lambda a: mx4.linear(a, q), backend=backend, fullgraph=True)
        assert torch.equal(f(x), x @ wq.t()) and torch.equal(f(t), t @ wq.t())
        leaf = x.detach().requires_grad_(True)
        f(leaf).backward(dy)
        assert torch.equal(leaf.grad, dy @ wq)
        got = torch.compile(lambda *a: _all(mx4, *a), backend=backend, fullgraph=True)(wq, x, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch._dynamo.reset()


def operators_refuse(mx4, dev):
    """the registered operators check what they are handed: sizes that do not fit reach no kernel"""
    import pytest
    x, t, dy, v, q, wq = data(mx4, dev)
    ops, c, s = torch.ops.linearcorex_amd, q.codes, q.scales
    bad = [lambda: ops.mx4_product(x, c, s, 24, 600, True), lambda: ops.mx4_product(x, c, s, 40, 70, True), lambda: ops.mx4_product(dy, c, s, 24, 70, True),
           lambda: ops.mx4_product(x, c, s, 24, 70, False), lambda: ops.mx4_product(x, c[1:], s, 24, 70, True), lambda: ops.mx4_product(x, c, s[::2], 24, 70, True),
           lambda: ops.mx4_product(x, c.float(), s, 24, 70, True), lambda: ops.mx4_dequantize(c, s, 40, 70, 1, torch.float32),
           lambda: ops.mx4_dequantize(c, s, 24, 70, 0, torch.float32), lambda: ops.mx4_matmul(c, s, 24, c, s, 24, 600, torch.float32),
           lambda: ops.mx4_matmul(c, s, 24, c, s, 40, 70, torch.float32), lambda: ops.mx4_product(x, c, s, -24, 70, True)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert torch.equal(ops.mx4_product(x, c, s, 24, 70, True), mx4.linear(x, q))


CHECKS += [compiled, operators_refuse]
