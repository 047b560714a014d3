"""Cases of the 4-bit microscaled operators (`linearcorex_amd.mx4`) and their plain forms.

A value is held as a 4-bit float (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), 32 neighbours along the
contracted axis share one power-of-two scale.  Operators:

  quantize      rows (axis 1) or columns (axis 0) of a matrix to 4 bits; returned as the values that the 4 bits stand for
  matmul        activations quantised in the call, times weights kept in 4 bits: Q(x) . Wq^T
  linear        activations as they are, times weights kept in 4 bits: x . Wq^T
  linear_grad   the gradient of `linear` with respect to x: dy . Wq; with "forward": both directions, as a training step makes them

`own` false: elementary torch operations in 32 bits; `own` true: the framework's kernels.
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
Q = 17.0 / 32.0            # bytes of a value in 4 bits with its share of the scale


def listed():
    return [
        # 32 tokens of activations on their way into a 4-bit product: a launch's latency
        {"name": "quantize_tokens", "op": "quantize", "rows": 32, "cols": 4096, "axis": 1, "dtype": "bf16"},
        # a large layer's weights, laid out once per load: bandwidth
        {"name": "quantize_weights", "op": "quantize", "rows": 16384, "cols": 8192, "axis": 1, "dtype": "bf16"},
        # the 10000 x 5000 data matrix of the benchmark, in blocks of samples: columns, a ragged last block
        {"name": "quantize_columns", "op": "quantize", "rows": 10000, "cols": 5000, "axis": 0, "dtype": "f32"},
        # eight sequences decoding through one layer, activations in 4 bits
        {"name": "matmul_decode", "op": "matmul", "m": 8, "n": 8192, "k": 8192, "dtype": "bf16"},
        # odd sizes in every direction
        {"name": "matmul_ragged", "op": "matmul", "m": 1000, "n": 5003, "k": 10007, "dtype": "f32"},
        # a large batch through a large layer: the matrix pipe
        {"name": "matmul_large", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16"},
        # one token, one layer
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16"},
        # a handful of sequences decoding, half precision
        {"name": "linear_batch", "op": "linear", "m": 13, "n": 14336, "k": 4096, "dtype": "f16"},
        # a prompt
        {"name": "linear_prompt", "op": "linear", "m": 4096, "n": 8192, "k": 4096, "dtype": "bf16"},
        # 64 factors against a 20000 x 20000 data matrix in 4 bits: the first product of a fit iteration
        {"name": "linear_factors", "op": "linear", "m": 64, "n": 20000, "k": 20000, "dtype": "f32"},
        # a training step through a frozen layer
        {"name": "grad_train", "op": "linear_grad", "m": 2048, "n": 8192, "k": 4096, "dtype": "bf16", "forward": True},
        # ... and the second product of a fit iteration
        {"name": "grad_factors", "op": "linear_grad", "m": 64, "n": 20000, "k": 20000, "dtype": "f32", "forward": False},
    ]


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * e * n, "flops": 4 * n}
    m, n, k = case["m"], case["n"], case["k"]
    both = 2 if case.get("forward") else 1
    if case["op"] == "linear_grad":
        act = m * n + m * k + ((m * k + m * n) if case["forward"] else 0)
    else:
        act = m * k + m * n
    return {"bytes": int(e * act + Q * n * k), "flops": both * 2 * m * n * k}


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "linear", "linear", "linear_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    while True:
        if op == "quantize":
            case = {"op": op, "rows": _log_int(rng, 1, 20000), "cols": _log_int(rng, 1, 20000), "axis": rng.choice([0, 1]), "dtype": dtype}
            if rng.random() < 0.5:
                case["cols"] = max(64, case["cols"] // 64 * 64)
            if case["rows"] * case["cols"] > 128 << 20:
                continue
            return case
        m = rng.choice([_log_int(rng, 1, 16), _log_int(rng, 1, 128), _log_int(rng, 16, 8192)])
        case = {"op": op, "m": m, "n": _log_int(rng, 64, 20000), "k": _log_int(rng, 32, 20000), "dtype": dtype}
        if rng.random() < 0.5:
            case["n"] = max(128, case["n"] // 128 * 128)
            case["k"] = max(128, case["k"] // 128 * 128)
        if op == "linear_grad":
            case["forward"] = rng.random() < 0.5
        cap = 2.0 * 8192 ** 3 if op == "matmul" else 2.8e11
        w = work(case)
        if w["flops"] > cap or w["bytes"] > 1.5e9:
            continue
        return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _activations(g, rows, cols):
    """unit normal values, a few channels thirty times larger (what layers hand to each other)"""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    gain = torch.ones(cols, device="cuda")
    gain[torch.rand(cols, generator=g, device="cuda") < 0.01] = 30.0
    return x * gain


def _weights(g, n, k):
    """rows of different size, as trained weights have"""
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    return w * torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["op"] == "quantize":
        if case["axis"] == 1 and case["rows"] >= 4096:
            state["x"] = _weights(g, case["rows"], case["cols"]).to(dt)
        else:
            state["x"] = _activations(g, case["rows"], case["cols"]).to(dt)
        return state
    m, n, k = case["m"], case["n"], case["k"]
    w = _weights(g, n, k)
    if case["op"] != "linear_grad" or case["forward"]:
        state["x"] = _activations(g, m, k).to(dt)
    if case["op"] == "linear_grad":
        state["dy"] = torch.randn(m, n, generator=g, device="cuda").to(dt)
    if own:
        from linearcorex_amd import mx4
        state["q"] = mx4.quantize(w)
        if "x" in state and case["op"] == "linear_grad":
            state["x"].requires_grad_(True)
    else:
        state["codes"], state["scales"] = _plain_pack(w)
    return state


# ---- plain forms ----------------------------------------------------------------------------------------------------------

def _plain_blocks(x):
    """(rows, blocks, 32) in float32, zeros behind the last column"""
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    xf = x.float()
    if nb * BLOCK != cols:
        xf = torch.cat([xf, xf.new_zeros(rows, nb * BLOCK - cols)], dim=1)
    return xf.reshape(rows, nb, BLOCK)


def _plain_scale(xb):
    """exponent of the shared scale: that of the largest magnitude less 2, kept within [-125, 125]"""
    amax = xb.abs().amax(dim=2, keepdim=True)
    e = torch.frexp(amax)[1] - 3
    return torch.where(amax > 0, e, torch.full_like(e, -125)).clamp(-125, 125)


def _plain_code(r):
    """index 0 .. 7 of the nearest magnitude; a tie goes to the even index"""
    return ((r > 0.25).to(torch.uint8) + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5) + (r >= 3.5) + (r > 5.0)).to(torch.uint8)


def _plain_pow2(e):
    """2 ** e in float32 from its bits (a library power may be off in the last place, which breaks ties the wrong way)"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _plain_table(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)


def _plain_round(x):
    """the values that 4 bits hold for x (rows, cols), in float32"""
    xb = _plain_blocks(x)
    e = _plain_scale(xb)
    r = xb.abs() * _plain_pow2(-e)
    v = _plain_table(x.device)[_plain_code(r).int()] * _plain_pow2(e)
    v = torch.where(xb < 0, -v, v)
    return v.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _plain_pack(w):
    """two codes a byte, one exponent a block: how a plain program keeps 4-bit weights"""
    wb = _plain_blocks(w)
    e = _plain_scale(wb)
    c = _plain_code(wb.abs() * _plain_pow2(-e)) + 8 * (wb < 0).to(torch.uint8)
    c = c.reshape(w.shape[0], -1)
    return c[:, 0::2] + 16 * c[:, 1::2], e.squeeze(2).to(torch.int8)


def _plain_unpack(codes, scales, k):
    table = torch.cat([_plain_table(codes.device), -_plain_table(codes.device)])
    n = codes.shape[0]
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=2).reshape(n, -1, BLOCK)
    return (v * _plain_pow2(scales.unsqueeze(2))).reshape(n, -1)[:, :k]


def _plain(state):
    case = state["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        x = state["x"]
        return _plain_round(x).to(dt) if case["axis"] == 1 else _plain_round(x.t()).t().contiguous().to(dt)
    w = _plain_unpack(state["codes"], state["scales"], case["k"])
    if case["op"] == "matmul":
        return (_plain_round(state["x"]) @ w.t()).to(dt)
    if case["op"] == "linear":
        return (state["x"].float() @ w.t()).to(dt)
    dx = (state["dy"].float() @ w).to(dt)
    if not case["forward"]:
        return dx
    return [(state["x"].float() @ w.t()).to(dt), dx]


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(state):
    if not own:
        return _plain(state)
    from linearcorex_amd import mx4
    case = state["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        return mx4.dequantize(mx4.quantize(state["x"], axis=case["axis"]), dt)
    if case["op"] == "matmul":
        return mx4.matmul(mx4.quantize(state["x"]), state["q"], dt)
    if case["op"] == "linear":
        return mx4.linear(state["x"], state["q"])
    if not case["forward"]:
        return mx4.linear_grad(state["dy"], state["q"])
    y = mx4.linear(state["x"], state["q"])
    dx, = torch.autograd.grad(y, state["x"], state["dy"])
    return [y.detach(), dx]


# ---- from the definition, in 64 bits --------------------------------------------------------------------------------------

def _exact_round(x):
    """nearest representable value in float64: the largest magnitude's binade gives the scale; candidates by their midpoints"""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    mags = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    step = max(1, (1 << 24) // max(1, x.shape[1]))
    for r0 in range(0, x.shape[0], step):
        xd = x[r0:r0 + step].double()
        for_blocks = torch.nn.functional.pad(xd, (0, (-x.shape[1]) % BLOCK)).reshape(xd.shape[0], -1, BLOCK)
        top = for_blocks.abs().max(dim=2).values
        unit = torch.zeros_like(top)
        nz = top > 0
        unit[nz] = torch.floor(torch.log2(top[nz]))
        low = ((unit.long() + 1023) << 52).view(torch.float64)
        unit[nz & (low > top)] -= 1                            # log2 may round the wrong way next to a power of two
        unit[nz & (2 * low <= top)] += 1
        unit = torch.where(nz, unit - 2, torch.full_like(unit, -125)).clamp(-125, 125)
        s = ((unit.long() + 1023) << 52).view(torch.float64).unsqueeze(2)
        a = for_blocks.abs() / s
        best = torch.zeros_like(a)
        dist = a.clone()
        for i, mag in enumerate(mags[1:], start=1):
            d = (a - mag).abs()
            closer = (d < dist) | ((d == dist) & (i % 2 == 0))
            best = torch.where(closer, torch.full_like(best, mag), best)
            dist = torch.where(closer, d, dist)
        v = torch.copysign(best * s, for_blocks)
        out[r0:r0 + step] = v.reshape(xd.shape[0], -1)[:, :x.shape[1]]
    return out


def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        make = _weights if case["axis"] == 1 and case["rows"] >= 4096 else _activations
        x = make(g, case["rows"], case["cols"]).to(dt)
        return _exact_round(x) if case["axis"] == 1 else _exact_round(x.t().contiguous()).t().contiguous()
    w = _exact_round(_weights(g, case["n"], case["k"]))
    x = dy = None
    if case["op"] != "linear_grad" or case["forward"]:
        x = _activations(g, case["m"], case["k"]).to(dt)
    if case["op"] == "linear_grad":
        dy = torch.randn(case["m"], case["n"], generator=g, device="cuda").to(dt)
    if case["op"] == "matmul":
        return _exact_round(x) @ w.t()
    if case["op"] == "linear":
        return x.double() @ w.t()
    dx = dy.double() @ w
    return [x.double() @ w.t(), dx] if case["forward"] else dx
