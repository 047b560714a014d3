"""The 4-bit format and its products restated in NumPy / float64 (test infrastructure): the definition in include/lcx.h, lcx_mx4_*."""
import numpy as np

MAGS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])      # a tie goes to the even code


def quantize(x):
    """x (R, C) float64 -> codes (R, C) in 0 .. 15, scale bytes (R, ceil(C / 32))"""
    r, c = x.shape
    nb = -(-c // 32)
    xb = np.zeros((r, nb * 32))
    xb[:, :c] = x
    xb = xb.reshape(r, nb, 32)
    bad = ~np.isfinite(xb).all(axis=2)
    amax = np.where(np.isfinite(xb), np.abs(xb), 0.0).max(axis=2)
    e = np.frexp(amax)[1] - 3
    e = np.clip(np.where(amax > 0, e, -125), -125, 125)
    a = np.where(np.isfinite(xb), np.abs(xb), 0.0) / np.ldexp(1.0, e)[:, :, None]
    code = np.zeros(xb.shape, np.int64)
    for i, m in enumerate(MIDS):
        code += (a > m) if i % 2 == 0 else (a >= m)
    code += 8 * np.signbit(xb)
    byte = np.where(bad, 255, e + 127)
    return code.reshape(r, -1)[:, :c], byte.astype(np.int64)


def values(code, byte):
    """the float64 values of codes and scale bytes"""
    v = np.where(code >= 8, -1.0, 1.0) * MAGS[code & 7]
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    return v * np.repeat(s, 32, axis=1)[:, :code.shape[1]]


def round4(x):
    return values(*quantize(np.asarray(x, np.float64)))


def unpack(codes, scales, rows, cols):
    """device buffers of lcx_mx4_layout's form -> codes (R', C'), scale bytes (R', C' / 32) of the padded matrix: 16-row tiles, 256 columns"""
    tiles, steps, quads = -(-rows // 16), -(-cols // 256) * 2, -(-cols // 512)
    c = codes.reshape(tiles, steps, 4, 16, 16).transpose(0, 3, 1, 2, 4).reshape(tiles * 16, steps * 64)       # [row][step, group, byte]
    code = np.empty((tiles * 16, steps * 128), np.int64)
    code[:, 0::2], code[:, 1::2] = c & 15, c >> 4
    b = scales.reshape(tiles, quads, 4, 16, 4).transpose(0, 3, 1, 4, 2).reshape(tiles * 16, quads * 16)       # [row][quad, step, group]
    return code, b.astype(np.int64)
