"""Microscaled floating point in numpy, 64 bits: the definition that the device kernels are held to."""
import numpy as np

from rgpu_amd import gpu as G

TABLE = {
    G.MXFP4: np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64),
    G.MXFP8: np.array([c / 512 for c in range(8)] + [(8 + c % 8) / 8 * 2.0 ** (c // 8 - 7) for c in range(8, 127)]),
}


def quantize(x, fmt):
    """(codes, scale bytes, values) of the rows of x: codes [rows, padded columns], bytes [rows, blocks].  Codes are
    0x7f for what is not finite in MXFP8; a block with such a value has byte 255 in MXFP4."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    pad = -cols % 128
    x = np.concatenate([x, np.zeros((rows, pad))], axis=1).reshape(rows, -1, 32)
    table, top = TABLE[fmt], TABLE[fmt][-1]
    finite = np.isfinite(x)
    amax = np.where(finite, np.abs(x), 0).max(axis=2)
    m, e = np.frexp(amax)
    tm, te = np.frexp(top)
    e = np.where(m > tm, e - te + 1, e - te)  # least e with amax <= top 2^e
    e = np.where(amax > 0, np.maximum(e, -127), -127)
    byte = e + 127
    q = np.where(finite, np.abs(x), 0) / np.ldexp(1.0, e)[:, :, None]
    middle = (table[1:] + table[:-1]) / 2
    code = np.searchsorted(middle, q, side="left")  # middles under q
    tie = (q == middle[np.minimum(code, len(middle) - 1)]) & (code < len(middle)) & (code % 2 == 1)
    code = code + tie
    values = np.copysign(table[code] * np.ldexp(1.0, e)[:, :, None], x)
    if fmt == G.MXFP4:
        code = code | (np.signbit(x).astype(int) << 3)
        bad = ~finite.all(axis=2)
        byte = np.where(bad, 255, byte)
        values[bad] = np.nan
    else:
        with np.errstate(invalid="ignore"):
            code = np.where(code == 0, np.where(x > 0, 0x80, 0), code | (np.signbit(x).astype(int) << 7))
        code = np.where(finite, code, 0x7F)
        values[~finite] = np.nan
    return (code.reshape(rows, -1).astype(np.uint8), byte.astype(np.uint8),
            values.reshape(rows, -1)[:, :cols])


def pack(code, byte, fmt):
    """The bytes of the tensor in the layout of include/rtensor_hip.h, element by element as it is written there."""
    rows, padded = code.shape
    flat = (code[:, 0::2] | (code[:, 1::2] << 4) if fmt == G.MXFP4 else code).reshape(-1)
    steps, groups = padded // 128, -(-rows // 64)
    at = -(-flat.size // 256) * 256
    out = np.zeros(at + steps * groups * 256, np.uint8)
    out[:flat.size] = flat
    row, block = np.meshgrid(np.arange(rows), np.arange(padded // 32), indexing="ij")
    where = ((block // 4) * groups + row // 64) * 256 + 4 * (16 * (block % 4) + row % 16) + row % 64 // 16
    out[at + where.reshape(-1)] = byte.reshape(-1)
    return out


def values(rng, rows, cols, spread=1.0):
    """Activations: features of different sizes, some exact zeros, a row of zeros."""
    x = rng.normal(size=(rows, cols)) * np.exp(rng.normal(size=(1, cols)) * spread)
    x[rng.random((rows, cols)) < 0.1] = 0
    if rows > 2:
        x[rows // 2] = 0
    return x.astype(np.float32)
