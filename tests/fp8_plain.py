"""The quantizer's and the product's definitions in numpy, 64 bits, element by element where it matters:
what the tests of the 8-bit operators compare with."""
import numpy as np

BLOCK = 128
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
FORMAT = {"e4m3": (3, -6), "e5m2": (2, -14)}    # mantissa bits, smallest normal exponent


def round_to(v, fmt):
    """Nearest value of the format, ties to even; v within its range."""
    bits, low = FORMAT[fmt]
    v = np.asarray(v, dtype=np.float64)
    out = v.copy()
    fine = np.isfinite(v) & (v != 0)
    _, e = np.frexp(v[fine])                     # v = f 2^e, 0.5 <= f < 1
    step = np.exp2(np.maximum(e - 1, low) - bits)
    out[fine] = np.rint(v[fine] / step) * step
    if fmt == "e4m3":
        out[np.isinf(v)] = np.nan
    return out


def block_bytes(x, blocks, fmt):
    """Scale byte of every element's block, [rows, cols]."""
    x = np.asarray(x, dtype=np.float64)
    r, c = x.shape
    mag = np.where(np.isfinite(x), np.abs(x), 0.0)
    br = 1 if blocks == "row" else BLOCK
    bc = 1 if blocks == "col" else BLOCK
    out = np.ones((r, c), dtype=np.int64)
    for i in range(0, r, br):
        for j in range(0, c, bc):
            amax = mag[i:i + br, j:j + bc].max()
            if amax > 0:
                e = -200
                while amax > LARGEST[fmt] * 2.0 ** e:
                    e += 1
                out[i:i + br, j:j + bc] = min(254, max(1, e + 127))
    return out


def quantize(x, blocks, fmt):
    """(values before scaling back, scale bytes by element)."""
    b = block_bytes(x, blocks, fmt)
    return round_to(np.asarray(x, dtype=np.float64) * np.exp2(127.0 - b), fmt), b


def packed(bytes_by_element, dim):
    """The scale array for a contraction over `dim`, from the bytes by element."""
    b = bytes_by_element if dim == 1 else bytes_by_element.T
    outer, length = b.shape
    out = np.zeros((-(-length // 512), -(-outer // BLOCK), 32, 4, 4), dtype=np.uint8)
    for o in range(outer):
        for kb in range(-(-length // BLOCK)):
            out[kb // 4, o // BLOCK, o % 32, o % BLOCK // 32, kb % 4] = b[o, kb * BLOCK]
    return out
