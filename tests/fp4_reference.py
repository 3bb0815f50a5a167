"""The 4-bit formats from their definition, in numpy and 64 bits: tables of what a code and a scale byte
stand for, the nearest entry of a table, the storage."""
import numpy as np

MX, NV = 0, 1
BLOCK = {MX: 32, NV: 16}
MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
CODES = np.concatenate([MAGNITUDES, -MAGNITUDES])


def _e4m3():
    t = np.full(256, np.nan)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        if e != 15 or m != 7:
            t[b] = (-1 if b & 128 else 1) * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return t


E4M3 = _e4m3()
E8M0 = np.concatenate([2.0 ** np.arange(-127.0, 128.0), [np.nan]])


def scale_value(byte, fmt):
    return (E4M3 if fmt == NV else E8M0)[byte]


def nearest(v, table):
    """Index of the entry of an ascending table nearest to v >= 0, ties to the even index."""
    half = (table[:-1] + table[1:]) / 2
    lo, hi = np.searchsorted(half, v, side="left"), np.searchsorted(half, v, side="right")
    return np.where((lo != hi) & (lo % 2 == 1), hi, lo)


def quantize(x, fmt, exponent=0):
    """(codes [rows, cols] 0..15 with +0 for a zero, scale bytes [rows, blocks]) of x (any float type)."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    block = BLOCK[fmt]
    n = -(-cols // block)
    u = np.zeros((rows, n * block))
    u[:, :cols] = x * 2.0 ** -exponent
    u = u.reshape(rows, n, block)
    bad = ~np.isfinite(u).all(2)
    u = np.where(bad[:, :, None], 0.0, u)
    top = np.abs(u).max(2)
    if fmt == NV:
        byte = nearest(np.minimum(top / 6, 448.0), E4M3[:127])
    else:
        byte = np.maximum(np.frexp(top)[1] - 1 - 2, -127) + 127
        byte = np.where(top == 0, 0, byte)
    s = scale_value(byte, fmt)
    q = np.abs(u) / np.where(s == 0, 1, s)[:, :, None]
    mag = np.where((s == 0)[:, :, None], 0, nearest(np.minimum(q, 100.0), MAGNITUDES))
    code = np.where((u < 0) & (mag > 0), mag + 8, mag)
    code = np.where(bad[:, :, None], 2, code)  # 1.0 under a scale that is NaN
    byte = np.where(bad, 0x7F if fmt == NV else 0xFF, byte)
    return code.reshape(rows, -1)[:, :cols].astype(np.uint8), byte.astype(np.uint8)


def values(code, byte, fmt, exponent=0):
    """float64 values of codes [rows, cols] under scale bytes [rows, blocks]."""
    with np.errstate(invalid="ignore"):
        return CODES[code] * np.repeat(scale_value(byte, fmt), BLOCK[fmt], 1)[:, :code.shape[1]] * 2.0 ** exponent


def pitch(cols):
    return -(-cols // 32) * 16


def tiles(cols, fmt):
    return -(-cols // (4 * BLOCK[fmt]))


def pack_codes(code):
    rows, cols = code.shape
    wide = np.zeros((rows, 2 * pitch(cols)), np.uint8)
    wide[:, :cols] = code
    return wide[:, 0::2] | wide[:, 1::2] << 4


def unpack_codes(packed, cols):
    return np.stack([packed & 15, packed >> 4], 2).reshape(packed.shape[0], -1)[:, :cols]


def scale_offsets(rows, cols, fmt):
    """Byte offsets [rows, blocks of whole tiles] of the stored scales."""
    t = tiles(cols, fmt)
    r, b = np.arange(rows)[:, None], np.arange(4 * t)[None, :]
    return ((r // 128) * t + b // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + b % 4


def pack_scales(byte, cols, fmt, fill=0):
    rows = byte.shape[0]
    out = np.full(-(-rows // 128) * tiles(cols, fmt) * 512, fill, np.uint8)
    wide = np.zeros((rows, 4 * tiles(cols, fmt)), np.uint8)
    wide[:, :byte.shape[1]] = byte
    out[scale_offsets(rows, cols, fmt)] = wide
    return out
