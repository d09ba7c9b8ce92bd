"""The numbers of a K/V cache of 8 or 4 bits in numpy, in 64 bits, by search among all numbers of the type."""
import numpy as np

MOST = {4: 7.0, 8: 464.0}


def grid(bits):
    """Magnitudes by code, without the sign: e2m1 has 8, e4m3 127."""
    if bits == 4:
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    e, f = np.divmod(np.arange(127), 8)
    return np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))


def exponent(m, bits):
    """The least e with m <= L 2^e, at least -100."""
    e = np.full(np.shape(m), -100)
    for _ in range(260):
        e = np.where(m > MOST[bits] * 2.0 ** e.astype(np.float64), e + 1, e)
    return e


def quantise(x, bits):
    """(codes [.., d] without packing, scale bytes [.., d / 32]) of x [.., d] in 64 bits."""
    x = np.asarray(x, np.float64)
    shape = x.shape
    x = x.reshape(*shape[:-1], shape[-1] // 32, 32)
    none = ~(np.abs(x) < 2.0 ** 127).all(-1)
    y = np.where(none[..., None], 0.0, x)
    e = exponent(np.abs(y).max(-1), bits)
    a = np.abs(y) * 2.0 ** -e.astype(np.float64)[..., None]
    g = grid(bits)
    up = np.clip(np.searchsorted(g, a), 1, len(g) - 1)
    d_up, d_down = g[up] - a, a - g[up - 1]
    n = np.where((d_up < d_down) | ((d_up == d_down) & (up % 2 == 0)), up, up - 1)
    n = n + np.where(np.signbit(y), 1 << (bits - 1), 0)
    n = np.where(none[..., None], 0, n)
    return n.reshape(shape).astype(np.uint8), np.where(none, 255, e + 127).astype(np.uint8)


def unsure(x, off, bits):
    """Components of x [.., d], each off by at most off [.., d], that could have another code: next to the border of two
    numbers, or in a group that could have another power of two (whose exact components then have other codes, too)."""
    shape = np.shape(x)
    x, off = (np.asarray(t, np.float64).reshape(*shape[:-1], shape[-1] // 32, 32) for t in (x, off))
    low, high = exponent((np.abs(x) - off).max(-1), bits), exponent((np.abs(x) + off).max(-1), bits)
    p = 2.0 ** high.astype(np.float64)[..., None]
    borders = (grid(bits)[1:] + grid(bits)[:-1]) / 2
    a = np.abs(x) / p
    at = np.searchsorted(borders, a)
    near = np.abs(x)  # the sign turns at zero
    for i in (at, at - 1):
        near = np.minimum(near, np.abs(a - borders[np.clip(i, 0, len(borders) - 1)]) * p)
    return (((near <= off) & (off > 0)) | (low != high)[..., None]).reshape(shape)


def values(codes, byte, bits):
    """What codes without packing and scale bytes stand for."""
    g = np.concatenate([grid(bits), [np.nan]]) if bits == 8 else grid(bits)
    half = 1 << (bits - 1)
    v = g[codes & (half - 1)] * np.where(codes & half, -1.0, 1.0)
    byte = np.asarray(byte, np.int64)
    p = np.where(byte == 255, np.nan, 2.0 ** (byte - 127.0))
    return v * np.repeat(p, 32, -1)


def pack(codes, bits):
    return codes if bits == 8 else (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)


def unpack(codes, bits):
    codes = np.asarray(codes)
    return codes if bits == 8 else np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
