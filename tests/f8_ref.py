"""e4m3 blocks in 64 bits: the codec by its table of values, packing by its
definition and the bound on the product's error."""
import numpy as np


def e4m3_values():
    """Value of every code: sign, 4 exponent bits (bias 7), 3 mantissa bits; exponent 15 with mantissa 7 is NaN."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(c & 128, -v, v)


_POS = e4m3_values()[:127]  # 0 .. 448, ascending


def e4m3_round(r):
    """Codes nearest to r (ties to the even code, saturating); NaN gives 0x7F."""
    r = np.asarray(r, dtype=np.float64)
    a = np.minimum(np.abs(np.nan_to_num(r, nan=0.0)), 448.0)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(np.signbit(r), c | 128, c)
    return np.where(np.isnan(r), 0x7F, c).astype(np.uint8)


def pack(x, block_rows):
    """(codes, scales) of x [rows x cols] (fp32): scale and quotient are fp32 roundings by definition."""
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), -(-cols // 128)
    p = np.zeros((nr * block_rows, nc * 128), np.float32)
    p[:rows, :cols] = x
    p = p.reshape(nr, block_rows, nc, 128)
    s = (np.fmax.reduce(np.fmax.reduce(np.abs(p), axis=3, initial=0), axis=1, initial=0) / np.float32(448)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        r = p / s[:, None, :, None]
    r = np.where((s[:, None, :, None] == 0) & ~np.isnan(p), np.float32(0), r)
    return e4m3_round(r).reshape(nr * block_rows, nc * 128)[:rows, :cols], s


def unpack(codes, scales, block_rows):
    """float64 values of codes [rows x cols]."""
    rows, cols = codes.shape
    s = np.repeat(np.repeat(scales.astype(np.float64), block_rows, 0)[:rows], 128, 1)[:, :cols]
    return e4m3_values()[codes] * s


def product_bound(xv, wv, eps):
    """Largest error of x . W^T (values in float64, [N x K] and [M x K]).

    Products of e4m3 codes are exact in fp32.  The 128 of a block are added in
    fp32 (each addition off by at most 2^-23 of the sum of magnitudes, as the
    tensor core may truncate), then the block sums are scaled (a product of
    scales and an FMA: two roundings) and added, at most 8 partial sums after
    that; the result is rounded once to a type of machine epsilon `eps`."""
    nkb = -(-xv.shape[1] // 128)
    mag = np.abs(xv) @ np.abs(wv).T
    y = xv @ wv.T
    return (128 * 2.0 ** -23 + (2 * nkb + 10) * 2.0 ** -24) * mag + eps / 2 * np.abs(y) * (1 + 1e-3) + 1e-37
