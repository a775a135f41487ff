"""The 8-bit format and its products in numpy, from their definition: f32 for
the format's own roundings, 64 bits for everything else."""
import numpy as np

BLOCK = 128
F16, F32, BF16 = 1, 2, 4


def up(n, m):
    return -(-n // m) * m


def _table():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v[c] = (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) * (-1 if c & 128 else 1)
        if c & 127 == 127:
            v[c] = np.nan
    return v


E4M3 = _table()  # the value of each code


def e4m3(x):
    """Codes of f32 values: nearest, ties to the even code, clamped to +-448, NaN 0x7F."""
    x = np.asarray(x, np.float32).astype(np.float64)
    mag = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=1e9, neginf=1e9)), 448.0)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(mag, 2.0 ** -60))), -6) - 3)
    q = np.rint(mag / step) * step
    code = np.searchsorted(E4M3[:127], q).astype(np.uint8)
    code |= (np.signbit(x).astype(np.uint8) << 7)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def quant_rows(x):
    """x [R, C] -> codes u8 [R, C], scales f32 [blocks, R]."""
    x = np.asarray(x, np.float32)
    R, C = x.shape
    nb = up(C, BLOCK) // BLOCK
    codes, scales = np.zeros((R, C), np.uint8), np.zeros((nb, R), np.float32)
    for b in range(nb):
        v = x[:, b * BLOCK:(b + 1) * BLOCK]
        a = np.where(np.isfinite(v), np.abs(v), np.float32(0)).max(1)
        s = np.maximum(a * np.float32(1 / 448), np.float32(2.0 ** -100))
        with np.errstate(over="ignore", invalid="ignore"):
            codes[:, b * BLOCK:(b + 1) * BLOCK] = e4m3(v * (np.float32(1) / s)[:, None])
        scales[b] = s
    return codes, scales


def quant_weight(w):
    """w [E, N, K] -> codes [E, N, K], scales f32 [E, N blocks, K blocks]."""
    E, N, K = w.shape
    nb, kb = up(N, BLOCK) // BLOCK, up(K, BLOCK) // BLOCK
    codes, scales = np.zeros(w.shape, np.uint8), np.zeros((E, nb, kb), np.float32)
    for n in range(nb):
        for k in range(kb):
            v = w[:, n * BLOCK:(n + 1) * BLOCK, k * BLOCK:(k + 1) * BLOCK].astype(np.float32)
            s = np.maximum(np.abs(v).max((1, 2)) * np.float32(1 / 448), np.float32(2.0 ** -100))
            codes[:, n * BLOCK:(n + 1) * BLOCK, k * BLOCK:(k + 1) * BLOCK] = e4m3(v * (np.float32(1) / s)[:, None, None])
            scales[:, n, k] = s
    return codes, scales


def rows_value(codes, scales):
    return E4M3[codes] * np.repeat(scales.T.astype(np.float64), BLOCK, 1)[:, :codes.shape[1]]


def weight_value(codes, scales):
    """codes [N, K], scales [N blocks, K blocks]."""
    n, k = codes.shape
    return E4M3[codes] * np.repeat(np.repeat(scales.astype(np.float64), BLOCK, 0)[:n], BLOCK, 1)[:, :k]


def product_bound(a, w, y, out, extra=0.0):
    """How far an f32 evaluation of a @ w.T (values a [M, K], w [N, K], result y incl. bias) may be off: every partial
    sum of a block of 128 and of the blocks rounds (or truncates) by at most 2^-23 of the sum of magnitudes, the scale
    product and each add of a block once more, then the output's own rounding."""
    K = a.shape[1]
    mags = np.abs(a) @ np.abs(w).T + extra
    half_ulp = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[out]
    tiny = {F32: 0.0, F16: 2.0 ** -24, BF16: 0.0}[out]
    return (min(K, BLOCK) + up(K, BLOCK) // BLOCK + 6) * 2.0 ** -23 * mags + half_ulp * np.abs(y) + tiny


def pitched(codes, pitch=None, fill=0xFF):
    """codes [..., C] in rows of `pitch` bytes (a multiple of 16); the bytes past C hold `fill` (a NaN code: nothing may
    use them)."""
    C = codes.shape[-1]
    full = np.full(codes.shape[:-1] + (pitch or up(C, 16),), fill, np.uint8)
    full[..., :C] = codes
    return full
