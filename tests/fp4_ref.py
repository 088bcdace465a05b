"""4-bit rows in numpy, in 64 bits: what the codes and scales of include/nemo_kernels.h stand for."""
import numpy as np

MAGS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def row_bytes(k):
    return -(-k // 128) * 64


def quant(x):
    """(codes, scales) as bytes of padded rows: scale exponent floor(log2 max) - 2, at least 0 as a byte; nearest
    magnitude, ties to the even code; blocks with an infinity or a NaN get scale 255 and zero codes."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    kp = 2 * row_bytes(k)
    v = np.zeros((m, kp))
    v[:, :k] = x
    v = v.reshape(m, -1, 32)
    top = np.abs(v).max(-1)
    fine = np.isfinite(top)
    s = np.where(fine, np.maximum(np.frexp(np.where(fine, top, 1.0))[1] - 1 - 2 + 127, 0), 255)
    s = np.where(top == 0, 0, s)
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.abs(v) / np.exp2(s.astype(np.float64) - 127)[..., None]
    code = np.zeros(a.shape, np.uint8)
    for i in range(7):  # past the border between i and i + 1; on it only towards an even code
        border = (MAGS[i] + MAGS[i + 1]) / 2
        code = np.where((a > border) | ((a == border) & (i % 2 == 1)), i + 1, code)
    code = np.where(np.signbit(v), code + 8, code)
    code = np.where(fine[..., None], code, 0).reshape(m, kp).astype(np.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, s.astype(np.uint8)


def values(q, s, k):
    code = np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)
    mag = MAGS[code & 7] * np.where(code & 8, -1.0, 1.0)
    f = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return (mag * np.repeat(f, 32, axis=1))[:, :k]


def random_rows(rng, n, k, lo=118, hi=126):
    """Random codes and scales of n rows, padded with zeros."""
    kp = 2 * row_bytes(k)
    code = rng.integers(0, 16, (n, kp)).astype(np.uint8)
    code[:, k:] = 0
    s = rng.integers(lo, hi, (n, kp // 32)).astype(np.uint8)
    s[:, -(-k // 32):] = 0
    return code[:, 0::2] | code[:, 1::2] << 4, s
