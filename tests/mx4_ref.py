"""Microscaled 4-bit rows and their products in 64 bits, from the format's definition (include/eif_hip_mx.h)."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def kpad(cols):
    return -(-cols // 256) * 256


def quantise(x):
    """(codes [R, kpad / 2], scales [R, kpad / 32]) of rows x."""
    x = np.asarray(x)
    rows, cols = x.shape
    b = np.zeros((rows, kpad(cols)))
    b[:, :cols] = x.astype(np.float64)
    b = b.reshape(rows, -1, 32)
    finite = np.isfinite(b).all(2)
    amax = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0.0)).max(2), 1.0)
    _, e = np.frexp(amax)                      # amax = m 2^e, m in [0.5, 1): floor(log2 amax) = e - 1
    byte = np.where(amax > 0, np.maximum(e - 1 + 125, 0), 0)
    a = np.abs(np.where(finite[:, :, None], b, 0.0)) / np.exp2(byte - 127.0)[:, :, None]
    dist = np.abs(a[..., None] - GRID)
    near = dist == dist.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code + 8 * (np.signbit(b) & finite[:, :, None])
    code = code.reshape(rows, -1).astype(np.uint8)
    byte = np.where(finite, byte, 255).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte


def values(codes, scales, cols):
    """float64 values [..., cols] of packed rows."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v[..., :32 * scales.shape[-1]] * np.repeat(s, 32, -1)[..., :v.shape[-1]])[..., :cols]


def product(a, w, bias=None, glu=False):
    """(y, tolerance) of operand values a [M, K] and matrix values w [N, K].

    A block's 32 products are multiples of a quarter of its scales' product that sum to at most 32 * 36, exact in FP32;
    each of the K / 32 blocks, and each of up to 16 partial sums of the waves, is added with at most one unit in the last
    place of a running sum that the sum of magnitudes bounds: 2^-23 of it. The bias adds one more. Gated: the slope of SiLU
    is at most 1.1; expf, the quotient and the products are within 2^-21 of the result in all."""
    k = a.shape[1]
    tiny = 2.0 ** -126   # sums below the smallest normal number may come out as 0
    y = a @ w.T
    tol = (-(-k // 32) + 16) * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T) + tiny
    if bias is not None:
        y = y + bias
        tol = tol + 2.0 ** -23 * (np.abs(y) + np.abs(bias))
    if not glu:
        return y, tol
    h = w.shape[0] // 2
    g, u, tg, tu = y[:, :h], y[:, h:], tol[:, :h], tol[:, h:]
    with np.errstate(over="ignore"):
        silu = g / (1.0 + np.exp(-g))
    return silu * u, 1.1 * tg * (np.abs(u) + tu) + (np.abs(silu) + 1.1 * tg) * tu + 2.0 ** -21 * np.abs(silu * u) + tiny


def activations(rng, m, k):
    x = rng.standard_normal((m, k))
    return np.where(rng.random((m, k)) < 0.01, 20.0 * x, x).astype(np.float32)


def matrix(rng, n, k):
    return (rng.standard_normal((n, k)) * np.exp2(rng.standard_normal((n, 1))) / np.sqrt(k)).astype(np.float32)
