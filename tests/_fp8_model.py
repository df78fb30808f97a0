"""The 8-bit matrices, the norm and the rotation from their definitions, in numpy and 64 bits (no code of
the library)."""

import numpy as np

GROUP = 128


def grid():
    """The values of the 256 codes, NaN where the code is one."""
    c = np.arange(256)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, np.ldexp(f, -9), np.ldexp(8.0 + f, e - 10))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


def encode(y):
    """The code of each value of magnitude at most 448 (1 + 2^-5): the nearest, of two the even one."""
    a = np.abs(y)
    mags = grid()[:127]
    hi = np.searchsorted(mags, a).clip(1, 126)
    lo = hi - 1
    up, down = mags[hi] - a, a - mags[lo]
    code = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    return (code + 128 * np.signbit(y)).astype(np.uint8)


def scale_byte(top):
    """The smallest e with top <= 448 2^e, plus 127, 1 at least; 255 for an infinity or a NaN."""
    with np.errstate(invalid="ignore"):
        part, e = np.frexp(np.where(np.isfinite(top), top, 1.0))  # 448 = 0.875 * 2^9
    byte = np.where(part == 0, 1, e - 9 + (part > 0.875) + 127)
    return np.where(np.isfinite(top), byte.clip(1, 254), 255).astype(np.uint8)


def blocks_of(x, square):
    """x [R, C] zero-padded and seen as [row groups, rows of one, column groups, 128]."""
    r, c = x.shape
    h = GROUP if square else 1
    full = np.zeros((-(-r // h) * h, -(-c // GROUP) * GROUP))
    full[:r, :c] = x
    return full.reshape(-1, h, full.shape[1] // GROUP, GROUP)


def quantise(x, square=False):
    """x [R, C] float64 -> codes uint8 [R, C rounded up to 16], scales uint8."""
    r, c = x.shape
    g = blocks_of(x, square)
    byte = scale_byte(np.abs(g).max((1, 3)))
    inv = np.where(byte == 255, 0.0, np.ldexp(1.0, 127 - byte.astype(int)))
    with np.errstate(invalid="ignore"):
        y = np.nan_to_num(g * inv[:, None, :, None], nan=0.0)
    full = y.reshape(y.shape[0] * y.shape[1], -1)[:r, : -(-c // 16) * 16]
    return encode(full), byte


def values(codes, scales):
    """What codes [R, C] and scales stand for, float64."""
    r, c = codes.shape
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    if len(s) != r:
        s = s.repeat(GROUP, 0)[:r]
    return grid()[codes] * s.repeat(GROUP, 1)[:, :c]


def cancelling(rng, m, n, k):
    """Codes [m, k] and [n, k]: of eight neighbouring products one is +-2^12, alternating, the others are +-2^-2."""
    at = np.arange(k)
    big, flip = at % 8 == 0, np.where(at // 8 % 2 == 0, 1.0, -1.0)
    a, b = (np.where(rng.random((r, k)) < 0.5, 0.5, -0.5) for r in (m, n))
    a[:, big], b[:, big] = 64.0 * flip[big], 64.0
    return encode(a), encode(b)


def cut_product(a, b, digits):
    """a b^T where of eight neighbouring products the digits below 2^-digits of the largest one's power of two are cut."""
    p = (a[:, None, :] * b[None, :, :]).reshape(len(a), len(b), -1, 8)
    unit = np.ldexp(1.0, np.frexp(np.abs(p).max(-1, keepdims=True))[1] - 1 - digits)
    return (np.trunc(p / unit) * unit).sum((-1, -2))


def norm(s, w, eps):
    """s / sqrt(mean(s^2) + eps) * w."""
    return s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * w


def norm_backward(dy, s, w, dsum, eps):
    """(dx, dw) of the sum over all outputs of dy * norm(s, w), plus dsum for s."""
    r = 1.0 / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    g = dy * w
    dx = r * (g - s * r * r * (g * s).mean(-1, keepdims=True)) + dsum
    return dx, (dy * s * r).reshape(-1, s.shape[-1]).sum(0)


def rotate(x, positions, freqs, axis, pairs, inverse=False):
    """x [B, H, T, D], positions [B, T, A] -> the pairs of each row turned, and each pair's length at both its dims."""
    half = len(freqs)
    angle = positions[:, None, :, axis] * freqs * (-1 if inverse else 1)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if pairs == "interleaved" else (i, i + half)
    out, size = x.copy(), np.zeros(x.shape)
    c, s = np.cos(angle), np.sin(angle)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = np.hypot(x[..., a], x[..., b])
    return out, size
