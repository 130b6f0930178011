"""CPU restatement, in numpy, of the 8-bit operators and the rotation: what the tests hold the GPU's results against.

An e4m3 code is a sign, 4 bits of exponent (bias 7) and 3 of mantissa, without infinities: 0x7F and 0xFF are NaN, 448 the
largest. 128 consecutive channels of a row (128 x 128 values of a weight) share a scale s = max(amax / 448, 2^-126), amax the
largest finite magnitude; a code is x * (1 / s) rounded to the nearest, ties to the even code. The scale and the product are
fp32 operations here as there; sums and norms are float64.
"""
import numpy as np

TINY = np.float32(2.0 ** -126)


def _values():
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


VALUES = _values()


def encode(v):
    """values (|v| < 464 or not finite) -> codes"""
    v = np.asarray(v, np.float64)
    a = np.abs(np.where(np.isfinite(v), v, 0.0))
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    q = np.rint(a / step) * step                     # ties to the even multiple of the step: to the even code
    e = np.floor(np.log2(np.maximum(q, 2.0 ** -6)))
    c = np.where(q < 2.0 ** -6, q * 512, (e + 6) * 8 + q / 2.0 ** (e - 3)).astype(np.int64)
    c = np.where(np.isfinite(v), c, 127)
    return (c | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def blocks(n):
    return -(-n // 128)


def padded(x, rows=1):
    """[n, d] -> the same with zeros up to whole blocks of 128 channels (and of `rows` rows)"""
    n, d = x.shape
    out = np.zeros((-(-n // rows) * rows, 128 * blocks(d)), x.dtype)
    out[:n, :d] = x
    return out


def _scales(x, axis):
    most = np.where(np.isfinite(x), np.abs(x), 0).max(axis).astype(np.float32)
    return np.maximum(most / np.float32(448), TINY)


def quantise(x):
    """rows [M, D] (taken as fp32) -> codes [M, K], scales [K / 128, M]"""
    b = padded(np.asarray(x, np.float32)).reshape(len(x), -1, 128)
    s = _scales(b, 2)
    with np.errstate(invalid="ignore"):
        y = b * (np.float32(1) / s)[..., None]
    return encode(y).reshape(len(x), -1), np.ascontiguousarray(s.T)


def pack(x):
    """a weight [N, K] -> codes [N, K rounded up], scales [N / 128, K / 128]"""
    n = len(x)
    b = padded(np.asarray(x, np.float32), 128)
    b = b.reshape(len(b) // 128, 128, -1, 128)
    s = _scales(b, (1, 3))
    with np.errstate(invalid="ignore"):
        y = b * (np.float32(1) / s)[:, None, :, None]
    return encode(y).reshape(len(b) * 128, -1)[:n], s


def values(codes, s):
    """rows of activations back, in float64"""
    return (VALUES[codes].reshape(len(codes), -1, 128) * s.T.astype(np.float64)[..., None]).reshape(codes.shape)


def weight(codes, s):
    n = len(codes)
    return (VALUES[codes].reshape(n, -1, 128) * np.repeat(s.astype(np.float64), 128, 0)[:n, :, None]).reshape(codes.shape)


def gemm(x, xs, w, ws):
    with np.errstate(invalid="ignore"):
        return values(x, xs) @ weight(w, ws).T


def glu(kind, g, u):
    g, u = g.astype(np.float64), u.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == "silu":
            return g / (1 + np.exp(-g)) * u
        return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u


def norm(x, t=None, tw=None, w=None, b=None, w_one=False, mode=1, scale=1.0, eps=1e-6, rounded=lambda r: r):
    """-> the stream, what is quantised (both before any rounding but `rounded`, the stream's to its type)"""
    r = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if t is not None:
            t = t.astype(np.float64)
            if tw is not None:
                t = t / np.sqrt((t ** 2).mean(1, keepdims=True) + eps) * tw
            r = r + t
        r = rounded(r * scale)
        d = r - r.mean(1, keepdims=True) if mode == 0 else r
        y = d / np.sqrt((d ** 2).mean(1, keepdims=True) + eps)
        g = (0.0 if w_one else 1.0) if w is None else w.astype(np.float64)
        y = y * (g + (1.0 if w_one else 0.0))
        return r, y + (0.0 if b is None else b.astype(np.float64))


def rope(x, pos, axis_dim, theta=10000.0, mode="inter", freq="own", hq=0, qw=None, kw=None, eps=1e-6):
    """heads [rows, heads, dim], pos [axes, rows] -> the rotated ones"""
    x = x.astype(np.float64)
    rows, heads, dim = x.shape
    for h in range(heads):
        w = qw if h < hq else kw
        if w is not None:
            x[:, h] = x[:, h] / np.sqrt((x[:, h] ** 2).mean(1, keepdims=True) + eps) * w
    R, out, at = sum(axis_dim), x.copy(), 0
    for a, d in enumerate(axis_dim):
        for j in range(d // 2):
            i = at + j
            e = 2 * j / d if freq == "own" else 2 * i / R
            angle = pos[a].astype(np.float64) * theta ** -e
            c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
            lo, hi = (2 * i, 2 * i + 1) if mode == "inter" else (i, i + R // 2)
            out[..., lo] = x[..., lo] * c - x[..., hi] * s
            out[..., hi] = x[..., hi] * c + x[..., lo] * s
        at += d // 2
    return out
