"""Plain 64-bit forms of the 8-bit operands, the RMS norm and clipping, in numpy, for the tests."""
import numpy as np

BLOCK = 128


def pitch(n):
    return -(-n // BLOCK) * BLOCK


def scale_pitch(n):
    return -(-n // (4 * BLOCK)) * 4


def round_e4m3(v):
    """f64 values of magnitude <= 448 to the nearest e4m3 value, ties to the even one; NaN stays NaN."""
    _, e = np.frexp(v)
    step = np.ldexp(1.0, np.maximum(e, -5) - 4)  # 2^-3 of the leading power; 2^-9 from the smallest normal 2^-6 on down
    return np.round(v / step) * step


def quantize(x):
    """f32 x [rows, n] -> (values of q [rows, pitch] in f64, scale bytes [rows, scale_pitch])."""
    x = np.asarray(x, dtype=np.float32)
    rows, n = x.shape
    nb = pitch(n) // BLOCK
    v = np.zeros((rows, nb * BLOCK))
    v[:, :n] = x
    v = v.reshape(rows, nb, BLOCK)
    finite = np.isfinite(v)
    top = np.where(finite, np.abs(v), 0.0).max(2, initial=0.0)
    # the smallest e with top <= 448 * 2^e: comparisons of exact f64 values
    _, e = np.frexp(np.where(top > 0, top, 1.0))
    e = e - 9
    e = np.where(top > 448.0 * np.ldexp(1.0, e), e + 1, e)
    e = np.where(top > 0, np.maximum(e, -117), 0)
    with np.errstate(invalid="ignore"):
        q = round_e4m3(np.where(finite, v, np.nan) / np.ldexp(1.0, e)[:, :, None])
    bytes_ = np.full((rows, scale_pitch(n)), 127, dtype=np.uint8)
    bytes_[:, :nb] = e + 127
    return q.reshape(rows, nb * BLOCK), bytes_


def rounded(x):
    """The f64 values that x stands for after rounding to 8 bits along its rows."""
    q, b = quantize(x)
    rows, p = q.shape
    s = np.ldexp(1.0, b[:, : p // BLOCK].astype(np.int64) - 127)
    return (q.reshape(rows, -1, BLOCK) * s[:, :, None]).reshape(rows, p)[:, : np.shape(x)[1]]


def rms_norm(h, w, eps):
    """(y, r) in f64 of f32 rows h."""
    h = np.asarray(h, dtype=np.float64)
    r = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return h * r * np.asarray(w, dtype=np.float64), r[:, 0]


def rms_norm_grad(h, w, eps, gy, gh=None):
    """(gx, gw, magnitude of the terms of gx, of gw) in f64."""
    h, w, gy = (np.asarray(a, dtype=np.float64) for a in (h, w, gy))
    n = h.shape[1]
    r = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    first = gy * w * r
    second = h * (gy * w * h).sum(1, keepdims=True) / n * r ** 3
    gx, size = first - second, np.abs(first) + np.abs(second)
    if gh is not None:
        gx, size = gx + gh, size + np.abs(gh)
    return gx, (gy * h * r).sum(0), size, np.abs(gy * h * r).sum(0)
