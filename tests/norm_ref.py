"""Plain 64-bit forms of the norms and rotary positions (numpy), with what f32
arithmetic may be off by, for the tests."""
import numpy as np

U = 2.0 ** -24  # half a step of f32


def half_step(y, dtype):
    """Half a step of the type at |y|."""
    bits, least = {"f16": (10, -24), "bf16": (7, -133), "f32": (23, -149)}[dtype]
    e = np.floor(np.log2(np.maximum(np.abs(y), 1e-300)))
    return np.ldexp(0.5, np.maximum(e - bits, least).astype(np.int64))


def norm(x, w, b, kind, eps):
    """(y, its f32 error bound, h, h's bound, rstd).  A sum goes over at most 64 values a lane, 6 steps of the wave and 16
    waves: at most 90 additions deep, each off by U of the sum of magnitudes."""
    n = x.shape[1]
    depth = 90 * U
    mean = x.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(x), 1))
    d = x - mean
    var = np.square(d).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    off = (depth * np.abs(x).mean(1, keepdims=True) if kind == "layer" else 0) + U * np.abs(d)     # of x - mean
    # the variance's own: its sum's, and 2 |d| off for each of its terms; rstd's is half of that, and 3 roundings
    rel = 0.5 * (depth * var + 2 * (np.abs(d) * off).mean(1, keepdims=True) + np.square(off).mean(1, keepdims=True)) \
        / (var + eps) + 4 * U
    h = d * rstd
    eh = off * rstd + np.abs(h) * (rel + U)
    w = 1.0 if w is None else w
    b = 0.0 if b is None else b
    return h * w + b, eh * np.abs(w) + 2 * U * (np.abs(h * w) + np.abs(b)), h, eh, rstd, rel


def norm_backward(dy, x, w, kind, eps, add):
    """dx, dweight, dbias, each with its f32 error bound."""
    _, _, h, eh, rstd, rel = norm(x, None, None, kind, eps)
    w = 1.0 if w is None else w
    g = dy * w
    depth = 90 * U
    m0 = g.mean(1, keepdims=True) if kind == "layer" else 0.0
    e0 = (depth + 2 * U) * np.abs(g).mean(1, keepdims=True) if kind == "layer" else 0.0
    m1 = (g * h).mean(1, keepdims=True)
    e1 = (np.abs(g) * eh).mean(1, keepdims=True) + (depth + 3 * U) * np.abs(g * h).mean(1, keepdims=True)
    size = np.abs(g) + np.abs(m0) + np.abs(h * m1)
    dx = (g - m0 - h * m1) * rstd
    ex = (4 * U * size + e0 + np.abs(h) * e1 + np.abs(m1) * eh) * rstd + np.abs(dx) * (rel + 2 * U)
    if add is not None:
        dx, ex = dx + add, ex + 2 * U * (np.abs(dx) + np.abs(add))
    rows = len(x) + 8                # additions of a column's sum, at most
    dw, ew = (dy * h).sum(0), (np.abs(dy) * eh).sum(0) + rows * U * np.abs(dy * h).sum(0)
    db, eb = dy.sum(0), rows * U * np.abs(dy).sum(0)
    return (dx, ex), (dw, ew), (db, eb)


def rotary(x, pos, freq, sections, interleaved, inverse):
    """(y, its f32 error bound).  The reduced angle is off by half a step of f32 at half a turn (2^-26 turns, 2^-23.3), sine
    and cosine by at most 2 steps (2^-22), product and sum by one each.  In 64 bits an angle is off by 2^-53 of itself here and
    three times that where it is counted in turns (two products and their constant)."""
    pairs = len(freq)
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = pos[axis].T.astype(np.float64) * freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None] * (-1 if inverse else 1)
    j = np.arange(pairs)
    i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    y, e = x.copy(), np.zeros_like(x)
    a, b = x[..., i], x[..., k]
    y[..., i], y[..., k] = a * c - b * s, b * c + a * s
    e[..., i] = e[..., k] = (np.abs(a) + np.abs(b)) * (2.0 ** -23.3 + 2.0 ** -22 + 2 * U + 2.0 ** -51 * np.abs(angle)[:, None])
    return y, e
