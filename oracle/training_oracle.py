"""Float64 restatement, in plain numpy, of the operators around the scores:
layer norm, unit rows, the AdamW step and its 8-bit states.  Nothing here
calls the package.

Forward and backward come with an error bound of an fp32 implementation: the
sums' rounding by their length, what it does to each element by the formula.
"""

from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24  # unit roundoff of fp32


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def layer_norm(x, w, b, eps):
    """y, mean, rstd of rows x [R, D] (w, b [D] or None)."""
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    y = (x - mean) * rstd
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    return y, mean[:, 0], rstd[:, 0]


def layer_norm_error(x, w, b, eps):
    """Bound of |y - exact| before y is rounded.  A mean of D fp32 numbers is
    off by at most n U32 mean|x| for chains of n additions (n <= 48: 24 in a
    lane, then a tree), which moves x - mean by as much; the variance and the
    root are off by another few dozen roundings, relatively."""
    _, mean, rstd = layer_norm(x, None, None, eps)
    mean, rstd = mean[:, None], rstd[:, None]
    xh = np.abs((x - mean) * rstd)
    shift = np.abs(x).mean(1, keepdims=True) * rstd
    w = np.ones(x.shape[1]) if w is None else np.abs(w)
    return U32 * (w * (50 * shift + 80 * xh) + 4 * (0 if b is None else np.abs(b)))


def layer_norm_backward(dy, x, w, eps):
    """dx, dw, db."""
    _, mean, rstd = layer_norm(x, None, None, eps)
    mean, rstd = mean[:, None], rstd[:, None]
    xh = (x - mean) * rstd
    g = dy if w is None else dy * w
    dx = rstd * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def layer_norm_backward_error(dy, x, w, eps):
    """Bounds of dx, dw and db before rounding, by the same count: xh is off
    by e = U32 (50 shift + 80 |xh|)."""
    _, mean, rstd = layer_norm(x, None, None, eps)
    mean, rstd = mean[:, None], rstd[:, None]
    xh = np.abs((x - mean) * rstd)
    e = U32 * (50 * np.abs(x).mean(1, keepdims=True) * rstd + 80 * xh)
    g = np.abs(dy if w is None else dy * w)
    c1, c2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    ec2 = (g * e).mean(1, keepdims=True) + 50 * U32 * c2
    dx = rstd * (80 * U32 * (g + c1 + xh * c2) + 50 * U32 * c1 + e * c2 + xh * ec2)
    n = 64 + x.shape[0]
    return dx, (np.abs(dy) * (e + n * U32 * xh)).sum(0), n * U32 * np.abs(dy).sum(0)


# ---------------------------------------------------------------------------
# Unit rows
# ---------------------------------------------------------------------------
def real_tokens(shape, lengths):
    n, length = shape[:2]
    if lengths is None:
        return np.ones((n, length), dtype=bool)
    return np.arange(length) < np.clip(np.asarray(lengths), 0, length)[:, None]


def unit_rows(x, lengths, eps):
    """y [N, L, D] with zeros for padding."""
    real = real_tokens(x.shape, lengths)[..., None]
    x = np.where(real, x, 0.0)
    return x / np.maximum(np.sqrt((x * x).sum(-1, keepdims=True)), eps)


def unit_rows_backward(dy, x, lengths, eps):
    """dx for dy [N, L, D] (whatever stands in padding)."""
    real = real_tokens(x.shape, lengths)[..., None]
    x, dy = np.where(real, x, 0.0), np.where(real, dy, 0.0)
    norm = np.sqrt((x * x).sum(-1, keepdims=True))
    y = x / np.maximum(norm, eps)
    along = np.where(norm > eps, (y * dy).sum(-1, keepdims=True), 0.0)
    return np.where(real, (dy - y * along) / np.maximum(norm, eps), 0.0)


def unit_rows_backward_error(dy, x, lengths, eps):
    real = real_tokens(x.shape, lengths)[..., None]
    x, dy = np.where(real, x, 0.0), np.where(real, dy, 0.0)
    norm = np.maximum(np.sqrt((x * x).sum(-1, keepdims=True)), eps)
    y = np.abs(x) / norm
    along = (y * np.abs(dy)).sum(-1, keepdims=True)
    return 100 * U32 * (np.abs(dy) + y * along) / norm


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
def adamw(p, g, m, v, step, lr, beta1, beta2, eps, decay):
    """p, m, v after the step."""
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    mh, vh = m / (1 - beta1 ** step), v / (1 - beta2 ** step)
    with np.errstate(invalid="ignore", divide="ignore"):
        return p - lr * (mh / (np.sqrt(vh) + eps) + decay * p), m, v


BLOCK = 256
TOP = {True: 14, False: 30}
LOWEST = {True: 32, False: 48}


def dither(position, step, seed):
    """What is added to the 20 bits below a code of the first and second moment
    of the elements at ``position`` (uint64 array): 16 random bits, and half of
    the last of them."""
    low = np.uint64(0xFFFFFFFF)
    key = np.uint64((seed * 0x9E3779B1 + step * 0x3C6EF373) & 0xFFFFFFFF)
    with np.errstate(over="ignore"):
        x = ((position & low) * np.uint64(0x9E3779B1)
             + (position >> np.uint64(32)) * np.uint64(0xA54FF53B) + key) & low
        x ^= x >> np.uint64(16)
        x = (x * np.uint64(0x6A09E667)) & low
        x ^= x >> np.uint64(15)
        x = (x * np.uint64(0xBB67AE85)) & low
        x ^= x >> np.uint64(16)
    return ((x & np.uint64(0xFFFF)) * np.uint64(16) + np.uint64(8)).astype(np.int64), \
        ((x >> np.uint64(16)) * np.uint64(16) + np.uint64(8)).astype(np.int64)


def _blocks(x, fill=0):
    pad = -len(x) % BLOCK
    return np.concatenate([x, np.full(pad, fill, dtype=x.dtype)]).reshape(-1, BLOCK)


def encode(x, signed, bits20):
    """Codes and block exponents of fp32 values x [n]: each magnitude in units
    of its own code step (a power of two), cut, and one more where the rest and
    the random bits reach a whole step."""
    x = np.asarray(x, dtype=np.float32)
    n = len(x)
    a = np.abs(_blocks(x)).astype(np.float64)
    field = (_blocks(x).view(np.int32) & 0x7FFFFFFF) >> 23
    e = np.maximum(field.max(1), LOWEST[signed])[:, None]
    fine = e < 255
    a = np.where(fine, a, 0.0)
    # exponent field of each code, 0 for the evenly spaced ones below
    own = np.maximum(np.frexp(np.maximum(a, 1e-300))[1] - 1 + 127 - e + TOP[signed], 1)
    step = np.ldexp(1.0, own - TOP[signed] + e - 127 - 3)
    units = a / step
    whole = np.floor(units)
    up = (units - whole) * 2.0 ** 20 + _blocks(np.asarray(bits20, dtype=np.int64)) >= 2.0 ** 20
    q = ((own - 1) * 8 + whole + up).astype(np.int64)
    if signed:
        q |= np.signbit(_blocks(x)).astype(np.int64) << 7
    else:
        q = np.where((a > 0) & (q == 0), 1, q)
    q = np.where(fine, q, 0)
    return q.reshape(-1)[:n].astype(np.uint8), e[:, 0].astype(np.uint8)


def decode(codes, e, signed):
    """float64 values of codes [n]."""
    n = len(codes)
    q = _blocks(np.asarray(codes).astype(np.int64))
    e = np.asarray(e).astype(np.int64)[:, None]
    mag = q & 127 if signed else q
    field, frac = mag >> 3, mag & 7
    at = np.maximum(e, LOWEST[signed]) - TOP[signed] - 127
    x = np.where(field > 0, np.ldexp((8 + frac) / 8.0, field + at), np.ldexp(frac / 8.0, 1 + at))
    if signed:
        x = np.where(q > 127, -x, x)
    return np.where(e == 255, np.nan, x).reshape(-1)[:n]
