"""Plain 64-bit forms of layer norm, of checkpoints in 8 bits and of a fully
connected layer's weight gradient, and the error bounds that their kernels are
held to.

u = 2^-24 is half a step of fp32.  A sum of n terms is made of chains of at most
chain(n) additions in fp32, whose error is at most chain(n) u times the sum of
the terms' magnitudes; 64-bit additions add nothing to speak of."""
import numpy as np

from logits_ref import BF16, EPS, F16, F32, TINY, U, from_bits, half_step, to_bits  # noqa: F401

LARGEST = {F32: float(np.finfo(np.float32).max), BF16: 255 * 2.0 ** 120, F16: 65504.0}
BLOCK = 32


def chain(n):
    """additions one after the other in a row's sum: a thread's own values, at
    most 64 or the 256th part of a long row, and what joins the threads'"""
    return min(n, 64 + n / 256) + 24


def span_chain(rows):
    """the same of a sum over rows: spans of at most 256, joined in 64 bits"""
    return min(rows, 256) + 24


# ---- layer norm -------------------------------------------------------------
def forward(x, scales, biases, eps, kind):
    """{name: (value, bound)} of y, mean, rstd and x_norm, by rows.

    The mean is taken relative to the row's first value f: a chain of additions
    of x - f, a division, the sum with f.  The squares are about the rounded
    mean m': their sum is n (var + (m' - mean)^2), with two roundings a term
    and a chain of additions, then a division, the sum with eps, a root and a
    reciprocal: rstd is off by half of the sum's error and 3 u.  x_norm takes
    the error of the mean times rstd, that of rstd, and two roundings, y one of
    the product and one of the sum (the sum's and the type's)."""
    rows, n = x.shape
    c = chain(n)
    mean = x.mean(1, keepdims=True)
    f = x[:, :1]
    var = np.square(x - mean).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    e_mean = (c + 3) * U * np.abs(x - f).mean(1, keepdims=True) + 2 * U * np.abs(mean)
    e_rstd = rstd * (((c + 5) * U + e_mean ** 2 * rstd ** 2) / 2 + 4 * U)
    xn = (x - mean) * rstd
    e_xn = np.abs(xn) * (e_rstd / rstd + 3 * U) + e_mean * rstd * 1.01
    s = 1.0 if scales is None else scales.astype(np.float64)
    b = 0.0 if biases is None else biases.astype(np.float64)
    y = xn * s + b
    e_y = e_xn * np.abs(s) + 2 * U * (np.abs(xn * s) + np.abs(y)) + half_step(y, kind)
    return dict(y=(y, e_y), mean=(mean[:, 0], e_mean[:, 0]), rstd=(rstd[:, 0], e_rstd[:, 0]),
                x_norm=(xn, e_xn))


def backward(delta, x_norm, e_xn, rstd, scales, kind):
    """{name: (value, bound)} of dx, scale_updates and bias_updates; x_norm is
    off by at most e_xn in the kernel."""
    rows, n = delta.shape
    c, cr = chain(n), span_chain(rows)
    s = 1.0 if scales is None else scales.astype(np.float64)
    g = delta * s
    rstd = rstd.reshape(-1, 1)
    m1 = g.mean(1, keepdims=True)
    m2 = (g * x_norm).mean(1, keepdims=True)
    e1 = (c + 3) * U * np.abs(g).mean(1, keepdims=True)
    e2 = ((c + 5) * U * np.abs(g * x_norm) + np.abs(g) * e_xn).mean(1, keepdims=True)
    dx = rstd * (g - m1 - x_norm * m2)
    size = np.abs(g) + np.abs(m1) + np.abs(x_norm * m2)
    e_dx = rstd * (5 * U * size + e1 + np.abs(x_norm) * e2 + e_xn * np.abs(m2)) + half_step(dx, kind)
    ds, db = (delta * x_norm).sum(0), delta.sum(0)
    e_ds = ((cr + 3) * U * np.abs(delta * x_norm) + np.abs(delta) * e_xn).sum(0) + U * np.abs(ds)
    e_db = cr * U * np.abs(delta).sum(0) + U * np.abs(db)
    return dict(dx=(dx, e_dx), scales=(ds, e_ds), biases=(db, e_db))


# ---- checkpoints ----------------------------------------------------------------
def width(n):
    return -(-n // BLOCK) * BLOCK


def pack(x):
    """codes [rows][width] and steps [rows][width / 32] of values in 64 bits"""
    rows, n = x.shape
    b = np.zeros((rows, width(n)))
    b[:, :n] = x
    b = b.reshape(rows, -1, BLOCK)
    bad = ~np.isfinite(b).all(2)
    fine = np.where(bad[..., None], 0, b)
    top = np.abs(fine).max(2)
    step = np.full(top.shape, 7)
    for s in range(7, 254):  # the definition: the smallest that will do
        step = np.where((step == s) & (np.rint(np.ldexp(top, 133 - s)) > 127), s + 1, step)
    codes = np.clip(np.rint(np.ldexp(fine, (133 - step)[..., None])), -127, 127).astype(np.int8)
    step = np.where(bad, 255, step).astype(np.uint8)
    return codes.reshape(rows, -1), step


def values(codes, steps, n):
    """what they stand for, in 64 bits"""
    rows = len(codes)
    v = np.ldexp(codes.reshape(rows, -1, BLOCK).astype(np.float64),
                 steps.astype(np.int64)[..., None] - 133)
    return np.where((steps == 255)[..., None], np.nan, v).reshape(rows, -1)[:, :n]


def buffer(codes, steps):
    """a checkpoint's bytes"""
    return np.concatenate([codes.view(np.uint8).ravel(), steps.ravel()])


def parts(raw, rows, n):
    w = width(n)
    return raw[:rows * w].view(np.int8).reshape(rows, w), raw[rows * w:].reshape(rows, w // BLOCK)


# ---- a fully connected layer's weight gradient ---------------------------------
def weights(delta, x):
    """dw and its bound: exact products, rows additions at most one after the
    other, each off by at most a whole step (2 u: the matrix unit cuts off what
    it aligns) of what has been summed by then, and parts of an fp32 delta below
    2^-126 lost; a few more where the partial sums of row spans are joined."""
    dw = delta.T @ x
    size = np.abs(delta).T @ np.abs(x)
    floor = 4 * 2.0 ** -126 * (1 + np.abs(x).sum(0, keepdims=True)) * (1 + np.abs(delta).max(initial=0))
    return dw, 2 * (min(len(delta), 4096) + 16) * U * size + floor
