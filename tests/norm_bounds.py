"""Error bounds of layer norm's forward pass from what its kernels compute:
64-bit sums, in one pass, of d = x - f and d^2, f the row's first value.

u = 2^-24 is half a step of fp32, v = 2^-53 of 64 bits.  A sum is made of at most
c = chain(n) additions one after the other, each off by at most v of the sum of
the terms' magnitudes.  d is rounded once, its square and the addition together
once.

mean   f + (sum d)/n: c + 3 roundings of mean |d|, then u of the result.
var    q/n - m^2 with m = (sum d)/n: c + 4 roundings of q/n; m^2 <= q/n is off by
       twice m's relative error and one rounding, the difference by one more:
       3 c + 16 roundings of q/n in all.
rstd   the rounding of var + eps to 32 bits counts half, a reciprocal root within
       two steps (4 u) is improved once: what is left of it is 3/2 (4 u)^2, and one
       rounding each of the product of the argument and the root (half of it),
       of what that leaves of 1 (nothing to speak of) and of the result: 2 u.  Above
       2^120 a division and a root in 64 bits, then u, or 2^-150 where the result is
       subnormal.  Half of var's relative error comes on top.
x_norm takes the mean's error times rstd, rstd's, and two roundings.
y      one rounding of the product, one of the sum, one to its type."""
import numpy as np

from norm_ref import U, chain, half_step

V = 2.0 ** -53


def forward(x, scales, biases, eps, kind):
    """{name: (value, bound)} of y, mean, rstd and x_norm, by rows"""
    x = x.astype(np.longdouble)
    n = x.shape[1]
    c = chain(n)
    mean = x.mean(1, keepdims=True)
    d = x - x[:, :1]
    q = np.square(d).mean(1, keepdims=True)
    var = np.square(x - mean).mean(1, keepdims=True) + eps
    rstd = 1 / np.sqrt(var)
    e_mean = U * np.abs(mean) + (c + 3) * V * np.abs(d).mean(1, keepdims=True)
    e_rstd = rstd * (2.01 * U + (3 * c + 16) * V * q / var / 2) + 2.0 ** -150
    xn = (x - mean) * rstd
    e_xn = (np.abs(xn) * (e_rstd / rstd + 2 * U) + e_mean * rstd) * 1.01
    s = np.longdouble(1) if scales is None else scales.astype(np.longdouble)
    b = np.longdouble(0) if biases is None else biases.astype(np.longdouble)
    y = xn * s + b
    e_y = (e_xn * np.abs(s) + U * (np.abs(xn * s) + np.abs(y))) * 1.01 + half_step(y, kind)
    out = dict(y=(y, e_y), mean=(mean[:, 0], e_mean[:, 0]), rstd=(rstd[:, 0], e_rstd[:, 0]),
               x_norm=(xn, e_xn))
    return {k: (v.astype(np.float64), e.astype(np.float64)) for k, (v, e) in out.items()}
