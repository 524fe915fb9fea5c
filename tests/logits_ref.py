"""Plain 64-bit forms of the operators on logits, and the error bounds that
their kernels are held to.

Rounding to nearest is off by at most half a step: u = 2^-24 relative for
fp32, finfo.eps/2 for 16-bit outputs.

Bounds.  A kernel forms z = (x - m)/T with a handful of roundings (the
difference, 1/T, their product, a change of base): 5 u |z|, which is also the
relative error of exp(z), with 2 u more from the exponential itself.  A sum
of n such terms by w lanes adds n/w + 20 roundings to each, w >= 64, and as
many for the moves of the running maximum, each of which scales with its own
exponential.  So with D(z) = (5 |z| + 2 n/64 + 48) u the sum of the terms e is off by
at most sum e D(z)."""
import numpy as np

U = 2.0 ** -24
F32, BF16, F16 = 0, 1, 2
EPS = {F32: 2.0 ** -23, BF16: 2.0 ** -7, F16: 2.0 ** -10}
TINY = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -14}  # smallest normal


def to_bits(a, kind):
    """float values as the element type's bits, rounded to nearest even"""
    a = np.asarray(a, np.float32)
    if kind == F32:
        return a.copy()
    if kind == F16:
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    u = a.view(np.uint32)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7fc0), r).astype(np.uint16)


def from_bits(b, kind):
    """the element type's bits as float64"""
    if kind == BF16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def slack(z, n):
    with np.errstate(invalid="ignore"):
        z = np.where(np.isfinite(z), np.abs(z), 0)
    return (5 * z + 2 * n / 64 + 48) * U


def half_step(v, kind):
    """the last rounding of an output of value v"""
    return EPS[kind] / 2 * np.maximum(np.abs(v), TINY[kind])


def _softmax_parts(x, t):
    """z, e = exp(z), and the sum without one of the largest, of each row"""
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        z = np.where(np.isfinite(x), (x - np.where(np.isfinite(m), m, 0)) / t, x)
    e = np.exp(np.where(np.isnan(z), -np.inf, z))
    first = x.argmax(1)
    others = e.copy()
    others[np.arange(len(x)), first] = 0
    return m[:, 0], z, e, others


def logprobs(x, ids, k, t):
    """The outputs of ach_logprobs_fwd and their bounds, for rows without NaN
    or +inf: dict of (value, bound)."""
    rows, n = x.shape
    m, z, e, others = _softmax_parts(x, t)
    empty = ~np.isfinite(m)
    rest = others.sum(1)
    total = 1 + rest
    log_s = np.where(empty, -np.inf, np.log1p(rest))
    s_err = (others * slack(z, n)).sum(1) / total
    ls_err = s_err + 4 * U * np.abs(np.where(empty, 0, log_s))
    with np.errstate(invalid="ignore"):
        ez = np.where(others > 0, others * z, 0)
    mean = ez.sum(1) / total  # <= 0
    ent = np.where(empty, 0, np.log1p(rest) - mean)
    ent_err = ls_err + (np.abs(ez) * (slack(z, n) + 8 * U)).sum(1) / total + np.abs(mean) * (s_err + 4 * U)
    given = (ids >= 0) & (ids < n)
    at = np.where(given, ids, 0)
    zi = z[np.arange(rows), at]
    with np.errstate(invalid="ignore"):
        lp = np.where(given, np.where(empty, -np.inf, zi - log_s), 0)
    fin = np.where(np.isfinite(zi), np.abs(zi), 0)
    ranks = np.where(given, (x > x[np.arange(rows), at][:, None]).sum(1), -1)
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    zt = np.take_along_axis(z, order, 1)
    with np.errstate(invalid="ignore"):
        tlp = np.where(empty[:, None], -np.inf, zt - log_s[:, None])
    tfin = np.where(np.isfinite(zt), np.abs(zt), 0)
    return dict(logprobs=(lp, np.where(given, ls_err + 6 * U * fin, 0)), ranks=(ranks, 0),
                entropy=(ent, np.where(empty, 0, ent_err)),
                stats=(np.stack((m, log_s), 1), np.stack((0 * ls_err, np.where(empty, 0, ls_err)), 1)),
                top_ids=(order, 0), top_logprobs=(tlp, ls_err[:, None] + 6 * U * tfin))


def logprobs_bwd(x, ids, t, stats, entropy, g, h, kind):
    """The output of ach_logprobs_bwd from these stats and entropies, and its
    bound; g or h may be None."""
    rows, n = x.shape
    ids = np.full(rows, -1) if ids is None else ids
    given = (ids >= 0) & (ids < n)
    gg = np.where(given, g, 0) if g is not None else np.zeros(rows)
    hh = h if h is not None else np.zeros(rows)
    none = ((gg == 0) & (hh == 0)) | (stats[:, 0] == -np.inf)
    m = np.where(none, 0, stats[:, 0])[:, None]
    ls = np.where(none, 0, stats[:, 1])[:, None]
    with np.errstate(invalid="ignore", over="ignore"):
        z = (x - m) / t
        logp = z - ls
        p = np.exp(logp)
        away = p.copy()  # |p - [j == id]|
        r = np.flatnonzero(given)
        away[r, ids[r]] = -np.expm1(logp[r, ids[r]])
        sign = -np.ones_like(p)
        sign[r, ids[r]] = 1
        v = gg[:, None] * sign * away
        ent = np.zeros(rows) if entropy is None else entropy
        pe = np.where(p > 0, p * (logp + ent[:, None]), 0)
        v = (v - hh[:, None] * pe) / t
        fz = np.where(np.isfinite(z), np.abs(z), 0)
        lerr = (5 * fz + 2 * np.abs(ls) + 2 * np.abs(np.where(np.isfinite(logp), logp, 0)) + 6) * U
        scale = np.where(np.isfinite(logp), np.abs(logp), 0) + np.abs(ent)[:, None]
        err = (np.abs(gg)[:, None] * (away * 8 * U + np.minimum(p, 1e300) * lerr) +
               np.abs(hh)[:, None] * p * (lerr * (1 + scale) + 8 * U * scale)) / t
    v = np.where(none[:, None], 0, v)
    err = np.where(none[:, None], 0, err + half_step(v, kind) + 4 * U * np.abs(v))
    return v, err


def distill(x, ids, values, labels, weights, t, tail, soft, hard, kind):
    """loss, delta and their bounds of ach_distill_xent, row by row; x in
    float64 without NaN or +inf in rows of weight not 0."""
    rows, n = x.shape
    loss, lerr = np.zeros(rows), np.zeros(rows)
    delta, derr = np.zeros((rows, n)), np.zeros((rows, n))
    for r in range(rows):
        w = 1.0 if weights is None else float(weights[r])
        m = x[r].max()
        if w == 0 or m == -np.inf:
            continue
        member, p = np.zeros(n, bool), np.zeros(n)
        use_soft = soft != 0 and ids is not None
        if use_soft:
            for i, v in zip(ids[r], values[r]):
                if 0 <= i < n and not member[i]:
                    member[i], p[i] = True, v
            v = p[member] / (1 if tail else t)
            if tail:
                p[member] = np.exp(v)
            elif len(v) and v.max() > -np.inf:
                p[member] = np.exp(v - v.max()) / np.exp(v - v.max()).sum()
            else:
                p[member] = 0
        y = int(labels[r]) if hard != 0 and labels is not None else -1
        with np.errstate(divide="ignore", invalid="ignore"):
            z, z1 = (x[r] - m) / t, x[r] - m
            e, e1 = np.exp(z), np.exp(z1)
            first = x[r].argmax()
            oth, oth1 = e.copy(), e1.copy()
            oth[first] = oth1[first] = 0
            total, total1 = 1 + oth.sum(), 1 + oth1.sum()
            lse, lse1 = np.log1p(oth.sum()), np.log1p(oth1.sum())
            fz, fz1 = np.where(np.isfinite(z), -z, 0), np.where(np.isfinite(z1), -z1, 0)
            d_e, d_e1 = slack(z, n), slack(z1, n)
            s_err = (oth * d_e).sum() / total + 4 * U
            s_err1 = (oth1 * d_e1).sum() / total1 + 4 * U * lse1
            q = e / total
            q_err = q * (d_e + s_err)
            g, g_err = np.zeros(n), np.zeros(n)
            if use_soft:
                sp = p.sum()
                use = p > 0
                kd = (p[use] * (np.log(p[use]) - (z[use] - lse))).sum()
                kd_err = (p[use] * (6 * U * fz[use] + s_err)).sum()
                P, rest, out = sp, 0.0, e[~member].sum()
                if tail and out > 0:
                    rest = max(0.0, 1 - sp)
                    P += rest
                    if rest > 0:
                        kd += rest * (np.log(rest) - (np.log(out) - np.log(total)))
                        kd_err += rest * ((e[~member] * d_e[~member]).sum() / out + s_err + 8 * U * abs(np.log(out / total)))
                g = P * q - p
                g_err = P * q_err + 8 * U * p
                if rest > 0:
                    over = rest * e / out
                    over_err = over * (d_e + (e[~member] * d_e[~member]).sum() / out + 8 * U)
                    g = np.where(member, g, g - over)
                    g_err = g_err + np.where(member, 0, over_err)
                loss[r] += soft * t * t * kd
                lerr[r] += abs(soft) * t * t * kd_err
                g, g_err = soft * t * g, abs(soft) * t * g_err
            if 0 <= y < n:
                q1 = e1 / total1
                loss[r] += hard * (lse1 - z1[y])
                lerr[r] += abs(hard) * (s_err1 + 6 * U * fz1[y])
                g1 = q1.copy()
                g1[y] -= 1
                g = g + hard * g1
                g_err = g_err + abs(hard) * q1 * (d_e1 + s_err1 + 4 * U)
                g_err[y] += abs(hard) * 4 * U
        loss[r] *= w
        lerr[r] = abs(w) * lerr[r] + 2 * U * abs(loss[r])
        delta[r] = -w * g
        derr[r] = abs(w) * g_err + half_step(delta[r], kind) + 4 * U * np.abs(delta[r])
    return loss, lerr, delta, derr
