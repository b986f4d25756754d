"""Plain forms, in long double and whole numbers, of RMS norm, rows in 8 bits and
log probabilities of tokens, with bounds for computations in the kernels'
precision: straight from the definitions in include/neural_api.h."""

import numpy as np

from sublayer_ref import D, U

L = np.longdouble


def tiny_of(dt):
    return np.finfo(dt).smallest_subnormal


def rms(h, gamma, eps):
    """out, rstd and their bounds.  A sum of C squares in any order is off by (C + 1) D of
    itself, the division and eps by 2 D, the root by half of that and 4 D; out has two more
    products, and the rounding to the type."""
    hl, C, u = h.astype(L), h.shape[-1], U[h.dtype]
    g = np.ones(C, L) if gamma is None else gamma.astype(L)
    with np.errstate(all="ignore"):
        total = (hl * hl).sum(-1)
        rstd = 1 / np.sqrt(total / C + L(eps))
        rstd = np.where(np.isfinite(total.astype(np.float64)), rstd, L(np.nan))
        out = hl * rstd[..., None] * g
        er = 0.5 * (C + 4) * D + 4 * D
        tiny = tiny_of(h.dtype)
        return (out, rstd), (1.01 * (u + er + 3 * D) * np.abs(out) + tiny, 1.01 * (u + er) * np.abs(rstd) + tiny)


def rms_grad(dy, h, gamma, rstd, dh, parts):
    """grad_in, grad_gamma from the given rstd, and bounds (those of the layer norm's
    gradient without its mean; with dh a second rounding, of the sum)."""
    C, u = h.shape[-1], U[h.dtype]
    R = h.size // C
    dy, hl, r = dy.astype(L).reshape(R, C), h.astype(L).reshape(R, C), rstd.astype(L)[:, None]
    g = np.ones(C, L) if gamma is None else gamma.astype(L)
    xh, w = hl * r, dy * g
    c2 = (w * xh).mean(-1, keepdims=True)
    dx = r * (w - xh * c2)
    e2 = (C + 8) * D * np.abs(w * xh).mean(-1, keepdims=True)
    ex = np.abs(r) * (np.abs(xh) * e2 + 6 * D * (np.abs(w) + np.abs(xh * c2)))
    bx = u * np.abs(dx) + ex
    if dh is not None:
        bx = bx + u * np.abs(dx + dh.astype(L).reshape(R, C))
        dx = dx + dh.astype(L).reshape(R, C)
    dg, ag = (dy * xh).sum(0), np.abs(dy * xh).sum(0)
    rows = (R + 8) * D + (u if parts > 1 else 0.0)
    tiny = tiny_of(h.dtype) * (1 + parts)
    return ((dx.reshape(h.shape), dg),
            ((1.02 * bx + tiny).reshape(h.shape), 1.01 * (u * np.abs(dg) + rows * ag) + tiny))


def codes(w):
    """Codes (int64) and max |w| of rows of float64 values: 127 w / a to the nearest whole
    number, halves away from zero, decided by whole-number products that long double holds
    exactly (53 + 8 bits)."""
    a = np.abs(w).max(-1)
    live = np.isfinite(a) & (a > 0)
    al = np.where(live, a, 1.0).astype(L)[..., None]
    with np.errstate(all="ignore"):
        m = np.where(live[..., None], np.abs(w), 0.0).astype(L)
        b = np.floor(m * 127 / al + L(0.5))
        b = np.where(254 * m >= (2 * b + 1) * al, b + 1, b)
        b = np.where(254 * m < (2 * b - 1) * al, b - 1, b)
        return np.where(w < 0, -b, b).astype(np.int64), a


def quantized(w, dt, by=None):
    """codes, scale (rounded to dt) of rows w, as the library leaves them; by: what the codes'
    values are multiplied by."""
    c, a = codes(w)
    with np.errstate(all="ignore"):
        s = a.astype(L) / 127 * (1 if by is None else by)
        s = np.where(np.isfinite(a), s, L(np.nan))
    return c, s


def logprobs(x, tokens, k, temperature):
    """lse, logprob, entropy, ids, top log probabilities and bounds of the first three.

    The kernels take d = x - m (off by u |d|), its exponential to 8 u (an exp2 within an ulp,
    2 u, of an argument kept to u beyond its rounding, and two products), and sum in double
    with a correction; the largest term is exactly 1.  So s is off by u sum' e (8 + |d| / T),
    and t = sum e d / T by that with one factor of d more.  f64 rows: D in the place of u, and D
    per term of the sums."""
    rows, V = x.shape
    u = U[x.dtype]
    xl = x.astype(L)
    with np.errstate(all="ignore"):
        m = np.where(np.isneginf(xl), L(-np.inf), xl).max(1)
        m0 = np.where(np.isneginf(m), L(0), m)
        d = (xl - m0[:, None]) / L(temperature)
        e = np.exp(d)
        dz = np.where(np.isneginf(d), L(0), d)
        s = e.sum(1)
        t = (e * dz).sum(1)
        ls = np.log(s)
        lse = m0 / L(temperature) + ls
        entropy = np.where(s == 0, L(0), ls - t / s)
        mine = np.where(dz == 0, L(0), e)  # terms that are not exactly 1
        es = u * (mine * (8 + np.abs(dz))).sum(1) / s + (V + 8) * D * 2
        et = u * (mine * np.abs(dz) * (8 + np.abs(dz))).sum(1) / s + (V + 8) * D * 2 * np.abs(t / s)
        tok = np.clip(tokens, 0, V - 1)
        zt = (xl[np.arange(rows), tok] - m0) / L(temperature)
        lp = np.where(s == 0, L(-np.inf), zt - ls)
        lp = np.where(tokens >= V, L(np.nan), lp)
        tiny = tiny_of(x.dtype)
        blse = 1.01 * (u * np.abs(lse) + es + 4 * D * (np.abs(m0 / temperature) + np.abs(ls))) + tiny
        blp = 1.01 * (u * np.abs(lp) + es + 4 * D * (np.abs(zt) + np.abs(ls))) + tiny
        bent = 1.01 * (u * np.abs(entropy) + es * (1 + np.abs(t / s)) + et + 4 * D * np.abs(ls)) + tiny
        order = np.argsort(-x, axis=1, kind="stable")[:, :k]
        if order.shape[1] < k:
            order = np.concatenate([order, np.zeros((rows, k - order.shape[1]), order.dtype)], 1)
        best = np.take_along_axis(x, order, 1).astype(L)
        none = np.isneginf(best) | (np.arange(k) >= V)
        ids = np.where(none, -1, order)
        top = np.where(none, L(-np.inf), (best - m0[:, None]) / L(temperature) - ls[:, None])
        btop = 1.01 * (u * np.abs(top) + es[:, None] + 4 * D * (np.abs(best - m0[:, None]) / temperature
                                                                 + np.abs(ls)[:, None])) + tiny
        bad = np.isnan(s)
        ids = np.where(bad[:, None], -1, ids)
        top = np.where(bad[:, None], L(np.nan), top)
    off = tokens < 0
    for v, fill in ((lse, 0), (lp, 0), (entropy, 0), (ids, -1), (top, -np.inf)):
        v[off] = fill
    return {"lse": lse, "logprob": lp, "entropy": entropy, "ids": ids, "top": top}, \
        {"lse": blse, "logprob": blp, "entropy": bent, "top": btop}


def logprobs_grad(x, tokens, g, e, lse, entropy, temperature):
    """The gradient from the saved lse and entropy, and its bound: log p in double (3 D of its
    terms), p off by 8 u, three roundings to u of the terms and the result."""
    rows, V = x.shape
    u = U[x.dtype]
    inv = 1 / L(temperature)
    with np.errstate(all="ignore"):
        z = x.astype(L) * inv
        ls = lse.astype(L)[:, None]
        lp = z - ls
        p = np.exp(lp)
        at = (np.arange(V) == (tokens[:, None] if tokens is not None else -1)).astype(L)
        gl = np.zeros((rows, 1), L) if g is None else g.astype(L)[:, None]
        el = np.zeros((rows, 1), L) if e is None else e.astype(L)[:, None]
        h = np.zeros((rows, 1), L) if e is None else entropy.astype(L)[:, None]
        lz = np.where(p == 0, L(0), lp + h)
        grad = (gl * (at - p) - el * p * lz) * inv
        dp = p * (8 * u + 4 * D * (np.abs(z) + np.abs(ls)))
        dp = np.where(p == 0, L(0), dp)
        dl = np.where(p == 0, L(0), 4 * D * (np.abs(z) + np.abs(ls) + np.abs(h)) + u * np.abs(lz))
        err = np.abs(gl) * (dp + 2 * u * np.abs(at - p)) + np.abs(el) * (dp * np.abs(lz) + p * dl + 3 * u * p * np.abs(lz))
        bound = 1.02 * inv * err + 2 * u * np.abs(grad) + 4 * tiny_of(x.dtype) * (1 + np.abs(gl) + np.abs(el) + inv)
        if g is not None and tokens is not None:
            grad = np.where((tokens >= V)[:, None], L(np.nan), grad)
        zero = np.isneginf(lse)
        if tokens is not None:
            zero = zero | (tokens < 0)
        grad = np.where(zero[:, None], L(0), grad)
    return grad, bound
