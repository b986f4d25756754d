"""Plain 64-bit (and longer) forms of layer norm, counter-based dropout and their
join, for the tests: loops and reductions of numpy, straight from the
definitions in include/neural_api.h."""

import numpy as np

U = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float64): 2.0 ** -53}
D = 2.0 ** -53  # one rounding of the kernels' double arithmetic

M32 = np.uint64(0xFFFFFFFF)


def philox(block, offset, seed):
    """[n] 64-bit block numbers -> [n, 4] 32-bit words of Philox4x32-10 with
    counter (block, offset) and key seed."""
    block = np.asarray(block, dtype=np.uint64)
    s32 = np.uint64(32)
    c = [block & M32, block >> s32, np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s32) ^ c[1] ^ np.uint64(k[0]), p1 & M32, (p0 >> s32) ^ c[3] ^ np.uint64(k[1]), p0 & M32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1)


def draws(first, n, seed, offset):
    """The 32-bit draws of elements first .. first + n - 1."""
    g0, g1 = first // 8, (first + n + 7) // 8
    g = np.arange(g0, g1, dtype=np.uint64)
    r = np.zeros((g1 - g0, 8), dtype=np.uint64)
    for half, shift in ((0, 16), (1, 0)):
        w = philox(g * np.uint64(2) + np.uint64(half), offset, seed)
        for e in range(8):
            v = (w[:, e // 2] >> np.uint64(16 * (e % 2))) & np.uint64(0xFFFF)
            r[:, e] |= v << np.uint64(shift)
    return r.reshape(-1)[first - 8 * g0: first - 8 * g0 + n]


def keep(n, p, seed, offset, first=0):
    return draws(first, n, seed, offset) >= np.uint64(round(p * 2 ** 32))


def dropout(x, p, seed, offset, first=0):
    """Exactly what the library computes: one product in x's type, or +0."""
    k = keep(x.size, p, seed, offset, first).reshape(x.shape)
    scale = x.dtype.type(1.0 / (1.0 - p)) if p < 1.0 else x.dtype.type(0)
    with np.errstate(all="ignore"):
        return np.where(k, x * scale, x.dtype.type(0))


def norm(x, gamma, beta, eps):
    """y, mean, rstd in long double, and their error bounds for a computation
    in double that rounds each result once to x's type.

    Sums of C terms in any order are off by at most C D sum|terms|, so the mean
    by C D mean|x| =: em; the centred values by em + D |d|; their squares' sum
    by C D relative and 2 em sum|d| + C em^2 (the first order term: sum d = 0
    only exactly); rstd by half of that relative, and four roundings."""
    L = np.longdouble
    x64, C = x.astype(L), x.shape[-1]
    u = U[x.dtype]
    with np.errstate(all="ignore"):
        mean = x64.sum(-1) / C
        d = x64 - mean[..., None]
        var = (d * d).sum(-1) / C
        rstd = 1 / np.sqrt(var + L(eps))
        g = np.ones(C, L) if gamma is None else gamma.astype(L)
        b = np.zeros(C, L) if beta is None else beta.astype(L)
        xh = d * rstd[..., None]
        y = xh * g + b
        em = (C + 2) * D * np.abs(x64).mean(-1)
        # (var + eps)'s relative error; em^2 and 2 em mean|d| against it
        ev = (C + 6) * D + (em * em + 2 * em * np.abs(d).mean(-1)) * rstd * rstd
        er = 0.5 * ev + 4 * D
        ey = np.abs(g) * (em[..., None] * rstd[..., None] + np.abs(xh) * (er[..., None] + 4 * D)) + 2 * D * np.abs(y)
    # 1.01: products of two bounds above; a subnormal result is rounded to an absolute step
    tiny = np.finfo(x.dtype).smallest_subnormal
    return (y, mean, rstd), (1.01 * (u * np.abs(y) + ey) + tiny, 1.01 * (u * np.abs(mean) + em) + tiny,
                             1.01 * (u * np.abs(rstd) + er * np.abs(rstd)) + tiny)


def norm_grad(dy, x, gamma, mean, rstd, parts):
    """dx, dgamma, dbeta in long double from the given statistics, and bounds.
    `parts`: the sums over rows may round that many partial sums to x's type."""
    L = np.longdouble
    C, u = x.shape[-1], U[x.dtype]
    R = x.size // C
    dy, xl = dy.astype(L).reshape(R, C), x.astype(L).reshape(R, C)
    m, r = mean.astype(L)[:, None], rstd.astype(L)[:, None]
    g = np.ones(C, L) if gamma is None else gamma.astype(L)
    xh = (xl - m) * r
    w = dy * g
    c1, c2 = w.mean(-1, keepdims=True), (w * xh).mean(-1, keepdims=True)
    dx = r * (w - c1 - xh * c2)
    dg, db = (dy * xh).sum(0), dy.sum(0)
    # the terms of each sum carry up to four roundings, the sums C (or R) more
    e1, e2 = (C + 4) * D * np.abs(w).mean(-1, keepdims=True), (C + 8) * D * np.abs(w * xh).mean(-1, keepdims=True)
    ex = r * (e1 + np.abs(xh) * e2 + 6 * D * (np.abs(w) + np.abs(c1) + np.abs(xh * c2)))
    ag, ab = np.abs(dy * xh).sum(0), np.abs(dy).sum(0)
    rows = (R + 8) * D + (u if parts > 1 else 0.0)  # a partial is off by u of itself, at most u of its terms' sizes
    tiny = np.finfo(x.dtype).smallest_subnormal * (1 + parts)
    return ((dx.reshape(x.shape), dg, db),
            ((1.01 * (u * np.abs(dx) + ex) + tiny).reshape(x.shape), 1.01 * (u * np.abs(dg) + rows * ag) + tiny,
             1.01 * (u * np.abs(db) + rows * ab) + tiny))


def within(got, want, bound, what=""):
    """|got - want| <= bound elementwise, NaN and infinities by class."""
    got, want = np.asarray(got), np.asarray(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    gn, wn = np.isnan(got), np.isnan(want)
    assert np.array_equal(gn, wn), f"{what}: NaN positions differ ({int((gn != wn).sum())})"
    gi, wi = np.isinf(got), np.isinf(want)
    assert np.array_equal(np.where(gi, got, 0), np.where(wi, want, 0).astype(got.dtype)), f"{what}: infinities differ"
    m = ~(gn | gi)
    err = np.abs(got[m].astype(np.longdouble) - want[m])
    lim = np.broadcast_to(bound, got.shape)[m]
    bad = np.nonzero(err > lim)[0]
    assert bad.size == 0, (f"{what}: {bad.size} of {err.size} past their bound, worst "
                           f"{float(np.max(err[bad] / lim[bad])):.3g} times; got {got[m][bad[0]]!r} want "
                           f"{float(want[m][bad[0]])!r}")
