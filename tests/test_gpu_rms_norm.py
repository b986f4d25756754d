"""RMS norm with the residual's addition, its gradient, its output in 8 bits, and rows in 8
bits, against long double forms (tests/serving_ref.py) with bounds that count
roundings; codes exactly.  Widths around every group size and past the
registers, few and many rows, extreme rows, in place, alignment, streams,
graphs, threads and the refusals."""

import numpy as np
import pytest

import serving_ref as ref
import sublayer_ref
from conftest import GPU, same_bits
from sublayer_ref import within

pytestmark = GPU

DT = [np.float32, np.float64]
EPS = 1e-6
COLS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 19, 31, 33, 64, 65, 67, 96, 127, 128, 130, 197, 255, 256, 257, 260, 511, 512,
        514, 577, 768, 1001, 1023, 1024, 1025, 1032, 2047, 2048, 2049, 4095, 4096, 4097, 4104, 8191, 8192, 8193, 8200,
        16384, 16385]
WIDE = [32767, 32768, 32769, 65536, 65539, 70001]


def _p(t):
    return t._ptr if t is not None else None


def _case(rng, rows, cols, dt):
    x = rng.normal(0.1, 1.5, (rows, cols))
    x[:, rng.integers(0, cols, 1 + cols // 200)] *= 20
    return {"x": x.astype(dt), "res": rng.normal(0, 2, (rows, cols)).astype(dt),
            "g": rng.normal(1, 0.3, cols).astype(dt), "dy": rng.normal(0, 1, (rows, cols)).astype(dt),
            "dh": rng.normal(0, 1, (rows, cols)).astype(dt)}


def _forward(pn, x, res, g, eps=EPS, hidden=True):
    T = pn.Tensor
    tx, tr, tg = (None if v is None else T.from_numpy(v) for v in (x, res, g))
    R = int(np.prod(x.shape[:-1]))
    y, rstd = T.create(x.shape, tx.dtype), T.create([R], tx.dtype)
    h = T.create(x.shape, tx.dtype) if hidden and res is not None else None
    assert pn.core._lib.neural_rms_norm_forward(y._ptr, _p(h), tx._ptr, _p(tr), _p(tg), eps, rstd._ptr) == 0
    return y.numpy(), (h.numpy() if h is not None else None), rstd.numpy()


def _codes_of(pn, rows, cols, stride, dtype, call):
    """(codes, scale, the bytes between the rows) of call(codes' address, scale's pointer)."""
    import torch
    raw = torch.full((rows * stride + 64,), 77, dtype=torch.int8, device="cuda")
    scale = pn.Tensor.create([rows], dtype)
    torch.cuda.synchronize()
    assert call(raw.data_ptr(), scale._ptr) == 0
    pn.synchronize()
    raw = raw.cpu().numpy()
    grid = raw[:rows * stride].reshape(rows, stride)
    assert (raw[rows * stride:] == 77).all() and (grid[:, cols:] == 77).all()
    return grid[:, :cols].astype(np.int64), scale.numpy()


def _forward_q8(pn, x, res, g, eps=EPS, stride=None):
    T, lib = pn.Tensor, pn.core._lib
    tx, tr, tg = (None if v is None else T.from_numpy(v) for v in (x, res, g))
    h = T.create(x.shape, tx.dtype) if res is not None else None
    rows, cols = x.shape
    st = stride or cols
    c, s = _codes_of(pn, rows, cols, st, tx.dtype,
                     lambda q, sc: lib.neural_rms_norm_forward_q8(q, st, sc, _p(h), tx._ptr, _p(tr), _p(tg), eps))
    return c, s, h.numpy() if h is not None else None


def _quantize(pn, x, stride=None):
    tx = pn.Tensor.from_numpy(x)
    rows, cols = x.shape
    st = stride or cols
    return _codes_of(pn, rows, cols, st, tx.dtype,
                     lambda q, sc: pn.core._lib.neural_quantize_rows(q, st, sc, tx._ptr))


def _backward(pn, dy, h, g, rstd, dh=None, want=("dx", "dg")):
    T = pn.Tensor
    t = [None if v is None else T.from_numpy(v) for v in (dy, dh, h, g, rstd)]
    dx, dg = T.create(h.shape, t[2].dtype), T.create([h.shape[-1]], t[2].dtype)
    assert pn.core._lib.neural_rms_norm_backward(dx._ptr if "dx" in want else None, dg._ptr if "dg" in want else None,
                                                 *[_p(v) for v in t]) == 0
    return dx.numpy() if "dx" in want else None, dg.numpy() if "dg" in want else None


def _check_forward(pn, x, res, g, eps=EPS):
    y, h, rstd = _forward(pn, x, res, g, eps)
    total = x if res is None else res + x
    if res is not None:
        same_bits(h, total)
        same_bits(_forward(pn, x, res, g, eps, hidden=False)[0], y)
    (wy, wr), (by, br) = ref.rms(total, g, eps)
    within(y, wy, by, "out")
    within(rstd, wr, br, "rstd")
    return y, total, rstd


def _check_codes(pn, x, res, g, eps=EPS, stride=None):
    total = x if res is None else res + x
    c, s, h = _forward_q8(pn, x, res, g, eps, stride)
    if res is not None:
        same_bits(h, total)
    with np.errstate(all="ignore"):
        w = total.astype(np.float64) * (1.0 if g is None else g.astype(np.float64))
    (_, rstd), (_, br) = ref.rms(total, g, eps)
    cols, u = x.shape[1], ref.U[x.dtype]
    with np.errstate(all="ignore"):
        want, scale = ref.quantized(w, x.dtype, by=rstd)
        bound = 1.01 * (u + 0.5 * (cols + 4) * ref.D + 8 * ref.D) * np.abs(scale) + ref.tiny_of(x.dtype)
    assert np.array_equal(c, want), np.argwhere(c != want)[:3]
    within(s, scale, bound, "scale")


def _check_quantize(pn, x, stride=None):
    c, s = _quantize(pn, x, stride)
    want, scale = ref.quantized(x.astype(np.float64), x.dtype)
    assert np.array_equal(c, want), np.argwhere(c != want)[:3]
    with np.errstate(all="ignore"):
        within(s, scale, 1.01 * (ref.U[x.dtype] + ref.D) * np.abs(scale) + ref.tiny_of(x.dtype), "scale")
    return c, s


def _check_all(pn, rng, rows, cols, dt):
    c = _case(rng, rows, cols, dt)
    _, h0, rstd0 = _check_forward(pn, c["x"], None, c["g"])
    y, h, rstd = _check_forward(pn, c["x"], c["res"], c["g"])
    same_bits(_forward(pn, h, None, c["g"])[0], y)  # the joined form is the norm of the sum
    _check_codes(pn, c["x"], c["res"], c["g"])
    _check_codes(pn, c["x"], None, None, stride=cols + 5)
    _check_quantize(pn, c["x"], stride=cols + 3)
    for dh in (c["dh"], None):
        dx, dg = _backward(pn, c["dy"], h, c["g"], rstd, dh)
        (wx, wg), (bx, bg) = ref.rms_grad(c["dy"], h, c["g"], rstd, dh, parts=rows)
        within(dx, wx, bx, "dx")
        within(dg, wg, bg, "dgamma")
        same_bits(_backward(pn, c["dy"], h, c["g"], rstd, dh, ("dx",))[0], dx)
        same_bits(_backward(pn, c["dy"], h, c["g"], rstd, dh, ("dg",))[1], dg)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", COLS)
def test_widths(pn, rng, dt, cols):
    _check_all(pn, rng, 5 if cols > 64 else 131, cols, dt)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", WIDE)
def test_wide_rows(pn, rng, dt, cols):
    _check_all(pn, rng, 3, cols, dt)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 768), (2, 4096), (70000, 5), (40000, 16), (20011, 40), (9001, 100),
                                       (5000, 260), (4500, 520), (2100, 1030), (1300, 2100), (1100, 4099), (700, 6001)])
def test_row_counts(pn, rng, dt, rows, cols):
    _check_all(pn, rng, rows, cols, dt)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(511, 40), (512, 1001), (513, 1001), (513, 8192), (2049, 2048), (777, 6001),
                                       (600, 12003), (700, 16385), (520, 33000), (20000, 12), (6000, 130), (1200, 4100),
                                       (600, 70001)])
def test_column_sums_exact(pn, dt, rows, cols):
    """Small whole numbers and rstd 1: every sum of dgamma is a whole number below 2^24, so any
    order gives the same bits; dx to its bound (torch in double)."""
    import torch
    tdt = torch.float32 if dt == np.float32 else torch.float64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows * 7 + cols)
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=gen).to(tdt)  # noqa: E731
    x, dy, g, dh = draw(-3, 4, rows, cols), draw(-3, 4, rows, cols), draw(1, 4, cols), draw(-3, 4, rows, cols)
    r = torch.ones(rows, dtype=tdt, device="cuda")
    dx, dg = torch.empty_like(x), torch.full_like(g, 9)
    t = [pn.Tensor.from_torch(v) for v in (dx, dg, dy, dh, x, g, r)]
    torch.cuda.synchronize()
    assert pn.core._lib.neural_rms_norm_backward(*[v._ptr for v in t]) == 0
    pn.synchronize()
    X, DY, W = x.double(), dy.double(), dy.double() * g.double()
    assert torch.equal(dg.double(), (DY * X).sum(0))
    want = W - X * (W * X).mean(1, keepdim=True)
    # W and X are at most 9 and 3, the mean's sum exact: under 16 roundings of values below 100, and
    # two to the type, of the value and of its sum with dh
    lim = 100 * 16 * ref.D + (ref.U[np.dtype(dt)] if dt == np.float32 else 0) * (2 * want.abs() + 3)
    assert bool(((dx.double() - (want + dh.double())).abs() <= lim).all())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [24, 300, 2050, 70001])
def test_extreme_rows(pn, rng, dt, cols):
    """Rows of one value, zeros, the largest and subnormal values, NaN and infinities: in the
    norm, in its codes, and in rows to 8 bits; other rows keep their bits."""
    x = rng.normal(0, 1, (12, cols)).astype(dt)
    clean = _forward(pn, x, None, None)
    codes, scale = _quantize(pn, x)
    x[0] = 3.25
    x[1] = 0.0
    x[2] = 3e38 if dt == np.float32 else 1e150
    x[3] = (1e-42 if dt == np.float32 else 1e-310) * rng.normal(0, 1, cols)
    x[4] = 1e-20
    x[4, 0] = 1e20
    x[5, cols // 2] = np.nan
    x[6, 0] = np.inf
    x[7, cols - 1] = -np.inf
    for eps in (EPS, 1e-12, 100.0):
        _check_forward(pn, x, None, None, eps)
        _check_codes(pn, x, None, None, eps)
    c, s = _check_quantize(pn, x)
    assert np.isnan(s[5:8]).all() and not c[5:8].any() and s[1] == 0 and not c[1].any()
    y, _, rstd = _forward(pn, x, None, None)
    assert np.isnan(y[5:8]).all() and np.isnan(rstd[5:8]).all()
    for a, b in ((y, clean[0]), (rstd, clean[2]), (c, codes), (s, scale)):
        assert np.array_equal(a[8:], b[8:])
    if dt == np.float64:  # products past the range of double
        big = np.full((2, cols), 1e300)
        big[1] = -1e308
        big[:, 0] = 1.7e308
        _check_quantize(pn, big)
        _check_quantize(pn, np.full((2, cols), 5e-324))


@pytest.mark.parametrize("dt", DT)
def test_codes_at_halves(pn, dt):
    """Values that lie exactly on a half of a step, and one unit in the last place beside it,
    at largest values that are powers of two, odd, and far from exact in binary."""
    rows = []
    for a in (127.0, 254.0, 1.0, 3.0, 127.0 / 3, 0.1, 6.35e-20, 12345.678):
        a = dt(a)
        half = (np.arange(0, 127) + 0.5) * float(a) / 127  # (the nearest to a half that the type holds)
        v = half.astype(dt)
        vals = np.concatenate([v, np.nextafter(v, dt(np.inf)), np.nextafter(v, dt(0))])
        rows.append(np.concatenate([vals, -vals, [a]]))
    x = np.array(rows, dtype=dt)
    _check_quantize(pn, x)
    _check_codes(pn, x, None, None)
    c, _ = _quantize(pn, np.array([[254.0, 1.0, -1.0, 3.0, 5.0]], dtype=dt))  # 0.5, 1.5, 2.5 steps
    assert c.tolist() == [[127, 1, -1, 2, 3]]


def _numeric(f, x, at, step):
    lo, hi = x.copy(), x.copy()
    lo.reshape(-1)[at] -= step
    hi.reshape(-1)[at] += step
    return (f(hi) - f(lo)) / (hi.reshape(-1)[at] - lo.reshape(-1)[at])


def test_gradients_by_differences(pn, rng):
    """f64: against central differences of a weighted sum of both outputs (step^2 / 6 times a
    third derivative of order 10, and D of a sum of 1e2 over the step: 2e-8; held to 1e-6)."""
    c = _case(rng, 3, 21, np.float64)
    c["x"] = rng.normal(0, 1, (3, 21))

    def loss(**kw):
        v = {**c, **kw}
        y, h, _ = _forward(pn, v["x"], v["res"], v["g"])
        return float((y * c["dy"]).sum() + (h * c["dh"]).sum())

    _, h, rstd = _forward(pn, c["x"], c["res"], c["g"])
    dx, dg = _backward(pn, c["dy"], h, c["g"], rstd, c["dh"])
    for name, grad in (("x", dx), ("res", dx), ("g", dg)):
        for at in rng.choice(c[name].size, min(12, c[name].size), replace=False):
            d = _numeric(lambda v: loss(**{name: v}), c[name], at, 1e-4)
            assert abs(d - grad.reshape(-1)[at]) <= 1e-6 * max(1.0, abs(d)), (name, at)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [30, 64, 1001, 2048, 5000, 40000, 70001])
def test_in_place(pn, rng, dt, cols):
    lib, T = pn.core._lib, pn.Tensor
    c = _case(rng, 6, cols, dt)
    y, h, rstd = _forward(pn, c["x"], c["res"], c["g"])
    g, r = T.from_numpy(c["g"]), T.from_numpy(rstd)
    for out_over, hid_over in (("x", "res"), ("res", "x"), ("x", None), ("res", None), (None, "res"), (None, "x")):
        t = {k: T.from_numpy(c[k]) for k in ("x", "res")}
        out = t[out_over] if out_over else T.create(c["x"].shape, g.dtype)
        hid = t[hid_over] if hid_over else None
        assert lib.neural_rms_norm_forward(out._ptr, _p(hid), t["x"]._ptr, t["res"]._ptr, g._ptr, EPS, None) == 0
        same_bits(out.numpy(), y)
        if hid is not None:
            same_bits(hid.numpy(), h)
    x = T.from_numpy(h)
    assert lib.neural_rms_norm_forward(x._ptr, None, x._ptr, None, g._ptr, EPS, None) == 0
    same_bits(x.numpy(), y)
    dx, dg = _backward(pn, c["dy"], h, c["g"], rstd, c["dh"])
    for over in ("dy", "dh", "h"):
        t = {"dy": T.from_numpy(c["dy"]), "dh": T.from_numpy(c["dh"]), "h": T.from_numpy(h)}
        tg = T.create([cols], g.dtype)
        assert lib.neural_rms_norm_backward(t[over]._ptr, tg._ptr, t["dy"]._ptr, t["dh"]._ptr, t["h"]._ptr, g._ptr,
                                            r._ptr) == 0
        same_bits(t[over].numpy(), dx)
        same_bits(tg.numpy(), dg)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [7, 96, 513, 1024, 3001, 9000, 70001])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_alignment_and_guards(pn, rng, dt, cols, shift):
    """Buffers that start anywhere give the bits of aligned ones, and nothing around the
    outputs is written."""
    import torch
    rows = 7
    c = _case(rng, rows, cols, dt)
    y, h, rstd = _forward(pn, c["x"], c["res"], c["g"])
    dx, dg = _backward(pn, c["dy"], h, c["g"], rstd, c["dh"])
    codes, scale, _ = _forward_q8(pn, c["x"], c["res"], c["g"])
    tdt = torch.float32 if dt == np.float32 else torch.float64
    held = []

    def placed(v):
        big = torch.full((v.size + 64,), 5.0, dtype=tdt, device="cuda")
        view = big[16 + shift:16 + shift + v.size].view(v.shape)
        view.copy_(torch.from_numpy(v))
        held.append((big, view, v.size))
        return pn.Tensor.from_torch(view), view

    t = {k: placed(v) for k, v in {**c, "h": h, "r": rstd}.items()}
    o = {k: placed(np.zeros_like(v)) for k, v in {"y": y, "oh": h, "or": rstd, "dx": dx, "dg": dg, "s": scale,
                                                  "qh": h}.items()}
    P = lambda k: (o.get(k) or t.get(k))[0]._ptr  # noqa: E731
    raw = torch.full((rows * cols + 64,), 9, dtype=torch.int8, device="cuda")
    torch.cuda.synchronize()
    lib = pn.core._lib
    assert lib.neural_rms_norm_forward(P("y"), P("oh"), P("x"), P("res"), P("g"), EPS, P("or")) == 0
    assert lib.neural_rms_norm_backward(P("dx"), P("dg"), P("dy"), P("dh"), P("h"), P("g"), P("r")) == 0
    assert lib.neural_rms_norm_forward_q8(raw.data_ptr() + 16 + shift, cols, P("s"), P("qh"), P("x"), P("res"), P("g"),
                                          EPS) == 0
    pn.synchronize()
    for k, want in (("y", y), ("oh", h), ("or", rstd), ("dx", dx), ("dg", dg), ("s", scale), ("qh", h)):
        same_bits(o[k][1].cpu().numpy(), want)
    got = raw.cpu().numpy()
    assert np.array_equal(got[16 + shift:16 + shift + rows * cols].reshape(rows, cols), codes)
    assert (got[:16 + shift] == 9).all() and (got[16 + shift + rows * cols:] == 9).all()
    for big, view, n in held:
        assert bool((big[:16 + shift] == 5).all()) and bool((big[16 + shift + n:] == 5).all())


def test_equal_calls_equal_bits(pn, rng):
    for rows, cols in ((5000, 96), (3000, 768), (700, 5001)):
        c = _case(rng, rows, cols, np.float32)
        _, _, rstd = _forward(pn, c["x"], None, c["g"])
        first = _backward(pn, c["dy"], c["x"], c["g"], rstd)
        for _ in range(3):
            for a, w in zip(_backward(pn, c["dy"], c["x"], c["g"], rstd), first):
                same_bits(a, w)


@pytest.mark.parametrize("dt", DT)
def test_host_buffers(pn, rng, dt):
    """Tensors and codes in host memory: written back by each call, the bytes between the
    codes' rows as they were."""
    c = _case(rng, 11, 100, dt)
    want = _forward(pn, c["x"], c["res"], c["g"])
    codes, scale, _ = _forward_q8(pn, c["x"], c["res"], c["g"])
    Z, lib = pn.Tensor.from_numpy_zero_copy, pn.core._lib
    y, h, r, s = np.zeros_like(c["x"]), np.zeros_like(c["x"]), np.zeros(11, dt), np.zeros(11, dt)
    t = {k: Z(v) for k, v in {**c, "y": y, "h": h, "r": r, "s": s}.items()}
    P = lambda k: t[k]._ptr  # noqa: E731
    assert lib.neural_rms_norm_forward(P("y"), P("h"), P("x"), P("res"), P("g"), EPS, P("r")) == 0
    for a, w in zip((y, h, r), want):
        same_bits(a, w)
    raw = np.full((11, 103), 7, np.int8)
    assert lib.neural_rms_norm_forward_q8(raw.ctypes.data, 103, P("s"), P("h"), P("x"), P("res"), P("g"), EPS) == 0
    assert np.array_equal(raw[:, :100], codes) and (raw[:, 100:] == 7).all()
    same_bits(s, scale)


def test_empty(pn):
    import torch
    lib, T = pn.core._lib, pn.Tensor
    x, g, m, y = T.create([0, 5]), T.ones([5]), T.create([0]), T.create([0, 5])
    raw = torch.zeros(16, dtype=torch.int8, device="cuda")
    assert lib.neural_rms_norm_forward(y._ptr, None, x._ptr, None, g._ptr, EPS, m._ptr) == 0
    assert lib.neural_quantize_rows(raw.data_ptr(), 5, m._ptr, x._ptr) == 0
    dg = T.ones([5])
    assert lib.neural_rms_norm_backward(y._ptr, dg._ptr, x._ptr, None, x._ptr, g._ptr, m._ptr) == 0
    assert not dg.numpy().any()


def test_refusals(pn):
    import torch
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    f, b = lib.neural_rms_norm_forward, lib.neural_rms_norm_backward
    q, n = lib.neural_rms_norm_forward_q8, lib.neural_quantize_rows
    x, w, y, h, z = (T.zeros([4, 6]) for _ in range(5))
    g, r, s, dg = T.ones([6]), T.zeros([4]), T.zeros([4]), T.zeros([6])
    X, W, Y, H, Z, G, R, S, DG = (t._ptr for t in (x, w, y, h, z, g, r, s, dg))
    raw = torch.zeros(64, dtype=torch.int8, device="cuda")
    C = raw.data_ptr()
    assert f(None, None, X, None, G, EPS, R) == E.NULL_POINTER and f(Y, None, None, None, G, EPS, R) == E.NULL_POINTER
    assert q(None, 6, S, None, X, None, G, EPS) == E.NULL_POINTER and q(C, 6, None, None, X, None, G, EPS) == E.NULL_POINTER
    assert n(C, 6, S, None) == E.NULL_POINTER
    assert b(None, None, Y, None, X, G, R) == E.NULL_POINTER and b(Z, DG, None, None, X, G, R) == E.NULL_POINTER
    assert b(Z, DG, Y, None, X, G, None) == E.NULL_POINTER
    d6, d46 = T.ones([6], pn.float64), T.zeros([4, 6], pn.float64)
    assert f(d46._ptr, None, X, None, G, EPS, R) == E.DTYPE_MISMATCH and f(Y, None, X, None, d6._ptr, EPS, R) == E.DTYPE_MISMATCH
    assert f(Y, None, X, d46._ptr, G, EPS, R) == E.DTYPE_MISMATCH and b(Z, d6._ptr, Y, None, X, G, R) == E.DTYPE_MISMATCH
    s5, s46 = T.ones([5]), T.zeros([6, 4])
    assert f(Y, None, X, None, s5._ptr, EPS, R) == E.SHAPE_MISMATCH and f(Y, None, X, s46._ptr, G, EPS, R) == E.SHAPE_MISMATCH
    assert q(C, 6, s5._ptr, None, X, None, G, EPS) == E.SHAPE_MISMATCH and b(Z, s5._ptr, Y, None, X, G, R) == E.SHAPE_MISMATCH
    s0, s0b = T.create([]), T.create([])
    assert f(s0b._ptr, None, s0._ptr, None, None, EPS, None) == E.DIM_MISMATCH
    for eps in (-1e-9, float("nan"), float("inf")):
        assert f(Y, None, X, None, G, eps, R) == E.INVALID_ARGUMENT and q(C, 6, S, None, X, None, G, eps) == E.INVALID_ARGUMENT
    assert f(Y, H, X, None, G, EPS, R) == E.INVALID_ARGUMENT       # hidden without a residual
    assert q(C, 5, S, None, X, None, G, EPS) == E.INVALID_ARGUMENT and n(C, 5, S, X) == E.INVALID_ARGUMENT
    assert n(C, 1 << 62, S, X) == E.TENSOR_TOO_LARGE
    t = torch.zeros(8, 6, device="cuda")
    strided, lower, upper = (T.from_torch(v) for v in (t[::2], t[:4], t[2:6]))
    assert f(strided._ptr, None, X, None, G, EPS, R) == E.INVALID_ARGUMENT
    assert f(upper._ptr, None, lower._ptr, None, G, EPS, R) == E.INVALID_ARGUMENT
    assert f(Y, Y, X, W, G, EPS, R) == E.INVALID_ARGUMENT
    assert b(Z, G, Y, None, X, G, R) == E.INVALID_ARGUMENT         # grad_gamma over gamma
    assert n(t.data_ptr(), 6, S, lower._ptr) == E.INVALID_ARGUMENT  # codes over the input
    assert n(x.device_ptr, 6, S, X) == E.INVALID_ARGUMENT
    assert q(C, 6, S, None, X, None, T.from_torch(raw.view(torch.float32)[:6])._ptr, EPS) == E.INVALID_ARGUMENT
    for v in (y, z, h):
        assert not v.numpy().any()
    assert not raw.cpu().numpy().any()
    one = T.ones([1, 6])  # of one row, grad_gamma may not replace the rows
    o1, r1 = T.ones([1, 6]), T.ones([1])
    assert b(None, o1._ptr, o1._ptr, None, one._ptr, G, r1._ptr) == E.INVALID_ARGUMENT
    assert b(Z, one._ptr, o1._ptr, None, one._ptr, G, r1._ptr) != E.OK


def test_graphs_and_streams(pn, rng):
    """Two captured steps (norm, codes, gradient) on two streams, replayed at once with the
    program's own calls in between: each its own workspace, every replay the eager result."""
    import torch
    lib, T = pn.core._lib, pn.Tensor
    rows, cols = 700, 1030
    streams, sides = [torch.cuda.Stream(), torch.cuda.Stream()], []
    try:
        for i in range(2):
            c = _case(rng, rows, cols, np.float32)
            t = {k: torch.from_numpy(v).cuda() for k, v in c.items()}
            for k, n in (("y", None), ("h", None), ("dx", None), ("r", rows), ("s", rows), ("dg", cols)):
                t[k] = torch.zeros(n if n else (rows, cols), device="cuda")
            q = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
            w = {k: T.from_torch(v) for k, v in t.items()}
            pn.set_stream(streams[i].cuda_stream)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[i]):
                P = lambda k: w[k]._ptr  # noqa: E731
                assert lib.neural_rms_norm_forward(P("y"), P("h"), P("x"), P("res"), P("g"), EPS, P("r")) == 0
                assert lib.neural_quantize_rows(q.data_ptr(), cols, P("s"), P("y")) == 0
                assert lib.neural_rms_norm_backward(P("dx"), P("dg"), P("dy"), P("dh"), P("h"), P("g"), P("r")) == 0
            sides.append((c, t, q, w, graph))
        pn.set_stream(None)
        torch.cuda.synchronize()
        for _ in range(3):
            for i, side in enumerate(sides):
                with torch.cuda.stream(streams[i]):
                    side[-1].replay()
            torch.cuda.synchronize()
            for c, t, q, w, graph in sides:
                y, h, r = _forward(pn, c["x"], c["res"], c["g"])
                codes, scale = _quantize(pn, y)
                dx, dg = _backward(pn, c["dy"], h, c["g"], r, c["dh"])
                for k, v in (("y", y), ("h", h), ("r", r), ("s", scale), ("dx", dx), ("dg", dg)):
                    same_bits(t[k].cpu().numpy(), v)
                    t[k].fill_(9.0)
                assert np.array_equal(q.cpu().numpy(), codes)
                q.fill_(3)
            lib.neural_hip_empty_cache()
            torch.cuda.synchronize()
    finally:
        pn.set_stream(None)


def test_threads(pn, rng):
    import threading
    cases = [_case(rng, 400 + 100 * i, 700 + 300 * i, np.float32) for i in range(4)]
    want = []
    for c in cases:
        _, _, r = _forward(pn, c["x"], None, c["g"])
        want.append((r, _backward(pn, c["dy"], c["x"], c["g"], r)))
    bad = []

    def work(i):
        for _ in range(5):
            got = _backward(pn, cases[i]["dy"], cases[i]["x"], cases[i]["g"], want[i][0])
            if not all(np.array_equal(a, b) for a, b in zip(got, want[i][1])):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_many_elements(pn):
    """More than 2^32 elements: the first and last rows of the norm, of codes and of the
    gradient (every row the same, so dgamma is rows times one row's product)."""
    import torch
    cols, rows = 4096, (1 << 20) + 3
    torch.cuda.empty_cache()
    pn.core._lib.neural_hip_empty_cache()
    if torch.cuda.mem_get_info()[0] < 10 * rows * cols:
        pytest.skip("not enough free device memory")
    lib, T = pn.core._lib, pn.Tensor
    one = torch.arange(cols, device="cuda", dtype=torch.float32) % 7 - 3
    x = one.repeat(rows, 1)
    q = torch.zeros(rows, cols, dtype=torch.int8, device="cuda")
    s, r, dg = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(cols, device="cuda")
    X, S, R, DG = (T.from_torch(v) for v in (x, s, r, dg))
    torch.cuda.synchronize()
    assert lib.neural_quantize_rows(q.data_ptr(), cols, S._ptr, X._ptr) == 0
    pn.synchronize()
    want = torch.sign(one) * torch.floor(one.abs() * 127 / 3 + 0.5)
    assert torch.equal(q[-1].float(), want) and torch.equal(q[0].float(), want) and bool((s == s[0]).all())
    y0 = one.repeat(2, 1)
    Y0 = T.from_torch(y0)
    torch.cuda.synchronize()
    assert lib.neural_rms_norm_forward(Y0._ptr, None, Y0._ptr, None, None, EPS, None) == 0
    assert lib.neural_rms_norm_forward(X._ptr, None, X._ptr, None, None, EPS, R._ptr) == 0
    pn.synchronize()
    assert torch.equal(x[-2:], y0) and torch.equal(x[:2], y0) and bool((r == r[0]).all())
    r.fill_(1.0)
    torch.cuda.synchronize()
    assert lib.neural_rms_norm_backward(None, DG._ptr, X._ptr, None, X._ptr, None, R._ptr) == 0
    pn.synchronize()
    d = y0[0].double()
    assert bool(((dg.double() - rows * d * d).abs() <= 2.0 ** -22 * rows * d * d).all())
    del X, x, q
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", DT)
def test_module(pn, rng, dt):
    """The module's forms are the entry points', its gradients go to an optimizer."""
    code = pn.float32 if dt == np.float32 else pn.float64
    c = _case(rng, 24, 190, dt)
    T = pn.Tensor
    m = pn.RMSNorm(190, dtype=code)
    m.gamma = T.from_numpy(c["g"])
    x, res = T.from_numpy(c["x"].reshape(4, 6, 190)), T.from_numpy(c["res"].reshape(4, 6, 190))
    y, h, rstd = _forward(pn, c["x"], c["res"], c["g"])
    out, hidden = m(x, res)
    same_bits(out.numpy().reshape(24, 190), y)
    same_bits(hidden.numpy().reshape(24, 190), h)
    dx, dg = _backward(pn, c["dy"], h, c["g"], rstd, c["dh"])
    gi = m.backward(T.from_numpy(c["dy"].reshape(4, 6, 190)), T.from_numpy(c["dh"].reshape(4, 6, 190)))
    same_bits(gi.numpy().reshape(24, 190), dx)
    same_bits(m.gamma.grad.numpy(), dg)
    same_bits(m(x).numpy().reshape(24, 190), _forward(pn, c["x"], None, c["g"])[0])
    q, hidden = m.forward_q8(x, res)
    codes, scale, _ = _forward_q8(pn, c["x"], c["res"], c["g"])
    assert np.array_equal(q.codes().reshape(24, 190), codes) and q.shape == (4, 6, 190)
    same_bits(q.scale.numpy(), scale)
    same_bits(hidden.numpy().reshape(24, 190), h)
    q2 = pn.QuantizedRows(x)
    codes, scale = _quantize(pn, c["x"])
    assert np.array_equal(q2.codes().reshape(24, 190), codes)
    same_bits(q2.numpy().reshape(24, 190), codes.astype(np.int8) * scale[:, None])
    opt = pn.AdamW(learning_rate=1e-2)
    before = m.gamma.numpy()
    opt.step(m.parameters(), [m.gamma.grad])
    assert not np.array_equal(before, m.gamma.numpy())
    with pytest.raises(ValueError):
        m(T.zeros([3, 191], code))
    assert sublayer_ref.D == ref.D
