"""Layer norm and its join with dropout and the residual add, forward and
backward, against long double forms of the definitions (tests/sublayer_ref.py)
with bounds that count roundings: widths around every group size and past the
registers, few and many rows, both dtypes, extreme rows, optional tensors, in
place, any alignment, streams, graphs, and the refusals."""

import ctypes

import numpy as np
import pytest

import sublayer_ref as ref
from conftest import GPU, keep, same_bits

pytestmark = GPU

DT = [np.float32, np.float64]
EPS = 1e-5
# group sizes end at these widths (f32, f64 half): 16 / 64 / 128 / 256 / 512 / 1024 / 2048 / ... values
COLS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 19, 20, 31, 33, 64, 65, 67, 96, 127, 128, 130, 197, 255, 256, 257, 260, 511,
        512, 514, 520, 577, 768, 1001, 1023, 1024, 1025, 1028, 1032, 2047, 2048, 2049, 2056, 4095, 4096, 4097, 4104,
        8191, 8192, 8193, 8200, 16384, 16385, 16392]
WIDE = [32767, 32768, 32769, 32776, 65536, 65539, 65544, 70001]


def _key(pn, seed, offset):
    return ctypes.byref(pn.core.DropoutKeyC(seed, offset))


def _p(t):
    return t._ptr if t is not None else None


def _rows(rng, rows, cols, dt):
    x = rng.normal(0.5, 1.5, (rows, cols))
    x[:, rng.integers(0, cols, 1 + cols // 200)] *= 20
    return x.astype(dt)


def _case(rng, rows, cols, dt):
    return {"x": _rows(rng, rows, cols, dt), "res": rng.normal(0, 2, (rows, cols)).astype(dt),
            "g": rng.normal(1, 0.3, cols).astype(dt), "b": rng.normal(0, 0.5, cols).astype(dt),
            "dy": rng.normal(0, 1, (rows, cols)).astype(dt), "dh": rng.normal(0, 1, (rows, cols)).astype(dt)}


def _forward(pn, x, g, b, eps=EPS):
    T = pn.Tensor
    tx, tg, tb = T.from_numpy(x), None if g is None else T.from_numpy(g), None if b is None else T.from_numpy(b)
    R = int(np.prod(x.shape[:-1]))
    y, mean, rstd = T.create(x.shape, tx.dtype), T.create([R], tx.dtype), T.create([R], tx.dtype)
    assert pn.core._lib.neural_layer_norm_forward(y._ptr, tx._ptr, _p(tg), _p(tb), eps, mean._ptr, rstd._ptr) == 0
    return y.numpy(), mean.numpy(), rstd.numpy()


def _backward(pn, dy, x, g, mean, rstd, want=("dx", "dg", "db")):
    T = pn.Tensor
    t = [T.from_numpy(v) if v is not None else None for v in (dy, x, g, mean, rstd)]
    C = x.shape[-1]
    outs = {"dx": T.create(x.shape, t[1].dtype), "dg": T.create([C], t[1].dtype), "db": T.create([C], t[1].dtype)}
    o = [outs[k]._ptr if k in want else None for k in ("dx", "dg", "db")]
    assert pn.core._lib.neural_layer_norm_backward(*o, *[_p(v) for v in t]) == 0
    return [outs[k].numpy() if k in want else None for k in ("dx", "dg", "db")]


def _joined(pn, c, p, key, eps=EPS, hidden=True):
    T = pn.Tensor
    x, res, g, b = (T.from_numpy(c[k]) for k in ("x", "res", "g", "b"))
    R = c["x"].size // c["x"].shape[-1]
    y, h = T.create(c["x"].shape, x.dtype), T.create(c["x"].shape, x.dtype) if hidden else None
    mean, rstd = T.create([R], x.dtype), T.create([R], x.dtype)
    assert pn.core._lib.neural_dropout_add_layer_norm_forward(y._ptr, _p(h), x._ptr, res._ptr, g._ptr, b._ptr, p,
                                                              key, eps, mean._ptr, rstd._ptr) == 0
    return y.numpy(), h.numpy() if hidden else None, mean.numpy(), rstd.numpy()


def _joined_grad(pn, c, h, mean, rstd, p, key, with_dh=True):
    T = pn.Tensor
    dy, dh, th, g, m, r = (T.from_numpy(v) for v in (c["dy"], c["dh"], h, c["g"], mean, rstd))
    C = h.shape[-1]
    dx, dres = T.create(h.shape, th.dtype), T.create(h.shape, th.dtype)
    dg, db = T.create([C], th.dtype), T.create([C], th.dtype)
    assert pn.core._lib.neural_dropout_add_layer_norm_backward(
        dx._ptr, dres._ptr, dg._ptr, db._ptr, dy._ptr, dh._ptr if with_dh else None, th._ptr, g._ptr, m._ptr, r._ptr,
        p, key) == 0
    return dx.numpy(), dres.numpy(), dg.numpy(), db.numpy()


def _check_forward(pn, x, g, b, eps=EPS):
    got = _forward(pn, x, g, b, eps)
    want, bound = ref.norm(x.reshape(-1, x.shape[-1]), g, b, eps)
    for name, o, w, lim in zip(("y", "mean", "rstd"), got, want, bound):
        ref.within(o.reshape(w.shape), w, lim, name)
    return got


def _check_all(pn, rng, rows, cols, dt, p=0.2):
    """Every form at one size: the stand-alone calls against the definitions, the
    joined ones against the stand-alone calls, bit for bit."""
    c = _case(rng, rows, cols, dt)
    _, mean, rstd = _check_forward(pn, c["x"], c["g"], c["b"])
    got = _backward(pn, c["dy"], c["x"], c["g"], mean, rstd)
    want, bound = ref.norm_grad(c["dy"], c["x"], c["g"], mean, rstd, parts=rows)
    for name, o, w, lim in zip(("dx", "dgamma", "dbeta"), got, want, bound):
        ref.within(o, w, lim, name)
    # only the input's gradient, and only the sums: the same bits
    same_bits(_backward(pn, c["dy"], c["x"], c["g"], mean, rstd, ("dx",))[0], got[0])
    only = _backward(pn, c["dy"], c["x"], c["g"], mean, rstd, ("dg", "db"))
    same_bits(only[1], got[1])
    same_bits(only[2], got[2])
    for q in (p, 0.0):
        key = _key(pn, 5, cols)
        h = c["res"] + (ref.dropout(c["x"], q, 5, cols) if q else c["x"])
        y, hg, m, r = _joined(pn, c, q, key if q else None)
        same_bits(hg, h)
        for o, w in zip((y, m, r), _forward(pn, h, c["g"], c["b"])):
            same_bits(o, w)
        same_bits(_joined(pn, c, q, key, hidden=False)[0], y)
        dx, dres, dg, db = _joined_grad(pn, c, h, m, r, q, key)
        sx, sg, sb = _backward(pn, c["dy"], h, c["g"], m, r)
        same_bits(dres, sx + c["dh"])
        same_bits(dx, ref.dropout(dres, q, 5, cols) if q else dres)
        same_bits(dg, sg)
        same_bits(db, sb)
        dx, dres, dg, db = _joined_grad(pn, c, h, m, r, q, key, with_dh=False)
        same_bits(dres, sx)
        same_bits(dx, ref.dropout(sx, q, 5, cols) if q else sx)


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
                                       (5000, 260), (4500, 520), (2100, 1030), (1300, 2100), (1100, 4099)])
def test_row_counts(pn, rng, dt, rows, cols):
    """One row, and more rows than the backward pass has groups of lanes."""
    _check_all(pn, rng, rows, cols, dt)


@pytest.mark.parametrize("dt", DT)
def test_optional_tensors(pn, rng, dt):
    """gamma or beta of ones / zeros and none give the same bits; statistics
    may be left out; leading dimensions do not matter."""
    lib, T = pn.core._lib, pn.Tensor
    x = _rows(rng, 24, 130, dt)
    one, zero = np.ones(130, dt), np.zeros(130, dt)
    y, mean, rstd = _check_forward(pn, x, None, None)
    for g, b in ((one, zero), (None, zero), (one, None)):
        same_bits(_forward(pn, x, g, b)[0], y)
    tx, ty = T.from_numpy(x.reshape(2, 3, 4, 130)), T.create([2, 3, 4, 130], T.from_numpy(x).dtype)
    assert lib.neural_layer_norm_forward(ty._ptr, tx._ptr, None, None, EPS, None, None) == 0
    same_bits(ty.numpy().reshape(24, 130), y)
    dy = rng.normal(0, 1, x.shape).astype(dt)
    for a, w in zip(_backward(pn, dy, x, None, mean, rstd), _backward(pn, dy, x, one, mean, rstd)):
        same_bits(a, w)
    v = T.from_numpy(x[0].copy())  # a rank-1 tensor is one row
    o = T.create([130], v.dtype)
    assert lib.neural_layer_norm_forward(o._ptr, v._ptr, None, None, EPS, None, None) == 0
    same_bits(o.numpy(), y[0])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(6, 50), (900, 50), (700, 5003), (3, 40000), (3, 70001)])
def test_each_output_alone(pn, rng, dt, rows, cols):
    """Every output of the backward calls left out in turn, or alone: the others
    keep their bits.  p of 1 drops the sublayer's output and its gradient."""
    lib, T = pn.core._lib, pn.Tensor
    c = _case(rng, rows, cols, dt)
    key = _key(pn, 6, 6)
    y, h, mean, rstd = _joined(pn, c, 0.3, key)
    want = _joined_grad(pn, c, h, mean, rstd, 0.3, key)
    dy, dh, th, g, m, r = (T.from_numpy(v) for v in (c["dy"], c["dh"], h, c["g"], mean, rstd))
    shapes = [h.shape, h.shape, [cols], [cols]]
    for take in ((0,), (1,), (2,), (3,), (0, 2), (1, 3), (0, 1), (1, 2, 3), (0, 2, 3)):
        o = [T.create(shapes[i], g.dtype) if i in take else None for i in range(4)]
        assert lib.neural_dropout_add_layer_norm_backward(*[_p(v) for v in o], dy._ptr, dh._ptr, th._ptr, g._ptr,
                                                          m._ptr, r._ptr, 0.3, key) == 0
        for i in take:
            same_bits(o[i].numpy(), want[i])
    y, h, mean, rstd = _joined(pn, c, 1.0, key)
    same_bits(h, c["res"] + dt(0))
    dx, dres, _, _ = _joined_grad(pn, c, h, mean, rstd, 1.0, key)
    assert not dx.any() and not np.signbit(dx).any() and dres.any()


@pytest.mark.parametrize("dt", DT)
def test_joined_on_host_buffers(pn, rng, dt):
    """Tensors over host memory in both joined calls, the hidden state in place
    of the residual, two wrappers of one buffer among them."""
    c = _case(rng, 9, 77, dt)
    key = _key(pn, 1, 5)
    y, h, mean, rstd = _joined(pn, c, 0.4, key)
    grads = _joined_grad(pn, c, h, mean, rstd, 0.4, key)
    Z, lib = pn.Tensor.from_numpy_zero_copy, pn.core._lib
    b = {k: v.copy() for k, v in c.items()}
    b.update(y=np.zeros_like(y), m=np.zeros_like(mean), r=np.zeros_like(rstd), dg=np.zeros_like(c["g"]),
             db=np.zeros_like(c["g"]))
    t = {k: Z(v) for k, v in b.items()}
    again = Z(b["res"])  # the same buffer: the hidden state goes over the residual
    assert lib.neural_dropout_add_layer_norm_forward(t["y"]._ptr, again._ptr, t["x"]._ptr, t["res"]._ptr, t["g"]._ptr,
                                                     t["b"]._ptr, 0.4, key, EPS, t["m"]._ptr, t["r"]._ptr) == 0
    for a, w in zip((b["y"], b["res"], b["m"], b["r"]), (y, h, mean, rstd)):
        same_bits(a, w)
    assert lib.neural_dropout_add_layer_norm_backward(t["dy"]._ptr, t["dh"]._ptr, t["dg"]._ptr, t["db"]._ptr,
                                                      t["dy"]._ptr, t["dh"]._ptr, t["res"]._ptr, t["g"]._ptr,
                                                      t["m"]._ptr, t["r"]._ptr, 0.4, key) == 0
    for a, w in zip((b["dy"], b["dh"], b["dg"], b["db"]), grads):
        same_bits(a, w)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [24, 300, 2050, 70001])
def test_extreme_rows(pn, rng, dt, cols):
    """Rows of one value, of a value far from their spread, of the largest and
    of subnormal values; eps of 0 and large."""
    x = _rows(rng, 12, cols, dt)
    x[0] = 3.25
    x[1] = 0.0
    x[2] = 1e6 + rng.normal(0, 1, cols)
    x[3] = -3e38 if dt == np.float32 else -1e150
    x[4] = (3e38 if dt == np.float32 else 1e150) * np.where(np.arange(cols) % 2, 1, -1)
    x[5] = 1e-42 * rng.normal(0, 1, cols)
    x[6] = 1e-20
    x[6, 0] = 1e20
    for eps in (EPS, 1e-12, 100.0):
        _check_forward(pn, x, None, None, eps)
    varied = x[7:]
    _check_forward(pn, varied, None, None, 0.0)
    # a constant row and eps = 0: (x - mean) / 0 = 0 / 0 where the mean is exact
    y = _forward(pn, np.full((2, 16), 3.0, dt), None, None, 0.0)
    assert np.isnan(y[0]).all() and np.isinf(y[2]).all() and (y[1] == 3.0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [10, 100, 777, 5000, 70001])
def test_nan_and_infinity_stay_in_their_rows(pn, rng, dt, cols):
    x = _rows(rng, 9, cols, dt)
    clean = _forward(pn, x, None, None)
    x[1, cols // 2] = np.nan
    x[4, 0] = np.inf
    x[7, cols - 1] = -np.inf
    y, mean, rstd = _forward(pn, x, None, None)
    bad = [1, 4, 7]
    assert np.isnan(y[bad]).all() and np.isnan(rstd[bad]).all()
    assert np.isnan(mean[1]) and mean[4] == np.inf and mean[7] == -np.inf
    good = [0, 2, 3, 5, 6, 8]
    for a, b in zip((y, mean, rstd), clean):
        same_bits(a[good], b[good])
    # dropped in the joined form, they are not there
    c = _case(rng, 4, cols, dt)
    keep = ref.keep(4 * cols, 0.5, 1, 2).reshape(4, cols)
    c["x"][~keep] = np.nan
    got = _joined(pn, c, 0.5, _key(pn, 1, 2))
    c["x"][~keep] = 0.0
    for a, b in zip(got, _joined(pn, c, 0.5, _key(pn, 1, 2))):
        same_bits(a, b)
    assert np.isfinite(got[0]).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(511, 40), (512, 1001), (513, 1001), (512, 8192), (513, 8192), (512, 8200),
                                       (2049, 2048), (777, 6001), (600, 12003), (700, 16385), (520, 33000), (20000, 12),
                                       (30001, 33), (6000, 130), (5003, 390), (1200, 4100), (600, 70001)])
def test_column_sums_exact(pn, dt, rows, cols):
    """Small whole numbers, mean 0 and rstd 1: every term and sum of dgamma and
    dbeta is a whole number below 2^24, so any order gives the same bits, in
    each form that the sizes select; dx to its bound (torch in double)."""
    import torch
    tdt = torch.float32 if dt == np.float32 else torch.float64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows * 7 + cols)
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=gen).to(tdt)  # noqa: E731
    x, dy, g = draw(-3, 4, rows, cols), draw(-3, 4, rows, cols), draw(1, 4, cols)
    m, r = torch.zeros(rows, dtype=tdt, device="cuda"), torch.ones(rows, dtype=tdt, device="cuda")
    dx, dg, db = torch.empty_like(x), torch.full_like(g, 9), torch.full_like(g, 9)
    T = pn.Tensor.from_torch
    t = [T(v) for v in (dx, dg, db, dy, x, g, m, r)]
    torch.cuda.synchronize()
    assert pn.core._lib.neural_layer_norm_backward(*[v._ptr for v in t]) == 0
    pn.synchronize()
    X, DY, W = x.double(), dy.double(), dy.double() * g.double()
    assert torch.equal(dg.double(), (DY * X).sum(0)) and torch.equal(db.double(), DY.sum(0))
    want = W - W.mean(1, keepdim=True) - X * (W * X).mean(1, keepdim=True)
    # W and X are at most 9 and 3, the means' sums exact: under 16 roundings of values below 100, and
    # the last to the type
    lim = 100 * 16 * ref.D + (ref.U[np.dtype(dt)] if dt == np.float32 else 0) * want.abs()
    assert bool(((dx.double() - want).abs() <= lim).all())


def _numeric(f, x, at, step):
    lo, hi = x.copy(), x.copy()
    lo.reshape(-1)[at] -= step
    hi.reshape(-1)[at] += step
    return (f(hi) - f(lo)) / (hi.reshape(-1)[at] - lo.reshape(-1)[at])


def test_gradients_by_differences(pn, rng):
    """f64: the joined form's gradients against central differences of a
    weighted sum of both its outputs.  The difference is off by step^2 / 6 times
    the third derivative (of order 10 here) and by roundings of the sum (of size
    1e2, D each) over the step: 1e-4 gives 2e-8 and 1e-9, held to 1e-6."""
    rows, cols, p = 3, 21, 0.3
    c = _case(rng, rows, cols, np.float64)
    c["x"] = rng.normal(0, 1, (rows, cols))
    key = _key(pn, 9, 9)

    def loss(**kw):
        y, h, _, _ = _joined(pn, {**c, **kw}, p, key)
        return float((y * c["dy"]).sum() + (h * c["dh"]).sum())

    _, h, mean, rstd = _joined(pn, c, p, key)
    dx, dres, dg, db = _joined_grad(pn, c, h, mean, rstd, p, key)
    for name, grad in (("x", dx), ("res", dres), ("g", dg), ("b", db)):
        for at in rng.choice(c[name].size, min(12, c[name].size), replace=False):
            d = _numeric(lambda v: loss(**{name: v}), c[name], at, 1e-4)
            assert abs(d - grad.reshape(-1)[at]) <= 1e-6 * max(1.0, abs(d)), (name, at, d, grad.reshape(-1)[at])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [30, 64, 1001, 2048, 5000, 40000, 70001])
def test_in_place(pn, rng, dt, cols):
    """Outputs over the inputs they may replace: the same bits."""
    lib, T = pn.core._lib, pn.Tensor
    c = _case(rng, 6, cols, dt)
    key = _key(pn, 3, 3)
    want = _forward(pn, c["x"], c["g"], c["b"])
    g, b = T.from_numpy(c["g"]), T.from_numpy(c["b"])
    x = T.from_numpy(c["x"])
    assert lib.neural_layer_norm_forward(x._ptr, x._ptr, g._ptr, b._ptr, EPS, None, None) == 0
    same_bits(x.numpy(), want[0])
    grads = _backward(pn, c["dy"], c["x"], c["g"], want[1], want[2])
    m, r = T.from_numpy(want[1]), T.from_numpy(want[2])
    for over in ("dy", "x"):
        t = {k: T.from_numpy(c[k]) for k in ("dy", "x")}
        dg, db = T.create([cols], g.dtype), T.create([cols], g.dtype)
        assert lib.neural_layer_norm_backward(t[over]._ptr, dg._ptr, db._ptr, t["dy"]._ptr, t["x"]._ptr, g._ptr,
                                              m._ptr, r._ptr) == 0
        for o, w in zip((t[over], dg, db), grads):
            same_bits(o.numpy(), w)
    y, h, hm, hr = _joined(pn, c, 0.3, key)
    for out_over, hid_over in (("x", "res"), ("res", "x"), ("x", None), ("res", None), (None, "res"), (None, "x")):
        t = {k: T.from_numpy(c[k]) for k in ("x", "res")}
        out = t[out_over] if out_over else T.create(c["x"].shape, g.dtype)
        hid = t[hid_over] if hid_over else None
        assert lib.neural_dropout_add_layer_norm_forward(out._ptr, _p(hid), t["x"]._ptr, t["res"]._ptr, g._ptr,
                                                         b._ptr, 0.3, key, EPS, None, None) == 0
        same_bits(out.numpy(), y)
        if hid is not None:
            same_bits(hid.numpy(), h)
    dx, dres, dg, db = _joined_grad(pn, c, h, hm, hr, 0.3, key)
    m, r = T.from_numpy(hm), T.from_numpy(hr)
    for dx_over, dres_over in (("dy", "dh"), ("dh", "dy"), ("h", "dh"), ("dh", "h"), ("dy", "h")):
        t = {"dy": T.from_numpy(c["dy"]), "dh": T.from_numpy(c["dh"]), "h": T.from_numpy(h)}
        tg, tb = T.create([cols], g.dtype), T.create([cols], g.dtype)
        assert lib.neural_dropout_add_layer_norm_backward(t[dx_over]._ptr, t[dres_over]._ptr, tg._ptr, tb._ptr,
                                                          t["dy"]._ptr, t["dh"]._ptr, t["h"]._ptr, g._ptr, m._ptr,
                                                          r._ptr, 0.3, key) == 0
        for o, w in zip((t[dx_over], t[dres_over], tg, tb), (dx, dres, dg, db)):
            same_bits(o.numpy(), w)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cols", [7, 96, 513, 1024, 3001, 9000, 70001])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_alignment_and_guards(pn, rng, dt, cols, shift):
    """Buffers that start anywhere give the bits of aligned ones, and nothing
    around the outputs is written."""
    import torch
    rows = 7
    c = _case(rng, rows, cols, dt)
    key = _key(pn, 2, 8)
    y, h, mean, rstd = _joined(pn, c, 0.1, key)
    grads = _joined_grad(pn, c, h, mean, rstd, 0.1, key)
    tdt = torch.float32 if dt == np.float32 else torch.float64
    held = []

    def placed(v):
        big = torch.full((v.size + 64,), 5.0, dtype=tdt, device="cuda")
        view = big[16 + shift:16 + shift + v.size].view(v.shape)
        view.copy_(torch.from_numpy(v))
        held.append((big, view, v.size))
        return pn.Tensor.from_torch(view), view

    def check(view, want):
        same_bits(view.cpu().numpy(), want)

    ins = {k: placed(v) for k, v in {**c, "h": h, "mean": mean, "rstd": rstd}.items()}
    outs = {k: placed(np.zeros_like(v)) for k, v in {"y": y, "oh": h, "om": mean, "or": rstd, "dx": grads[0],
                                                     "dres": grads[1], "dg": grads[2], "db": grads[3]}.items()}
    P = lambda k: (outs.get(k) or ins.get(k))[0]._ptr  # noqa: E731
    torch.cuda.synchronize()
    lib = pn.core._lib
    assert lib.neural_dropout_add_layer_norm_forward(P("y"), P("oh"), P("x"), P("res"), P("g"), P("b"), 0.1, key, EPS,
                                                     P("om"), P("or")) == 0
    assert lib.neural_dropout_add_layer_norm_backward(P("dx"), P("dres"), P("dg"), P("db"), P("dy"), P("dh"), P("h"),
                                                      P("g"), P("mean"), P("rstd"), 0.1, key) == 0
    pn.synchronize()
    for k, want in zip(("y", "oh", "om", "or", "dx", "dres", "dg", "db"), (y, h, mean, rstd, *grads)):
        check(outs[k][1], want)
    for big, view, n in held:
        assert bool((big[:16 + shift] == 5).all()) and bool((big[16 + shift + n:] == 5).all())


def test_equal_calls_equal_bits(pn, rng):
    for rows, cols in ((5000, 96), (3000, 768), (700, 5001)):
        c = _case(rng, rows, cols, np.float32)
        _, mean, rstd = _forward(pn, c["x"], c["g"], c["b"])
        first = _backward(pn, c["dy"], c["x"], c["g"], mean, rstd)
        for _ in range(3):
            for a, w in zip(_backward(pn, c["dy"], c["x"], c["g"], mean, rstd), first):
                same_bits(a, w)


def test_host_buffers(pn, rng):
    """Tensors over host memory: written back by each call."""
    c = _case(rng, 11, 100, np.float32)
    want = _forward(pn, c["x"], c["g"], c["b"])
    y, mean, rstd = np.zeros_like(c["x"]), np.zeros(11, np.float32), np.zeros(11, np.float32)
    Z = pn.Tensor.from_numpy_zero_copy
    t = [Z(v) for v in (y, c["x"], c["g"], c["b"], mean, rstd)]
    assert pn.core._lib.neural_layer_norm_forward(t[0]._ptr, t[1]._ptr, t[2]._ptr, t[3]._ptr, EPS, t[4]._ptr,
                                                  t[5]._ptr) == 0
    for a, w in zip((y, mean, rstd), want):
        same_bits(a, w)


def test_empty(pn):
    lib, T = pn.core._lib, pn.Tensor
    x, g, m = T.create([0, 5]), T.ones([5]), T.create([0])
    assert lib.neural_layer_norm_forward(x._ptr, x._ptr, g._ptr, g._ptr, EPS, m._ptr, None) == 0
    dg, db = T.ones([5]), T.ones([5])
    assert lib.neural_layer_norm_backward(x._ptr, dg._ptr, db._ptr, x._ptr, x._ptr, g._ptr, m._ptr, m._ptr) == 0
    assert not dg.numpy().any() and not db.numpy().any()  # sums over no rows
    e = T.create([5, 0])
    z = T.create([0])
    assert lib.neural_layer_norm_forward(e._ptr, e._ptr, z._ptr, z._ptr, EPS, None, None) == 0
    assert lib.neural_layer_norm_backward(e._ptr, None, None, e._ptr, e._ptr, None, z._ptr, z._ptr) == 0


def test_refusals(pn):
    import torch
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    f, k = lib.neural_layer_norm_forward, lib.neural_layer_norm_backward
    jf, jk = lib.neural_dropout_add_layer_norm_forward, lib.neural_dropout_add_layer_norm_backward
    x, y, z = T.zeros([4, 6]), T.zeros([4, 6]), T.zeros([4, 6])
    g, b, m, r = T.ones([6]), T.ones([6]), T.zeros([4]), T.zeros([4])
    X, Y, Z, G, B, M, R = (t._ptr for t in (x, y, z, g, b, m, r))
    key = _key(pn, 0, 0)
    assert f(None, X, G, B, EPS, M, R) == E.NULL_POINTER
    assert f(Y, None, G, B, EPS, M, R) == E.NULL_POINTER
    assert jf(Y, Z, X, None, G, B, 0.0, None, EPS, M, R) == E.NULL_POINTER
    w = T.zeros([4, 6])
    W = w._ptr
    assert jf(Y, Z, X, W, G, B, 0.5, None, EPS, M, R) == E.NULL_POINTER  # no key
    assert k(None, None, None, Y, X, G, M, R) == E.NULL_POINTER
    assert k(Z, None, None, None, X, G, M, R) == E.NULL_POINTER
    assert k(Z, None, None, Y, X, G, None, R) == E.NULL_POINTER
    assert k(Z, None, None, Y, X, G, M, None) == E.NULL_POINTER
    d6, d46 = T.ones([6], pn.float64), T.zeros([4, 6], pn.float64)
    assert f(d46._ptr, X, G, B, EPS, M, R) == E.DTYPE_MISMATCH
    assert f(Y, X, d6._ptr, B, EPS, M, R) == E.DTYPE_MISMATCH
    assert k(Z, d6._ptr, None, Y, X, G, M, R) == E.DTYPE_MISMATCH
    s5, s46, s24 = T.ones([5]), T.zeros([6, 4]), T.zeros([24])
    assert f(Y, X, s5._ptr, B, EPS, M, R) == E.SHAPE_MISMATCH
    assert f(Y, X, G, s5._ptr, EPS, M, R) == E.SHAPE_MISMATCH
    assert f(Y, X, G, B, EPS, s5._ptr, R) == E.SHAPE_MISMATCH
    assert f(s46._ptr, X, G, B, EPS, M, R) == E.SHAPE_MISMATCH
    assert f(s24._ptr, X, G, B, EPS, M, R) == E.SHAPE_MISMATCH
    assert k(Z, s5._ptr, None, Y, X, G, M, R) == E.SHAPE_MISMATCH
    assert k(Z, None, None, s46._ptr, X, G, M, R) == E.SHAPE_MISMATCH
    s0, s0b = T.create([]), T.create([])
    assert f(s0b._ptr, s0._ptr, None, None, EPS, None, None) == E.DIM_MISMATCH
    for eps in (-1e-9, float("nan"), float("inf")):
        assert f(Y, X, G, B, eps, M, R) == E.INVALID_ARGUMENT
    for p in (-0.1, 1.1, float("nan")):
        assert jf(Y, Z, X, W, G, B, p, key, EPS, M, R) == E.INVALID_ARGUMENT
        assert jk(Z, None, None, None, Y, None, X, G, M, R, p, key) == E.INVALID_ARGUMENT
    t = torch.zeros(8, 6, device="cuda")
    strided, lower, upper = (T.from_torch(v) for v in (t[::2], t[:4], t[2:6]))
    assert f(strided._ptr, X, G, B, EPS, M, R) == E.INVALID_ARGUMENT
    assert f(Y, strided._ptr, G, B, EPS, M, R) == E.INVALID_ARGUMENT
    assert f(upper._ptr, lower._ptr, G, B, EPS, M, R) == E.INVALID_ARGUMENT   # overlap, not in place
    assert f(Y, X, G, B, EPS, M, M) == E.INVALID_ARGUMENT                     # one tensor, two outputs
    assert jf(Y, Y, X, W, G, B, 0.0, None, EPS, M, R) == E.INVALID_ARGUMENT
    assert jk(Z, Z, None, None, Y, None, X, G, M, R, 0.5, key) == E.INVALID_ARGUMENT
    assert k(Z, G, None, Y, X, G, M, R) == E.INVALID_ARGUMENT                 # grad_gamma over gamma
    row = T.from_torch(t[0])
    assert k(Z, None, row._ptr, Y, lower._ptr, G, M, R) == E.INVALID_ARGUMENT  # grad_beta inside the input
    for v in (y, z):
        assert not v.numpy().any()
    same_bits(g.numpy(), np.ones(6, np.float32))


def _graph_of(torch, stream, calls):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    return graph


def test_graph_replays(pn, rng):
    """A captured step (joined forward, backward, with a key in device memory that the
    graph itself advances), replayed with the program's own calls in between;
    a second graph of the same calls, replayed on another stream at the same
    time, shares no workspace with it."""
    import torch
    lib, T = pn.core._lib, pn.Tensor
    rows, cols, p = 700, 1030, 0.2
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    sides = []
    try:
        for i in range(2):
            c = _case(rng, rows, cols, np.float32)
            t = {k: torch.from_numpy(v).cuda() for k, v in c.items()}
            for k, n in (("y", None), ("h", None), ("dx", None), ("dres", None), ("m", rows), ("r", rows),
                         ("dg", cols), ("db", cols)):
                t[k] = torch.zeros(n if n else (rows, cols), device="cuda")
            t["key"] = torch.tensor([i, 0], dtype=torch.int64, device="cuda")
            w = {k: T.from_torch(v) for k, v in t.items() if k != "key"}
            pn.set_stream(s[i].cuda_stream)
            torch.cuda.synchronize()

            def step(t=t, w=w):
                P = lambda k: w[k]._ptr  # noqa: E731
                key = t["key"].data_ptr()
                assert lib.neural_dropout_add_layer_norm_forward(P("y"), P("h"), P("x"), P("res"), P("g"), P("b"), p,
                                                                 key, EPS, P("m"), P("r")) == 0
                assert lib.neural_dropout_add_layer_norm_backward(P("dx"), P("dres"), P("dg"), P("db"), P("dy"),
                                                                  P("dh"), P("h"), P("g"), P("m"), P("r"), p, key) == 0
                t["key"][1] += 1

            sides.append((c, t, w, _graph_of(torch, s[i], step)))
        pn.set_stream(None)
        torch.cuda.synchronize()
        for replay in range(4):
            for i, (c, t, w, graph) in enumerate(sides):  # both at once
                with torch.cuda.stream(s[i]):
                    graph.replay()
            torch.cuda.synchronize()
            for i, (c, t, w, graph) in enumerate(sides):
                key = _key(pn, i, replay)
                y, h, m, r = _joined(pn, c, p, key)  # the program's own calls, which use the cached workspace
                grads = _joined_grad(pn, c, h, m, r, p, key)
                for k, v in zip(("y", "h", "m", "r", "dx", "dres", "dg", "db"), (y, h, m, r, *grads)):
                    same_bits(t[k].cpu().numpy(), v)
                    t[k].fill_(9.0)
            lib.neural_hip_empty_cache()
            torch.cuda.synchronize()
    finally:
        pn.set_stream(None)


def test_other_stream(pn, rng):
    """On a stream of the caller's, behind work that is still running there."""
    import torch
    c = _case(rng, 300, 1500, np.float32)
    want = _forward(pn, c["x"], c["g"], c["b"])
    s = torch.cuda.Stream()
    try:
        with torch.cuda.stream(s):
            x = torch.zeros(300, 1500, device="cuda")
            big = torch.randn(4096, 4096, device="cuda")
            y = torch.empty_like(x)
            g, b, src = (torch.from_numpy(c[k]).cuda() for k in ("g", "b", "x"))
            T = pn.Tensor.from_torch
            X, Y, Gm, Bt = T(x), T(y), T(g), T(b)
            pn.set_stream(s.cuda_stream)
            for _ in range(10):
                big = big @ big * 1e-3
            x.copy_(src)
            assert pn.core._lib.neural_layer_norm_forward(Y._ptr, X._ptr, Gm._ptr, Bt._ptr, EPS, None, None) == 0
            z = y + 0
        s.synchronize()
        same_bits(z.cpu().numpy(), want[0])
    finally:
        pn.set_stream(None)


def test_threads(pn, rng):
    """Backward calls from several host threads at once: each its own workspace."""
    import threading
    cases = [_case(rng, 400 + 100 * i, 700 + 300 * i, np.float32) for i in range(4)]
    want = []
    for c in cases:
        _, m, r = _forward(pn, c["x"], c["g"], c["b"])
        want.append((m, r, _backward(pn, c["dy"], c["x"], c["g"], m, r)))
    bad = []

    def work(i):
        m, r, w = want[i]
        for _ in range(5):
            got = _backward(pn, cases[i]["dy"], cases[i]["x"], cases[i]["g"], m, r)
            if not all(np.array_equal(a, b) for a, b in zip(got, w)):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_many_elements(pn):
    """More than 2^32 elements: the last rows, and the sums over all of them.
    Every row is the same, so dbeta is rows dy exactly, as are the rows' results."""
    import torch
    cols = 4096
    rows = (1 << 20) + 3
    need = 2 * 4 * rows * cols
    torch.cuda.empty_cache()
    pn.core._lib.neural_hip_empty_cache()
    if torch.cuda.mem_get_info()[0] < need + (4 << 30):
        pytest.skip("not enough free device memory")
    lib, T = pn.core._lib, pn.Tensor
    one = torch.arange(cols, device="cuda", dtype=torch.float32) % 7 - 3
    x = one.repeat(rows, 1)
    dy = torch.full((rows, cols), 0.5, device="cuda")
    m, r = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dg, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    X, DY, M, R, DG, DB = (T.from_torch(v) for v in (x, dy, m, r, dg, db))
    y0 = one.repeat(2, 1)
    Y0 = T.from_torch(y0)
    torch.cuda.synchronize()
    assert lib.neural_layer_norm_forward(Y0._ptr, Y0._ptr, None, None, EPS, None, None) == 0
    tail = x[-2:].clone()
    torch.cuda.synchronize()
    assert lib.neural_layer_norm_forward(X._ptr, X._ptr, None, None, EPS, M._ptr, R._ptr) == 0
    pn.synchronize()
    assert torch.equal(x[-2:], y0) and torch.equal(x[:2], y0) and not torch.equal(x[-2:], tail)
    assert bool((m == m[0]).all()) and bool((r == r[0]).all())
    M0, R1 = torch.zeros_like(m), torch.ones_like(r)
    Z, O = T.from_torch(M0), T.from_torch(R1)
    torch.cuda.synchronize()
    assert lib.neural_layer_norm_backward(DY._ptr, DG._ptr, DB._ptr, DY._ptr, X._ptr, None, Z._ptr, O._ptr) == 0
    pn.synchronize()
    # dy = 1/2 (rows is odd and under 2^24): exact in f32 up to the last rounding
    assert bool((db == rows * 0.5).all())
    want = y0[0].double() * (rows * 0.5)
    assert bool(((dg.double() - want).abs() <= 2.0 ** -22 * want.abs()).all())
    assert torch.equal(dy[-1], dy[0]) and torch.equal(dy[rows // 2], dy[0]) and not bool((dy[0] == 0.5).all())
    del X, DY, x, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", DT)
def test_modules_train_together(pn, rng, dt):
    """Two sublayers' ends as a program has them (normalise, dropout, join), forward
    and backward through the modules, against the same chain of long double
    forms.  Each f32 stage rounds once, and the stages' condition here is
    below 50: 4 stages of 2^-24, times 50, times the largest value."""
    code = pn.float32 if dt == np.float32 else pn.float64
    rows, cols = 60, 190
    x, r0 = _rows(rng, rows, cols, dt), rng.normal(0, 1, (rows, cols)).astype(dt)
    pre, drop, end = pn.LayerNorm(cols, dtype=code), pn.CounterDropout(0.1, 3), pn.DropoutAddLayerNorm(
        cols, 0.2, dtype=code, seed=4)
    gam = {m: (rng.normal(1, 0.2, cols).astype(dt), rng.normal(0, 0.2, cols).astype(dt)) for m in (pre, end)}
    for m, (g, b) in gam.items():
        m.gamma, m.beta = pn.Tensor.from_numpy(g), pn.Tensor.from_numpy(b)
    a = pre(pn.Tensor.from_numpy(x))
    d = drop(a)
    y, h = end(d, pn.Tensor.from_numpy(r0))
    dy, dh = rng.normal(0, 1, (rows, cols)).astype(dt), rng.normal(0, 1, (rows, cols)).astype(dt)
    gx, gr = end.backward(pn.Tensor.from_numpy(dy), pn.Tensor.from_numpy(dh))
    dx = pre.backward(drop.backward(gx))
    L = np.longdouble

    def ln(v, g, b):
        c = v - v.mean(-1, keepdims=True)
        s = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + L(EPS))
        return c * s * g + b, c * s, s

    def lnb(g_out, xh, s, g):
        w = g_out * g
        return s * (w - w.mean(-1, keepdims=True) - xh * (w * xh).mean(-1, keepdims=True))

    (g1, b1), (g2, b2) = (tuple(v.astype(L) for v in gam[m]) for m in (pre, end))
    la, xh1, s1 = ln(x.astype(L), g1, b1)
    m1 = ref.keep(rows * cols, 0.1, 3, 0).reshape(rows, cols) / L(0.9)
    m2 = ref.keep(rows * cols, 0.2, 4, 0).reshape(rows, cols) / L(0.8)
    lh = r0.astype(L) + la * m1 * m2
    ly, xh2, s2 = ln(lh, g2, b2)
    lr = lnb(dy.astype(L), xh2, s2, g2) + dh
    l1 = lr * m2 * m1
    ldx = lnb(l1, xh1, s1, g1)
    want = {"y": ly, "h": lh, "gr": lr, "dx": ldx, "dg2": (dy * xh2).sum(0), "db2": dy.astype(L).sum(0),
            "dg1": (l1 * xh1).sum(0), "db1": l1.sum(0)}
    got = {"y": y, "h": h, "gr": gr, "dx": dx, "dg2": end.gamma.grad, "db2": end.beta.grad, "dg1": pre.gamma.grad,
           "db1": pre.beta.grad}
    for k in want:
        lim = 200 * ref.U[np.dtype(dt)] * np.abs(want[k]).max() * (rows if k[0] == "d" and k != "dx" else 1)
        assert np.abs(got[k].numpy() - want[k]).max() <= lim, k
    for m in (pre, drop, end):
        m.eval()
    y2, h2 = end(drop(a), pn.Tensor.from_numpy(r0))
    same_bits(h2.numpy(), r0 + a.numpy())
    same_bits(y2.numpy(), _forward(pn, h2.numpy(), *gam[end])[0])
    # AdamW takes the parameters and the gradients the modules left
    opt = pn.AdamW(learning_rate=1e-2)
    ps = pre.parameters() + end.parameters()
    before = [p.numpy() for p in ps]
    opt.step(ps, [p.grad for p in ps])
    assert all(not np.array_equal(b, p.numpy()) for b, p in zip(before, ps))
    with pytest.raises(ValueError):
        pre(pn.Tensor.zeros([3, cols + 1], code))


@pytest.mark.parametrize("dt,cols", [(np.float32, c) for c in (8200, 10300, 12300, 14341, 16391, 20000)] +
                         [(np.float64, c) for c in (4200, 6150, 7200, 12003)])
def test_wide_forms_of_many_rows(pn, rng, dt, cols):
    """More rows than the one launch of few rows takes and than two for each block, at every
    number of vectors a lane past four, alone and joined."""
    _check_all(pn, rng, 530, cols, dt)


@pytest.mark.parametrize("rows,cols", [(20001, 5000), (20000, 8200), (20000, 10300), (20001, 13001), (20000, 16384),
                                       (9000, 20000)])
def test_column_sums_of_one_sign(pn, rows, cols):
    """f32 terms of one sign, 35 to 80 rows to a block's sums: dgamma and dbeta carry the
    rounding of the partials and of the result, u each, whatever the rows (sums in double:
    (rows + 8) 2^-53 beside them).  mean 0 and rstd 1, so xh is x itself."""
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows + cols)
    x = torch.rand(rows, cols, device="cuda", generator=gen) + 0.5
    dy = torch.full((rows, cols), 0.1, device="cuda")
    m, r = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dg, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    T = pn.Tensor.from_torch
    t = [T(v) for v in (dg, db, dy, x, m, r)]
    torch.cuda.synchronize()
    assert pn.core._lib.neural_layer_norm_backward(None, t[0]._ptr, t[1]._ptr, t[2]._ptr, t[3]._ptr, None, t[4]._ptr,
                                                   t[5]._ptr) == 0
    pn.synchronize()
    d = dy[0].double()
    lim = 1.01 * (2 * ref.U[np.dtype(np.float32)] + (rows + 8) * ref.D)
    for got, want in ((dg, d * x.double().sum(0)), (db, d * rows)):
        assert float(((got.double() - want).abs() / want).max()) <= lim


@pytest.mark.parametrize("cols", [6, 3000, 40000, 70001])
def test_refusals_of_one_row_or_column(pn, cols):
    """Where a row's tensors have as many values as gamma's gradient (one row), or as the
    statistics (one column), only the outputs of the rows' shape may replace an input."""
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    k, jk = lib.neural_layer_norm_backward, lib.neural_dropout_add_layer_norm_backward
    x, dy, dh, dx, g = (T.ones([1, cols]) for _ in range(5))
    m, r = T.zeros([1]), T.ones([1])
    X, DY, DH, DX, G, M, R = (t._ptr for t in (x, dy, dh, dx, g, m, r))
    for over in (X, DY):
        for also in (DX, over, None):
            assert k(also, over, None, DY, X, G, M, R) == E.INVALID_ARGUMENT
            assert k(also, None, over, DY, X, G, M, R) == E.INVALID_ARGUMENT
    for over in (X, DY, DH):
        assert jk(DX, None, over, None, DY, DH, X, G, M, R, 0.0, None) == E.INVALID_ARGUMENT
        assert jk(None, DX, None, over, DY, DH, X, G, M, R, 0.0, None) == E.INVALID_ARGUMENT
    c, res, o, h = (T.ones([cols, 1]) for _ in range(4))
    s = T.zeros([cols])
    C, RES, O, H, S = (t._ptr for t in (c, res, o, h, s))
    f, jf = lib.neural_layer_norm_forward, lib.neural_dropout_add_layer_norm_forward
    assert f(O, C, None, None, EPS, C, S) == E.INVALID_ARGUMENT
    assert f(O, C, None, None, EPS, S, C) == E.INVALID_ARGUMENT
    for over in (C, RES):
        assert jf(O, H, C, RES, None, None, 0.0, None, EPS, over, S) == E.INVALID_ARGUMENT
        assert jf(O, H, C, RES, None, None, 0.0, None, EPS, S, over) == E.INVALID_ARGUMENT
    for t in (x, dy, dh, dx, g, c, res, o, h):
        assert (t.numpy() == 1).all()
    # in place is still taken
    assert k(DY, DX, DH, DY, X, G, M, R) == 0 and f(C, C, None, None, EPS, S, None) == 0
    assert not c.numpy().any()


def test_tensors_over_a_device_address(pn, rng):
    """A tensor made over an owned tensor's device address is the same memory: refused
    where outputs may not meet it, and in place where they may replace it."""
    E, lib = pn.NeuralError, pn.core._lib
    rows, cols = 6, 50

    def over(t, shape, skip=0):
        return keep(pn.Tensor._wrap(lib.neural_tensor_from_buffer(
            t.device_ptr + 4 * skip, (ctypes.c_uint64 * len(shape))(*shape), len(shape), 0, None)))

    c = _case(rng, rows, cols, np.float32)
    want = _forward(pn, c["x"], c["g"], c["b"])
    grads = _backward(pn, c["dy"], c["x"], c["g"], want[1], want[2])
    x, dy, g, b, m, r = (pn.Tensor.from_numpy(v) for v in (c["x"], c["dy"], c["g"], c["b"], want[1], want[2]))
    y, dg = pn.Tensor.zeros([rows, cols]), pn.Tensor.zeros([cols])
    wide = pn.Tensor.ones([rows + 1, cols])
    low, high = over(wide, [rows, cols]), over(wide, [rows, cols], 1)
    k, f, d = lib.neural_layer_norm_backward, lib.neural_layer_norm_forward, lib.neural_counter_dropout_forward
    key = _key(pn, 1, 1)
    assert k(y._ptr, over(g, [cols]), None, dy._ptr, x._ptr, g._ptr, m._ptr, r._ptr) == E.INVALID_ARGUMENT
    assert k(y._ptr, None, over(x, [cols], 7), dy._ptr, x._ptr, g._ptr, m._ptr, r._ptr) == E.INVALID_ARGUMENT
    assert k(y._ptr, dg._ptr, over(dg, [cols]), dy._ptr, x._ptr, g._ptr, m._ptr, r._ptr) == E.INVALID_ARGUMENT
    assert f(high, low, None, None, EPS, None, None) == E.INVALID_ARGUMENT
    assert f(over(wide, [rows, cols], 1), over(wide, [rows, cols]), None, None, EPS, None,
             None) == E.INVALID_ARGUMENT
    assert d(high, low, 0.5, key) == E.INVALID_ARGUMENT
    assert d(over(wide, [rows, cols + 1], 1), over(wide, [rows, cols + 1]), 0.5, key) == E.INVALID_ARGUMENT
    assert (wide.numpy() == 1).all() and not y.numpy().any()
    same_bits(g.numpy(), c["g"])
    px, pd = over(x, [rows, cols]), over(dy, [rows, cols])
    assert k(pd, dg._ptr, None, dy._ptr, x._ptr, g._ptr, m._ptr, r._ptr) == 0
    same_bits(dy.numpy(), grads[0])
    same_bits(dg.numpy(), grads[1])
    assert f(px, x._ptr, g._ptr, b._ptr, EPS, None, None) == 0
    same_bits(x.numpy(), want[0])
    assert d(x._ptr, px, 0.25, key) == 0
    same_bits(x.numpy(), ref.dropout(want[0], 0.25, 1, 1))


def _room(pn, need):
    import torch
    torch.cuda.empty_cache()
    pn.core._lib.neural_hip_empty_cache()
    if torch.cuda.mem_get_info()[0] < need + (4 << 30):
        pytest.skip("not enough free device memory")


@pytest.mark.parametrize("cols,rows_too", [((1 << 26) + 5, True), ((1 << 31) + 13, False)])
def test_gradients_past_a_grid_of_columns(pn, cols, rows_too):
    """One row so wide that the column sums' blocks (of 1024 lanes, 32 columns; of 512,
    256 columns) have more lanes than one launch may: exact, of small whole numbers."""
    import torch
    _room(pn, 4 * cols * 10)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    x, dy = (torch.empty(1, cols, device="cuda").random_(0, 7, generator=gen).sub_(3) for _ in range(2))
    dx = torch.full((1, cols), 9.0, device="cuda") if rows_too else None
    dg, db = torch.full((cols,), 9.0, device="cuda"), torch.full((cols,), 9.0, device="cuda")
    m, r = torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")
    T = pn.Tensor.from_torch
    DX, DG, DB, DY, X, M, R = (T(v) if v is not None else None for v in (dx, dg, db, dy, x, m, r))
    torch.cuda.synchronize()
    assert pn.core._lib.neural_layer_norm_backward(_p(DX), DG._ptr, DB._ptr, DY._ptr, X._ptr, None, M._ptr,
                                                   R._ptr) == 0
    pn.synchronize()
    assert torch.equal(db, dy[0]) and torch.equal(dg, (dy * x)[0])
    if rows_too:
        w, xd = dy.double(), x.double()
        want = w - w.mean() - xd * (w * xd).mean()
        # whole sums below 2^53; under 16 roundings of values below 100, and the result's
        assert bool(((dx.double() - want).abs() <= 100 * 16 * ref.D + 2.0 ** -24 * want.abs()).all())
    torch.cuda.empty_cache()


def test_rows_past_a_grid_of_wide_blocks(pn):
    """2^22 rows and more of a block of 1024 lanes each (137 GB, in place): the first rows,
    those around the second launch's first, and the last."""
    import torch
    rows, cols = (1 << 22) + 5, 8196
    _room(pn, 4 * rows * cols)
    one = torch.arange(cols, device="cuda", dtype=torch.float32) % 11 - 5
    x = one.repeat(rows, 1)
    y0 = one.repeat(1, 1)
    T = pn.Tensor.from_torch
    X, Y0 = T(x), T(y0)
    torch.cuda.synchronize()
    f = pn.core._lib.neural_layer_norm_forward
    assert f(Y0._ptr, Y0._ptr, None, None, EPS, None, None) == 0
    assert f(X._ptr, X._ptr, None, None, EPS, None, None) == 0
    pn.synchronize()
    assert not torch.equal(y0[0], one)
    pick = torch.cat([torch.arange(3, device="cuda"), torch.arange((1 << 22) - 4, rows, device="cuda"),
                      torch.arange(0, rows, 65521, device="cuda")])
    assert bool((x[pick] == y0).all())
    del X, x
    torch.cuda.empty_cache()


def test_default_modules_drop_apart(pn):
    """Two sublayers' ends built alike drop different elements in the same step."""
    x, z = pn.Tensor.ones([40, 50]), pn.Tensor.zeros([40, 50])
    a, b = (pn.DropoutAddLayerNorm(50, 0.5) for _ in range(2))
    ha, hb = (m(x, z)[1].numpy() for m in (a, b))
    # 2000 independent pairs of halves: equal in 1000 +- 22 of them
    assert 800 < int((ha == hb).sum()) < 1200
    same_bits(ha, ref.dropout(np.ones((40, 50), np.float32), 0.5, a.dropout.seed, 0))


def test_a_failed_forward_changes_no_mask(pn, rng):
    """Neither the mask that backward makes again nor the next forward's; and another use
    of the joined module's dropout is a call of its own."""
    T, cols = pn.Tensor.from_numpy, 33
    c = _case(rng, 7, cols, np.float32)
    one = np.ones(cols, np.float32)
    x, res, dy, dh = (T(c[k]) for k in ("x", "res", "dy", "dh"))
    end = pn.DropoutAddLayerNorm(cols, 0.4, seed=3)
    h = end(x, res)[1].numpy()
    _, mean, rstd = _forward(pn, h, one, 0 * one)
    want = _joined_grad(pn, {**c, "g": one}, h, mean, rstd, 0.4, _key(pn, 3, 0))
    with pytest.raises(pn.NeuralException):
        end(x, T(c["res"][:3]))
    end.dropout(x)
    for a, w in zip(end.backward(dy, dh), want):
        same_bits(a.numpy(), w)
    same_bits(end(x, res)[1].numpy(), c["res"] + ref.dropout(c["x"], 0.4, 3, 2))  # after calls 0 and 1
    drop = pn.CounterDropout(0.5, seed=1)
    drop(x)
    drop.p = 2.0
    with pytest.raises(pn.NeuralException):
        drop(x)
    same_bits(drop.backward(dy).numpy(), ref.dropout(c["dy"], 0.5, 1, 0))


def test_a_failed_backward_leaves_the_gradients(pn, rng):
    T, cols = pn.Tensor.from_numpy, 33
    c = _case(rng, 7, cols, np.float32)
    x, res, dy = (T(c[k]) for k in ("x", "res", "dy"))
    end, norm = pn.DropoutAddLayerNorm(cols, 0.4, seed=3), pn.LayerNorm(cols)
    end(x, res)
    end.backward(dy)
    dg, db = end.gamma.grad.numpy(), end.beta.grad.numpy()
    for bad in (lambda: end.backward(T(c["dy"][:3])), lambda: end.backward(dy, T(c["dh"][:3]))):
        with pytest.raises(pn.NeuralException):
            bad()
        same_bits(end.gamma.grad.numpy(), dg)
        same_bits(end.beta.grad.numpy(), db)
    norm(x)
    with pytest.raises(pn.NeuralException):
        norm.backward(T(c["dy"][:3]))
    assert norm.gamma.grad is None and norm.beta.grad is None


def test_a_dropout_gradient_has_the_forward_elements(pn, rng):
    x = rng.normal(0, 1, (5, 8)).astype(np.float32)
    drop = pn.CounterDropout(0.5, seed=1)
    drop(pn.Tensor.from_numpy(x))
    for n in (3, 6):
        with pytest.raises(ValueError):
            drop.backward(pn.Tensor.from_numpy(np.ones((n, 8), np.float32)))
    same_bits(drop.backward(pn.Tensor.from_numpy(x.reshape(40))).numpy(), ref.dropout(x, 0.5, 1, 0).reshape(40))


def _hip():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as f:
        return ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))


def _alloc_counts(pn):
    a, m = ctypes.c_ulonglong(), ctypes.c_ulonglong()
    assert pn.core._lib.neural_hip_alloc_stats(ctypes.byref(a), ctypes.byref(m)) == 0
    return a.value, m.value


def test_a_stream_that_cannot_be_asked(pn, rng):
    """The null stream while a blocking stream is being captured cannot say whether it is
    captured itself: the call answers so, without memory or launches, and the
    capture goes on."""
    hip, lib, T = _hip(), pn.core._lib, pn.Tensor
    c = _case(rng, 600, 100, np.float32)  # more than the rows of a call that needs no memory
    _, mean, rstd = _forward(pn, c["x"], c["g"], c["b"])
    want = _backward(pn, c["dy"], c["x"], c["g"], mean, rstd)
    t = [T.from_numpy(v) for v in (c["dy"], c["x"], c["g"], mean, rstd)]
    dg, db = T.zeros([100]), T.zeros([100])
    args = [None, dg._ptr, db._ptr] + [v._ptr for v in t]
    pn.set_stream(None)
    own = ctypes.c_void_p(lib.neural_hip_get_stream())
    graph, asked = ctypes.c_void_p(), ctypes.c_int()
    pn.synchronize()
    try:
        pn.set_stream(0)
        assert hip.hipStreamBeginCapture(own, 2) == 0
        cannot = hip.hipStreamIsCapturing(None, ctypes.byref(asked)) != 0
        hip.hipGetLastError()
        if cannot:
            before = _alloc_counts(pn)
            assert lib.neural_layer_norm_backward(*args) == pn.NeuralError.INTERNAL
            assert _alloc_counts(pn) == before
        assert hip.hipStreamEndCapture(own, ctypes.byref(graph)) == 0
        assert hip.hipGraphDestroy(graph) == 0
    finally:
        pn.set_stream(None)
    assert cannot, "the null stream could be asked"
    assert not dg.numpy().any()
    assert lib.neural_layer_norm_backward(*args) == 0
    same_bits(dg.numpy(), want[1])
    same_bits(db.numpy(), want[2])


def _captured_grads(pn, torch, stream, cases):
    """A graph of the gradients of several norms in a row: the graph, its calls' (outputs,
    wanted, tensors), and how many hipMallocs the library made while it was captured."""
    lib, T = pn.core._lib, pn.Tensor
    calls = []
    for c in cases:
        _, mean, rstd = _forward(pn, c["x"], c["g"], c["b"])
        want = _backward(pn, c["dy"], c["x"], c["g"], mean, rstd)
        ins = [torch.from_numpy(v).cuda() for v in (c["dy"], c["x"], c["g"], mean, rstd)]
        outs = [torch.zeros_like(v) for v in (ins[1], ins[2], ins[2])]
        calls.append((outs, want, [T.from_torch(v) for v in outs + ins]))
    pn.set_stream(stream.cuda_stream)
    torch.cuda.synchronize()
    before = _alloc_counts(pn)[1]

    def step():
        for _, _, t in calls:
            assert lib.neural_layer_norm_backward(*[v._ptr for v in t]) == 0

    graph = _graph_of(torch, stream, step)
    made = _alloc_counts(pn)[1] - before
    pn.set_stream(None)
    return graph, calls, made


def _replayed(torch, replay, calls):
    for _ in range(2):
        for outs, _, _ in calls:
            [o.fill_(9.0) for o in outs]
        torch.cuda.synchronize()
        replay()
        torch.cuda.synchronize()
        for outs, want, _ in calls:
            for o, w in zip(outs, want):
                same_bits(o.cpu().numpy(), w)


def test_memory_of_captured_calls(pn, rng):
    """A capture's gradients share a block, a wider one behind them has its own; the memory
    stays while the graph lives and is given back when it is gone."""
    import gc
    import time
    import torch
    s = torch.cuda.Stream()
    case = lambda rows, cols: _case(rng, rows, cols, np.float32)  # noqa: E731
    try:
        _captured_grads(pn, torch, s, [case(600, 50)])  # whatever torch and HIP allocate once
        graph, calls, made = _captured_grads(pn, torch, s, [case(3000, 4096) for _ in range(3)])  # 16.8 MB of partials
        assert made == 1
        other, more, made = _captured_grads(pn, torch, s, [case(3000, 500), case(3000, 2048), case(2000, 300)])
        assert made == 2
        _replayed(torch, graph.replay, calls)
        _replayed(torch, other.replay, more)
        pn.release_graph_memory()  # both live: nothing of theirs
        x = torch.full((64 << 20,), 3.0, device="cuda")  # would take what had been freed

        def both():
            with torch.cuda.stream(s):
                graph.replay()
            other.replay()

        _replayed(torch, both, calls + more)
        assert bool((x == 3).all())
        had = torch.cuda.mem_get_info()[0]
        del graph, both
        gc.collect()
        for _ in range(100):  # HIP lets go of a destroyed graph in its own time
            torch.cuda.synchronize()
            pn.release_graph_memory()
            got = torch.cuda.mem_get_info()[0] - had
            if got >= 16 << 20:
                break
            time.sleep(0.02)
        assert 16 << 20 <= got < 48 << 20, got  # one block for the three calls
        _replayed(torch, other.replay, more)
    finally:
        pn.set_stream(None)
        pn.release_graph_memory()


def test_graph_memory_is_not_released_in_a_capture(pn, rng):
    import torch
    s = torch.cuda.Stream()
    y = torch.zeros(8, device="cuda")
    try:
        pn.set_stream(s.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert pn.core._lib.neural_hip_release_graph_memory() == pn.NeuralError.INTERNAL
            y.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert bool((y == 1).all())
    finally:
        pn.set_stream(None)
    assert pn.core._lib.neural_hip_release_graph_memory() == 0
