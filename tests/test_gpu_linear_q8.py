"""The product of 8-bit rows with 8-bit weights, with bias, activation and residual in its
epilogue: the sum exactly (whole numbers), its scaling in double and one rounding exactly
as numpy makes them, the activation bit for bit as the elementwise call, the residual
exactly.  Few and many rows, odd sizes, strides and addresses, extreme codes, graphs,
streams, threads and the refusals."""

import numpy as np
import pytest

from conftest import GPU, same_bits

pytestmark = GPU

DT = [np.float32, np.float64]


def _case(rng, m, k, n, dt, lo=-127):
    return {"a": rng.integers(lo, 128, (m, k), dtype=np.int8), "w": rng.integers(lo, 128, (n, k), dtype=np.int8),
            "sa": rng.uniform(1e-3, 2e-2, m).astype(dt), "sw": rng.uniform(1e-4, 1e-3, n).astype(dt),
            "bias": rng.normal(0, 0.3, n).astype(dt), "res": rng.normal(0, 2, (m, n)).astype(dt)}


def _product(a, w):
    """Exact: float64 sums of whole numbers below 2^31."""
    return a.astype(np.float64) @ w.astype(np.float64).T


def _scaled(c, bias=True):
    """scale * sum + bias in double, rounded to the dtype."""
    with np.errstate(all="ignore"):
        z = _product(c["a"], c["w"]) * (c["sa"].astype(np.float64)[:, None] * c["sw"].astype(np.float64)[None, :])
        z = z + (c["bias"].astype(np.float64) if bias else 0.0)
        return z.astype(c["sa"].dtype)


def _act(pn, z, act, alpha):
    """The elementwise call on z."""
    T = pn.Tensor
    t, zero = T.from_numpy(z), T.zeros([z.shape[1]], pn.float32 if z.dtype == np.float32 else pn.float64)
    out = T.create(z.shape, t.dtype)
    assert pn.core._lib.neural_bias_add_act(out._ptr, t._ptr, zero._ptr, act, alpha) == 0
    return out.numpy()


def _place(v, stride, shift):
    """Rows of codes at a stride, starting `shift` bytes into an allocation, junk around them."""
    import torch
    rows, k = v.shape
    raw = torch.full((shift + rows * stride + 64,), 91, dtype=torch.int8, device="cuda")
    raw[shift:shift + rows * stride].view(rows, stride)[:, :k].copy_(torch.from_numpy(v))
    return raw, raw.data_ptr() + shift


def _run(pn, c, act=0, alpha=0.0, bias=True, res=True, lda=None, ldw=None, shift=0, out=None):
    import torch
    T = pn.Tensor
    (m, k), n = c["a"].shape, c["w"].shape[0]
    lda, ldw = lda or k, ldw or k
    ha, pa = _place(c["a"], lda, shift)
    hw, pw = _place(c["w"], ldw, shift)
    sa, sw = T.from_numpy(c["sa"]), T.from_numpy(c["sw"])
    b = T.from_numpy(c["bias"]) if bias else None
    r = T.from_numpy(c["res"]) if res else None
    o = out or T.create([m, n], sa.dtype)
    torch.cuda.synchronize()
    rc = pn.core._lib.neural_linear_q8(o._ptr, pa, lda, sa._ptr, pw, ldw, sw._ptr, k, b._ptr if b else None, act, alpha,
                                       r._ptr if r else None)
    assert rc == 0
    got = o.numpy()
    del ha, hw
    return got


def _check(pn, c, act=0, alpha=0.0, bias=True, res=True, **kw):
    z = _scaled(c, bias)
    want = z if act == 0 else _act(pn, z, act, alpha)
    if res:
        want = want + c["res"]
    got = _run(pn, c, act, alpha, bias, res, **kw)
    if act == 0 or act == 1:  # (z + 0 of the elementwise call turns -0 into +0, as a residual would)
        assert np.array_equal(got, want, equal_nan=True)
    else:
        same_bits(got + c["sa"].dtype.type(0), want + c["sa"].dtype.type(0))


ROWS = [1, 2, 3, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m", ROWS)
def test_row_counts(pn, rng, dt, m):
    for k, n in ((64, 64), (200, 70), (1001, 333), (4096, 128)):
        _check(pn, _case(rng, m, k, n, dt))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("k", [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 255, 256, 257, 383, 384,
                               500, 511, 512, 513, 1023, 1024, 1025, 2049, 5000])
def test_depths(pn, rng, dt, k):
    for m, n in ((1, 33), (20, 130), (130, 70), (300, 260)):
        c = _case(rng, m, k, n, dt)
        _check(pn, c)
        ld = -(-k // 16) * 16  # read in place: rows padded to 16 bytes
        _check(pn, c, res=False, lda=ld, ldw=ld + 32)


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 2049])
def test_widths(pn, rng, n):
    for m, k in ((1, 512), (7, 130), (40, 64), (150, 257), (513, 192)):
        _check(pn, _case(rng, m, k, n, np.float32))


@pytest.mark.parametrize("m,k,n", [(1, 4096, 4096), (4, 16384, 1024), (16, 4096, 5000), (64, 4096, 4096), (64, 8192, 1000),
                                   (100, 16384, 512), (1024, 1024, 1024), (777, 2080, 1555), (2048, 512, 4096),
                                   (4096, 4096, 300), (300, 4096, 4096), (577, 1001, 3001), (1537, 4000, 2305)])
def test_larger(pn, rng, m, k, n):
    """Against torch's float64 product on the device: exact whole numbers."""
    import torch
    c = _case(rng, m, k, n, np.float32)
    a, w = (torch.from_numpy(c[q]).cuda().double() for q in ("a", "w"))
    acc = (a @ w.t().contiguous()).cpu().numpy()
    z = (acc * (c["sa"].astype(np.float64)[:, None] * c["sw"].astype(np.float64)) + c["bias"].astype(np.float64))
    want = z.astype(np.float32) + c["res"]
    assert np.array_equal(_run(pn, c), want)
    ld = -(-k // 64) * 64
    assert np.array_equal(_run(pn, c, lda=ld, ldw=ld), want)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,k,n", [(16, 100, 8192), (16, 100, 8193), (17, 6143, 70), (17, 6145, 70), (33, 8192, 65), (64, 8209, 130),
                                   (100, 20000, 300), (20, 131071, 33), (512, 300, 4096), (513, 300, 4097), (1024, 272, 4096),
                                   (1100, 272, 4100), (2048, 272, 4096), (2049, 129, 4097), (4096, 130, 4096), (4000, 64, 4200)])
def test_forms(pn, rng, dt, m, k, n):
    """Sizes around the changes of form: few rows, depth in parts, every tile; epilogue and copies of
    each."""
    c = _case(rng, m, k, n, dt)
    _check(pn, c)
    ld = -(-k // 16) * 16
    _check(pn, c, res=False, lda=ld, ldw=ld)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("ld", [1001, 1002, 1004])
@pytest.mark.parametrize("m,n", [(16, 8200), (17, 1000), (33, 700), (64, 100), (97, 1000), (129, 33), (500, 17), (32, 4096),
                                 (48, 4100)])
def test_unaligned_groups(pn, rng, dt, ld, m, n):
    """Rows at strides of 1, 2 and 4 bytes' alignment in groups of 16, from an odd address too."""
    c = _case(rng, m, 1001, n, dt)
    _check(pn, c, act=8, lda=ld, ldw=ld)
    _check(pn, c, res=False, lda=ld, ldw=ld, shift=3)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("act", range(13))
def test_activations(pn, rng, dt, act):
    """Every activation, with every part of the epilogue there or not, over the values that the
    elementwise functions branch on."""
    alpha = 0.2 if act in (5, 6) else 0.0
    for m, k, n in ((3, 100, 65), (70, 256, 130), (260, 128, 300)):
        c = _case(rng, m, k, n, dt)
        c["sa"] *= dt(20)  # wide: past the activations' saturation
        for bias, res in ((True, True), (True, False), (False, True), (False, False)):
            _check(pn, c, act, alpha, bias, res)


@pytest.mark.parametrize("shift,lda,ldw", [(0, 0, 0), (1, 0, 0), (4, 0, 0), (8, 0, 0), (16, 0, 0), (0, 3, 0), (0, 0, 7),
                                           (3, 16, 8), (16, 16, 48)])
@pytest.mark.parametrize("m,k,n", [(1, 256, 40), (20, 250, 100), (300, 512, 270)])
def test_strides_and_addresses(pn, rng, m, k, n, shift, lda, ldw):
    c = _case(rng, m, k, n, np.float32)
    _check(pn, c, lda=k + lda, ldw=k + ldw, shift=shift)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_extreme_codes(pn, rng, m):
    """All codes of the largest size, -128 among them, up to the largest depth: sums of up to
    131071 * 2^14, just below 2^31, in every order of signs."""
    k = 131071
    n = 20
    c = _case(rng, m, k, n, np.float64, lo=-128)
    c["a"][:] = -128
    c["w"][:] = -128
    c["w"][1] = 127
    c["w"][2, ::2] = 127
    c["sa"][:] = 1.0
    c["sw"][:] = 1.0
    c["bias"][:] = 0.0
    got = _run(pn, c, res=False)
    assert got[0, 0] == k * 16384 and np.array_equal(got, _product(c["a"], c["w"]))


@pytest.mark.parametrize("dt", DT)
def test_scales(pn, rng, dt):
    """NaN, infinite, zero and huge scales go where the product takes them, row by row."""
    for m in (5, 150):
        c = _case(rng, m, 96, 70, dt)
        c["a"][1] = 0
        c["sa"][1] = np.nan   # a row that held NaN: codes 0, scale NaN
        c["sa"][2] = 0.0
        c["sw"][3] = np.inf
        c["sa"][4] = dt(1e30)
        _check(pn, c)
        assert np.isnan(_run(pn, c, res=False)[1]).all()


@pytest.mark.parametrize("m", [1, 30, 300])
def test_in_place_and_guards(pn, rng, m):
    """out over the residual; nothing around out is written."""
    import torch
    c = _case(rng, m, 200, 130, np.float32)
    want = _scaled(c) + c["res"]
    T = pn.Tensor
    big = torch.full((m * 130 + 64,), 5.0, device="cuda")
    view = big[19:19 + m * 130].view(m, 130)
    view.copy_(torch.from_numpy(c["res"]))
    (ha, pa), (hw, pw) = _place(c["a"], 200, 0), _place(c["w"], 200, 0)
    o, sa, sw, b = T.from_torch(view), T.from_numpy(c["sa"]), T.from_numpy(c["sw"]), T.from_numpy(c["bias"])
    torch.cuda.synchronize()
    assert pn.core._lib.neural_linear_q8(o._ptr, pa, 200, sa._ptr, pw, 200, sw._ptr, 200, b._ptr, 0, 0.0, o._ptr) == 0
    pn.synchronize()
    assert np.array_equal(view.cpu().numpy(), want)
    assert bool((big[:19] == 5).all()) and bool((big[19 + m * 130:] == 5).all())


def test_host_buffers(pn, rng):
    c = _case(rng, 9, 77, 31, np.float32)
    Z = pn.Tensor.from_numpy_zero_copy
    out = np.zeros((9, 31), np.float32)
    t = {k: Z(c[k]) for k in ("sa", "sw", "bias", "res")}
    o = Z(out)
    assert pn.core._lib.neural_linear_q8(o._ptr, c["a"].ctypes.data, 77, t["sa"]._ptr, c["w"].ctypes.data, 77,
                                         t["sw"]._ptr, 77, t["bias"]._ptr, 0, 0.0, t["res"]._ptr) == 0
    assert np.array_equal(out, _scaled(c) + c["res"])


def test_leading_dimensions_and_empty(pn, rng):
    lib, T = pn.core._lib, pn.Tensor
    c = _case(rng, 6, 40, 10, np.float32)
    (ha, pa), (hw, pw) = _place(c["a"], 40, 0), _place(c["w"], 40, 0)
    o, sa, sw = T.create([2, 3, 10]), T.from_numpy(c["sa"]), T.from_numpy(c["sw"])
    import torch
    torch.cuda.synchronize()
    assert lib.neural_linear_q8(o._ptr, pa, 40, sa._ptr, pw, 40, sw._ptr, 40, None, 0, 0.0, None) == 0
    assert np.array_equal(o.numpy().reshape(6, 10), _scaled(c, bias=False))
    e, s0 = T.create([0, 10]), T.create([0])
    assert lib.neural_linear_q8(e._ptr, pa, 40, s0._ptr, pw, 40, sw._ptr, 40, None, 0, 0.0, None) == 0
    e = T.create([6, 0])
    assert lib.neural_linear_q8(e._ptr, pa, 40, s0._ptr, pw, 40, s0._ptr, 40, None, 0, 0.0, None) == 0


def test_refusals(pn):
    import torch
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    f = lib.neural_linear_q8
    raw = torch.zeros(4096, dtype=torch.int8, device="cuda")
    A, W = raw.data_ptr(), raw.data_ptr() + 2048
    o, r, sa, sw, b = T.zeros([4, 6]), T.zeros([4, 6]), T.ones([4]), T.ones([6]), T.ones([6])
    O, R, SA, SW, B = (t._ptr for t in (o, r, sa, sw, b))
    ok = [O, A, 32, SA, W, 32, SW, 32, B, 0, 0.0, R]

    def with_(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)

    assert with_() == 0
    for i in (0, 1, 3, 4, 6):
        assert with_(**{f"_{i}": None}) == E.NULL_POINTER
    d4, d6, d46 = T.ones([4], pn.float64), T.ones([6], pn.float64), T.ones([4, 6], pn.float64)
    for i, v in ((3, d4), (6, d6), (8, d6), (11, d46), (0, d46)):
        assert with_(**{f"_{i}": v._ptr}) == E.DTYPE_MISMATCH
    s5, s64 = T.ones([5]), T.ones([6, 4])
    for i, v in ((3, s5), (6, s5), (8, s5), (11, s64)):
        assert with_(**{f"_{i}": v._ptr}) == E.SHAPE_MISMATCH
    s0 = T.create([])
    assert with_(_0=s0._ptr) == E.DIM_MISMATCH
    assert with_(_2=31) == E.INVALID_ARGUMENT and with_(_5=31) == E.INVALID_ARGUMENT
    assert with_(_7=0) == E.INVALID_ARGUMENT and with_(_7=-1) == E.INVALID_ARGUMENT
    assert with_(_9=-1) == E.INVALID_ARGUMENT and with_(_9=13) == E.INVALID_ARGUMENT
    assert with_(_2=1 << 20, _5=1 << 20, _7=131072) == E.TENSOR_TOO_LARGE
    assert with_(_2=1 << 60) == E.TENSOR_TOO_LARGE and with_(_5=1 << 60) == E.TENSOR_TOO_LARGE
    t = torch.zeros(8, 6, device="cuda")
    strided, lower, upper = (T.from_torch(v) for v in (t[::2], t[:4], t[2:6]))
    assert with_(_0=strided._ptr) == E.INVALID_ARGUMENT and with_(_11=strided._ptr) == E.INVALID_ARGUMENT
    assert with_(_0=upper._ptr, _11=lower._ptr) == E.INVALID_ARGUMENT
    assert with_(_0=lower._ptr, _8=T.from_torch(t[1])._ptr) == E.INVALID_ARGUMENT   # out over the bias
    assert with_(_0=lower._ptr, _1=t.data_ptr()) == E.INVALID_ARGUMENT              # out over the codes
    assert with_(_0=lower._ptr, _4=t.data_ptr() + 64) == E.INVALID_ARGUMENT         # out over the weights
    assert not t.cpu().numpy().any()


@pytest.mark.parametrize("m,k,n", [(1, 700, 500), (40, 1001, 300), (40, 8209, 300), (500, 1001, 300)])
def test_graphs_and_streams(pn, rng, m, k, n):
    """Two captured products on two streams (unaligned rows, which are copied first: each graph
    its own memory), replayed at once, with eager calls in between."""
    import torch
    lib, T = pn.core._lib, pn.Tensor
    streams, sides = [torch.cuda.Stream(), torch.cuda.Stream()], []
    try:
        for i in range(2):
            c = _case(rng, m, k, n, np.float32)
            t = {q: torch.from_numpy(c[q]).cuda() for q in c}
            t["out"] = torch.zeros(m, n, device="cuda")
            w = {q: T.from_torch(v) for q, v in t.items() if v.is_floating_point()}
            pn.set_stream(streams[i].cuda_stream)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[i]):
                assert lib.neural_linear_q8(w["out"]._ptr, t["a"].data_ptr(), k, w["sa"]._ptr, t["w"].data_ptr(), k,
                                            w["sw"]._ptr, k, w["bias"]._ptr, 0, 0.0, w["res"]._ptr) == 0
            sides.append((_scaled(c) + c["res"], t, w, graph, c))
        pn.set_stream(None)
        torch.cuda.synchronize()
        for _ in range(3):
            for i, side in enumerate(sides):
                with torch.cuda.stream(streams[i]):
                    side[3].replay()
            torch.cuda.synchronize()
            for want, t, _, _, c in sides:
                assert np.array_equal(t["out"].cpu().numpy(), want)
                t["out"].fill_(9.0)
                assert np.array_equal(_run(pn, c), want)
            lib.neural_hip_empty_cache()
            torch.cuda.synchronize()
    finally:
        pn.set_stream(None)


def test_threads(pn, rng):
    import threading
    cases = [_case(rng, 50 + 100 * i, 301 + 64 * i, 200, np.float32) for i in range(4)]
    want = [_scaled(c) + c["res"] for c in cases]
    bad = []

    def work(i):
        for _ in range(5):
            if not np.array_equal(_run(pn, cases[i]), want[i]):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_offsets_past_32_bits(pn):
    """Weights of more than 2^32 bytes at a wide stride: the last channels."""
    import torch
    n, k, ld = 70001, 96, 65536
    if torch.cuda.mem_get_info()[0] < n * ld + (8 << 30):
        pytest.skip("not enough free device memory")
    w = torch.zeros(n, ld, dtype=torch.int8, device="cuda")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    w[:, :k] = torch.randint(-127, 128, (n, k), device="cuda", generator=gen).to(torch.int8)
    for m in (3, 200):
        a = torch.randint(-127, 128, (m, k), device="cuda", generator=gen).to(torch.int8)
        out, sa, sw = torch.empty(m, n, device="cuda"), torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
        T = pn.Tensor.from_torch
        O, SA, SW = T(out), T(sa), T(sw)
        torch.cuda.synchronize()
        assert pn.core._lib.neural_linear_q8(O._ptr, a.data_ptr(), k, SA._ptr, w.data_ptr(), ld, SW._ptr, k, None, 0, 0.0,
                                             None) == 0
        pn.synchronize()
        assert torch.equal(out, a.float() @ w[:, :k].float().t().contiguous())  # sums below 2^24
    del w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", DT)
def test_module(pn, rng, dt):
    T = pn.Tensor
    c = _case(rng, 12, 100, 37, dt)
    weight, x = rng.normal(0, 0.1, (37, 100)).astype(dt), rng.normal(0, 1, (3, 4, 100)).astype(dt)
    q, qx = pn.QuantizedRows(T.from_numpy(weight)), pn.QuantizedRows(T.from_numpy(x))
    c.update(a=qx.codes().reshape(12, 100), w=q.codes(), sa=qx.scale.numpy(), sw=q.scale.numpy())
    lin = pn.QuantizedLinear(T.from_numpy(weight), T.from_numpy(c["bias"]), activation="gelu")
    want = _act(pn, _scaled(c), 4, 0.0) + c["res"]
    res = T.from_numpy(c["res"].reshape(3, 4, 37))
    for arg in (T.from_numpy(x), qx):
        same_bits(lin(arg, res).numpy().reshape(12, 37), want)
    assert lin.in_features == 100 and lin.out_features == 37
    # the codes' error: half a step of each row's scale, over a sum of 100 products
    y = pn.QuantizedLinear(q)(T.from_numpy(x)).numpy().reshape(12, 37).astype(np.float64)
    xf, wf = x.reshape(12, 100).astype(np.float64), weight.astype(np.float64)
    lim = (0.5 * c["sa"][:, None] * np.abs(wf).sum(1) + 0.5 * c["sw"] * np.abs(xf).sum(1)[:, None]
           + 25 * c["sa"][:, None] * c["sw"]) * 1.001
    assert (np.abs(y - xf @ wf.T) <= lim).all()
    with pytest.raises(ValueError):
        lin(T.zeros([3, 99]))
