"""Log probabilities of given tokens, entropy, top alternatives and their gradient, against
long double forms (tests/serving_ref.py) with bounds that count roundings; indices exactly.
Few and many rows, vocabularies around every form's limits, ties, masks that leave few
logits or none, rows that are not used, NaN and infinities, temperatures, alignment,
streams, graphs, threads and the refusals; a quantized layer's path to its answer."""

import numpy as np
import pytest

import serving_ref as ref
from conftest import GPU, same_bits
from sublayer_ref import within

pytestmark = GPU

DT = [np.float32, np.float64]
VOCAB = [1, 2, 3, 5, 17, 63, 64, 65, 100, 255, 256, 257, 511, 1000, 1023, 1024, 1025, 2047, 2049, 4095, 4096, 4097, 5003,
         8192, 8193, 12289, 16383, 16384, 16385, 20011, 32000, 32769, 50257, 65536, 65537, 131072, 150001]


def _p(t):
    return t._ptr if t is not None else None


def _case(rng, rows, V, dt, masked=0.0, unused=0.2):
    x = rng.normal(0, 2.5, (rows, V))
    tokens = rng.integers(0, V, rows)
    x[np.arange(rows), rng.integers(0, V, rows)] += 8
    sure = rng.random(rows) < 0.3
    x[np.arange(rows)[sure], tokens[sure]] += 30  # nearly all the probability
    if masked:
        x[rng.random((rows, V)) < masked] = -np.inf
    if rows > 2 and unused:
        tokens[rng.random(rows) < unused] = -1
    return x.astype(dt), tokens.astype(np.int64)


def _forward(pn, x, tokens, k=0, temperature=1.0, want=("logprob", "entropy", "lse", "ids", "top")):
    import torch
    T, rows = pn.Tensor, x.shape[0]
    X = T.from_numpy(x)
    o = {n: T.create([rows], X.dtype) for n in ("logprob", "entropy", "lse")}
    o["top"] = T.create([rows, max(k, 1)], X.dtype)
    ids = torch.full((rows, max(k, 1)), -7, dtype=torch.int64, device="cuda")
    tok = torch.from_numpy(tokens).cuda() if tokens is not None else None
    torch.cuda.synchronize()
    P = lambda n: o[n]._ptr if n in want else None  # noqa: E731
    rc = pn.core._lib.neural_token_logprobs_forward(
        P("logprob"), P("entropy"), P("lse"), ids.data_ptr() if k and "ids" in want else None, P("top") if k else None, k,
        X._ptr, tok.data_ptr() if tok is not None else None, temperature)
    assert rc == 0
    pn.synchronize()
    got = {n: o[n].numpy() for n in ("logprob", "entropy", "lse")}
    got["ids"], got["top"] = ids.cpu().numpy()[:, :k], o["top"].numpy()[:, :k]
    return got


def _backward(pn, x, tokens, g, e, lse, entropy, temperature=1.0):
    import torch
    T = pn.Tensor
    t = [None if v is None else T.from_numpy(v) for v in (g, e, x)]
    s = [None if v is None else T.from_numpy(v) for v in (lse, entropy)]
    tok = torch.from_numpy(tokens).cuda() if tokens is not None else None
    dx = T.create(x.shape, t[2].dtype)
    torch.cuda.synchronize()
    rc = pn.core._lib.neural_token_logprobs_backward(dx._ptr, _p(t[0]), _p(t[1]), t[2]._ptr,
                                                     tok.data_ptr() if tok is not None else None, _p(s[0]), _p(s[1]),
                                                     temperature)
    assert rc == 0
    return dx.numpy()


def _check(pn, x, tokens, k=5, temperature=1.0):
    got = _forward(pn, x, tokens, k, temperature)
    want, bound = ref.logprobs(x, tokens, k, temperature)
    assert np.array_equal(got["ids"], want["ids"]), np.argwhere(got["ids"] != want["ids"])[:3]
    for n in ("logprob", "entropy", "lse", "top"):
        within(got[n], want[n], bound[n], n)
    return got


def _check_grad(pn, rng, x, tokens, got, temperature=1.0):
    rows, dt = x.shape[0], x.dtype.type
    g, e = rng.normal(0, 1, rows).astype(dt), rng.normal(0, 1, rows).astype(dt)
    for a, b in ((g, e), (g, None), (None, e)):
        dx = _backward(pn, x, tokens, a, b, got["lse"], got["entropy"], temperature)
        want, bound = ref.logprobs_grad(x, tokens, a, b, got["lse"], got["entropy"], temperature)
        within(dx, want, bound, "dx")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", VOCAB)
def test_vocabularies(pn, rng, dt, V):
    rows = 7 if V > 20000 else 23
    x, tokens = _case(rng, rows, V, dt)
    got = _check(pn, x, tokens, 20)
    _check_grad(pn, rng, x, tokens, got)
    for k in (1, 64):
        _check(pn, x[:3], np.abs(tokens[:3]) % V, k, 0.7)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,V", [(1, 1), (1, 100), (1, 131072), (2, 50257), (64, 32000), (300, 5003), (1000, 1000),
                                    (2100, 257), (5000, 64), (20000, 10), (3000, 1025), (600, 17000)])
def test_row_counts(pn, rng, dt, rows, V):
    x, tokens = _case(rng, rows, V, dt)
    got = _check(pn, x, tokens, 8, 1.3)
    _check_grad(pn, rng, x, tokens, got, 1.3)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 7, 8, 16, 20, 31, 32, 33, 50, 63, 64])
def test_alternatives(pn, rng, k):
    for rows, V in ((3, 40), (3, 3000), (3, 70001), (400, 700)):
        x, tokens = _case(rng, rows, V, np.float32)
        _check(pn, x, tokens, k)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [50, 300, 1024, 5000, 16384, 40000, 131072])
def test_ties_and_orders(pn, rng, dt, V):
    """All equal, few distinct values, sorted both ways, zeros of both signs, the largest ones
    in one place or one stride of the row: ids by value, then by index."""
    j = np.arange(V)
    rows = [np.zeros(V), np.full(V, -3.5), j % 3, (j * 7919) % 11, j / V, -j / V, np.where(j % 2, 0.0, -0.0),
            np.where(j < V // 2, 5.0, 5.0 + (j % 5)), np.where(j % 1024 < 4, 9.0, -(j % 17) * 1.0),
            np.where(j % 1024 >= 768, -5.0, (j % 89) * 0.125), np.where(j % 64 == 7, 3.0 + (j % 31), 0.0),
            np.where(j == V - 1, 1.0, 0.0)]
    x = np.array(rows).astype(dt)
    tokens = rng.integers(0, V, x.shape[0])
    for k in (1, 20, 64):
        _check(pn, x, tokens, k)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [6, 300, 5000, 33000, 131072])
def test_masks(pn, rng, dt, V):
    """Most logits masked, all but one, all of them, the token itself; the gradient too."""
    x, tokens = _case(rng, 12, V, dt, masked=0.9, unused=0)
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, V // 2] = 1.5
    x[2, tokens[2]] = -np.inf
    x[3] = -np.inf
    x[3, -3:] = [1.0, 2.0, 1.0]
    tokens[4] = -1
    tokens[5] = -(1 << 62)
    got = _check(pn, x, tokens, 10, 0.9)
    assert got["logprob"][0] == -np.inf and got["entropy"][0] == 0 and got["lse"][0] == -np.inf
    assert (got["ids"][0] == -1).all() and (got["top"][0] == -np.inf).all()
    assert got["entropy"][1] == 0 and got["ids"][1].tolist() == [V // 2] + [-1] * 9 and got["top"][1, 0] == 0
    assert got["ids"][3, :4].tolist() == [V - 2, V - 3, V - 1, -1]
    _check_grad(pn, rng, x, tokens, got, 0.9)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [6, 300, 5000, 33000, 131072])
def test_nan_and_infinity(pn, rng, dt, V):
    """NaN and +inf make their row NaN, in rows that are not used nothing; a token past the
    vocabulary makes its log probability NaN, and the row's gradient."""
    x, tokens = _case(rng, 12, V, dt, unused=0)
    clean = _forward(pn, x, tokens, 4)
    x[1, V // 3] = np.nan
    x[2, V - 1] = np.inf
    x[3] = np.nan
    x[4, 0], x[4, V - 1] = np.nan, np.inf
    x[5], tokens[5] = np.nan, -1
    x[6, :], tokens[6] = np.inf, -9
    tokens[7], tokens[8] = V, 1 << 40
    got = _check(pn, x, tokens, 4)
    bad = [1, 2, 3, 4]
    for n in ("logprob", "entropy", "top"):
        assert np.isnan(got[n][bad]).all()
    assert (got["ids"][bad] == -1).all() and np.isnan(got["logprob"][[7, 8]]).all()
    for n in clean:
        assert np.array_equal(got[n][[0, 9, 10, 11]], clean[n][[0, 9, 10, 11]])
    g = np.ones(12, dt)
    dx = _backward(pn, x, tokens, g, g, got["lse"], got["entropy"])
    assert np.isnan(dx[bad + [7, 8]]).all() and not dx[[5, 6]].any()
    assert np.isfinite(dx[[0, 9, 10, 11]]).all()
    dx = _backward(pn, x, tokens, None, g, got["lse"], got["entropy"])  # the entropy's alone: the token does not matter
    assert np.isfinite(dx[[7, 8]]).all()


@pytest.mark.parametrize("dt", DT)
def test_extreme_logits(pn, rng, dt):
    """One far above the rest, huge and tiny values and temperatures."""
    x, tokens = _case(rng, 8, 777, dt, unused=0)
    x[0] *= 30
    x[1] *= dt(1e4)
    x[2] = dt(3e38) if dt == np.float32 else 1e300
    x[3] = -x[2]
    x[4] *= dt(1e-30)
    x[5, tokens[5]] = 60.0
    for temperature in (1.0, 1e-3, 50.0):
        y = x.copy()
        if temperature < 1:
            y[2:4] = 0
        _check(pn, y, tokens, 6, temperature)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("temperature", [1e-10, 1e10])
def test_extreme_temperatures(pn, rng, dt, temperature):
    """The largest and smallest, with logits of their size, and with ordinary ones that are all
    alike beside the largest; masked ones among them."""
    x, tokens = _case(rng, 6, 777, dt, masked=0.3, unused=0)
    got = _check(pn, x * dt(temperature), tokens, 6, temperature)
    assert not np.isnan(got["logprob"]).any()
    if temperature > 1:
        _check(pn, x, tokens, 6, temperature)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [1000, 1111, 4099, 9000])
def test_rows_in_any_batch(pn, rng, dt, V):
    """A row has the bits of its batch of three in one of 600, which other forms take: values in no
    order, all alike, and mostly masked."""
    x, tokens = _case(rng, 600, V, dt)
    x[1] = 0.25
    x[2, rng.random(V) < 0.99] = -np.inf
    x[3] = np.where(rng.random(V) < 0.5, 1, 2)
    for k in (1, 20, 64):
        whole = _forward(pn, x, tokens, k)
        for r in (0, 2, 597):
            part = _forward(pn, x[r:r + 3], tokens[r:r + 3], k)
            for n in ("logprob", "entropy", "lse", "top"):
                same_bits(part[n], whole[n][r:r + 3])
            assert np.array_equal(part["ids"], whole["ids"][r:r + 3])


def test_outputs_left_out(pn, rng):
    """Every output alone has the bits that it has beside the others; no tokens: every row used."""
    for rows, V in ((5, 300), (5, 40000), (400, 2000)):
        x, tokens = _case(rng, rows, V, np.float32)
        full = _forward(pn, x, tokens, 7)
        for n in ("logprob", "entropy", "lse", "ids", "top"):
            same_bits(_forward(pn, x, tokens, 7, want=(n,))[n], full[n])
        x, tokens = _case(rng, rows, V, np.float32, unused=0)
        full = _forward(pn, x, tokens, 7)
        none = _forward(pn, x, None, 7, want=("entropy", "lse", "ids", "top"))
        for n in ("entropy", "lse", "ids", "top"):
            same_bits(none[n], full[n])
        e = rng.normal(0, 1, rows).astype(np.float32)
        same_bits(_backward(pn, x, None, None, e, full["lse"], full["entropy"]),
                  _backward(pn, x, tokens, None, e, full["lse"], full["entropy"]))


def test_gradients_by_differences(pn, rng):
    """f64, against central differences of a weighted sum of logprob and entropy (step^2 / 6
    times a third derivative of order 10: 2e-8; held to 1e-6)."""
    rows, V, temperature = 4, 23, 0.8
    x, tokens = _case(rng, rows, V, np.float64)
    x = np.clip(x, -5, 5)
    tokens[:] = [3, -1, 22, 0]
    g, e = rng.normal(0, 1, rows), rng.normal(0, 1, rows)

    def loss(v):
        o = _forward(pn, v, tokens, 0, temperature)
        return float((g * o["logprob"]).sum() + (e * o["entropy"]).sum())

    o = _forward(pn, x, tokens, 0, temperature)
    dx = _backward(pn, x, tokens, g, e, o["lse"], o["entropy"], temperature).reshape(-1)
    for at in range(0, rows * V, 3):
        lo, hi = x.copy(), x.copy()
        lo.reshape(-1)[at] -= 1e-4
        hi.reshape(-1)[at] += 1e-4
        d = (loss(hi) - loss(lo)) / 2e-4
        assert abs(d - dx[at]) <= 1e-6 * max(1.0, abs(d)), at


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [7, 65, 1001, 5003, 40001])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_alignment_guards_in_place(pn, rng, dt, V, shift):
    import torch
    rows, k = 6, 5
    x, tokens = _case(rng, rows, V, dt)
    want = _forward(pn, x, tokens, k)
    g, e = rng.normal(0, 1, rows).astype(dt), rng.normal(0, 1, rows).astype(dt)
    grad = _backward(pn, x, tokens, g, e, want["lse"], want["entropy"])
    tdt = torch.float32 if dt == np.float32 else torch.float64
    held = []

    def placed(v, t=tdt):
        big = torch.full((v.size + 64,), 5, dtype=t, device="cuda")
        view = big[16 + shift:16 + shift + v.size].view(v.shape)
        view.copy_(torch.from_numpy(v))
        held.append((big, v.size))
        return view

    X, G, E = placed(x), placed(g), placed(e)
    o = {n: placed(np.zeros_like(want[n])) for n in ("logprob", "entropy", "lse", "top")}
    ids, tok = placed(np.zeros((rows, k), np.int64), torch.int64), placed(tokens, torch.int64)
    T = {n: pn.Tensor.from_torch(v) for n, v in {**o, "x": X, "g": G, "e": E}.items()}
    torch.cuda.synchronize()
    lib = pn.core._lib
    P = lambda n: T[n]._ptr  # noqa: E731
    assert lib.neural_token_logprobs_forward(P("logprob"), P("entropy"), P("lse"), ids.data_ptr(), P("top"), k, P("x"),
                                             tok.data_ptr(), 1.0) == 0
    pn.synchronize()
    for n in o:
        same_bits(o[n].cpu().numpy(), want[n])
    assert np.array_equal(ids.cpu().numpy(), want["ids"])
    assert lib.neural_token_logprobs_backward(P("x"), P("g"), P("e"), P("x"), tok.data_ptr(), P("lse"), P("entropy"),
                                              1.0) == 0
    pn.synchronize()
    same_bits(X.cpu().numpy(), grad)
    for big, n in held:
        assert bool((big[:16 + shift] == 5).all()) and bool((big[16 + shift + n:] == 5).all())


def test_host_buffers_and_empty(pn, rng):
    lib, T = pn.core._lib, pn.Tensor
    for V in (90, 40000):
        x, tokens = _case(rng, 5, V, np.float32)
        want = _forward(pn, x, tokens, 3)
        o = {n: np.zeros_like(want[n]) for n in ("logprob", "entropy", "lse", "top")}
        ids = np.zeros((5, 3), np.int64)
        t = {n: T.from_numpy_zero_copy(v) for n, v in {**o, "x": x}.items()}
        P = lambda n: t[n]._ptr  # noqa: E731
        assert lib.neural_token_logprobs_forward(P("logprob"), P("entropy"), P("lse"), ids.ctypes.data, P("top"), 3, P("x"),
                                                 tokens.ctypes.data, 1.0) == 0
        for n in o:
            same_bits(o[n], want[n])
        assert np.array_equal(ids, want["ids"])
    e, z = T.create([0, 5]), T.create([0])
    t0 = np.zeros(1, np.int64)
    assert lib.neural_token_logprobs_forward(z._ptr, None, None, None, None, 0, e._ptr, t0.ctypes.data, 1.0) == 0


def test_refusals(pn):
    import torch
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    x, dx, a, b, c, top = T.zeros([4, 9]), T.zeros([4, 9]), T.zeros([4]), T.zeros([4]), T.zeros([4]), T.zeros([4, 3])
    ids = torch.full((4, 3), 6, dtype=torch.int64, device="cuda")
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    f, k = lib.neural_token_logprobs_forward, lib.neural_token_logprobs_backward
    ok = [a._ptr, b._ptr, c._ptr, ids.data_ptr(), top._ptr, 3, x._ptr, tok.data_ptr(), 1.0]
    gk = [dx._ptr, a._ptr, b._ptr, x._ptr, tok.data_ptr(), c._ptr, T.zeros([4])._ptr, 1.0]
    held = T.zeros([4])
    gk[6] = held._ptr

    def with_(fn, args, **kw):
        v = list(args)
        for i, w in kw.items():
            v[int(i[1:])] = w
        return fn(*v)

    assert with_(f, ok, _6=None) == E.NULL_POINTER and with_(f, ok, _7=None) == E.NULL_POINTER
    assert f(None, None, None, None, None, 3, x._ptr, tok.data_ptr(), 1.0) == E.NULL_POINTER
    assert f(None, None, None, ids.data_ptr(), top._ptr, 0, x._ptr, tok.data_ptr(), 1.0) == E.NULL_POINTER
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-320, 9e-11, 1.1e10):
        assert with_(f, ok, _8=t) == E.INVALID_ARGUMENT and with_(k, gk, _7=t) == E.INVALID_ARGUMENT
    for n in (-1, 65):
        assert with_(f, ok, _5=n) == E.INVALID_ARGUMENT
    d4, d49, s5, s94, s0 = T.zeros([4], pn.float64), T.zeros([4, 9], pn.float64), T.zeros([5]), T.zeros([9, 4]), T.create([])
    for i in (0, 1, 2):
        assert with_(f, ok, **{f"_{i}": d4._ptr}) == E.DTYPE_MISMATCH
        assert with_(f, ok, **{f"_{i}": s5._ptr}) == E.SHAPE_MISMATCH
    assert with_(f, ok, _4=s5._ptr) == E.SHAPE_MISMATCH and with_(f, ok, _6=s0._ptr) == E.DIM_MISMATCH
    assert with_(f, ok, _1=ok[0]) == E.INVALID_ARGUMENT
    big = torch.zeros(8, 9, device="cuda")
    assert with_(f, ok, _6=T.from_torch(big[::2])._ptr) == E.INVALID_ARGUMENT
    inside = T.from_torch(big.view(-1)[2:6])
    assert with_(f, ok, _6=T.from_torch(big[:4])._ptr, _0=inside._ptr) == E.INVALID_ARGUMENT
    assert with_(f, ok, _6=T.from_torch(big)._ptr, _0=None, _1=None, _2=None, _4=None, _3=big.data_ptr()) == E.INVALID_ARGUMENT
    assert with_(f, ok, _3=tok.data_ptr()) == E.INVALID_ARGUMENT  # ids over the tokens
    for i in (0, 3, 5):
        assert with_(k, gk, **{f"_{i}": None}) == E.NULL_POINTER
    assert with_(k, gk, _1=None, _2=None) == E.NULL_POINTER and with_(k, gk, _4=None) == E.NULL_POINTER
    assert with_(k, gk, _6=None) == E.NULL_POINTER
    assert with_(k, gk, _0=d49._ptr) == E.DTYPE_MISMATCH and with_(k, gk, _0=s94._ptr) == E.SHAPE_MISMATCH
    assert with_(k, gk, _1=s5._ptr) == E.SHAPE_MISMATCH
    assert with_(k, gk, _3=T.from_torch(big[:4])._ptr, _0=T.from_torch(big[2:6])._ptr) == E.INVALID_ARGUMENT
    assert with_(k, gk, _0=T.from_torch(big[:4])._ptr, _1=inside._ptr) == E.INVALID_ARGUMENT
    for t in (a, b, c, top, dx):
        assert not t.numpy().any()
    assert bool((ids == 6).all()) and not big.cpu().numpy().any()


@pytest.mark.parametrize("rows,V", [(3, 70001), (300, 1500)])
def test_graphs_and_streams(pn, rng, rows, V):
    """Two captured steps (forward with alternatives, gradient) on two streams, replayed at once
    with eager calls in between: each its own workspace; tokens changed between replays."""
    import torch
    lib, T, k = pn.core._lib, pn.Tensor, 9
    streams, sides = [torch.cuda.Stream(), torch.cuda.Stream()], []
    try:
        for i in range(2):
            x, tokens = _case(rng, rows, V, np.float32)
            g, e = rng.normal(0, 1, rows).astype(np.float32), rng.normal(0, 1, rows).astype(np.float32)
            t = {n: torch.zeros(rows, device="cuda") for n in ("logprob", "entropy", "lse")}
            t.update(x=torch.from_numpy(x).cuda(), g=torch.from_numpy(g).cuda(), e=torch.from_numpy(e).cuda(),
                     dx=torch.zeros(rows, V, device="cuda"), top=torch.zeros(rows, k, device="cuda"))
            ids, tok = torch.zeros(rows, k, dtype=torch.int64, device="cuda"), torch.from_numpy(tokens).cuda()
            w = {n: T.from_torch(v) for n, v in t.items()}
            pn.set_stream(streams[i].cuda_stream)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[i]):
                P = lambda n: w[n]._ptr  # noqa: E731
                assert lib.neural_token_logprobs_forward(P("logprob"), P("entropy"), P("lse"), ids.data_ptr(), P("top"), k,
                                                         P("x"), tok.data_ptr(), 1.0) == 0
                assert lib.neural_token_logprobs_backward(P("dx"), P("g"), P("e"), P("x"), tok.data_ptr(), P("lse"),
                                                          P("entropy"), 1.0) == 0
            sides.append((x, g, e, t, ids, tok, w, graph))
        pn.set_stream(None)
        torch.cuda.synchronize()
        for replay in range(3):
            for i, side in enumerate(sides):
                with torch.cuda.stream(streams[i]):
                    side[-1].replay()
            torch.cuda.synchronize()
            for x, g, e, t, ids, tok, w, graph in sides:
                tokens = tok.cpu().numpy()
                want = _forward(pn, x, tokens, k)
                for n in ("logprob", "entropy", "lse", "top"):
                    same_bits(t[n].cpu().numpy(), want[n])
                    t[n].fill_(9.0)
                assert np.array_equal(ids.cpu().numpy(), want["ids"])
                same_bits(t["dx"].cpu().numpy(), _backward(pn, x, tokens, g, e, want["lse"], want["entropy"]))
                ids.fill_(-3)
                tok.copy_(torch.randint(-1, V, (rows,), device="cuda"))
            lib.neural_hip_empty_cache()
            torch.cuda.synchronize()
    finally:
        pn.set_stream(None)


def test_host_memory_while_capturing(pn, rng):
    """Tokens, ids and codes in host memory are refused in a captured call, which goes on."""
    import torch
    lib, T = pn.core._lib, pn.Tensor
    x, lp, dx = torch.randn(3, 100, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, 100, device="cuda")
    dev = torch.tensor([1, 2, 3], device="cuda")
    tok, ids, codes = np.array([1, 2, 3]), np.full((3, 2), 7), np.full((3, 100), 7, np.int8)
    w, hw = torch.ones(100, 100, dtype=torch.int8, device="cuda"), np.ones((100, 100), np.int8)
    sw = torch.ones(100, device="cuda")
    X, LP, DX, SW = (T.from_torch(v) for v in (x, lp, dx, sw))
    want = torch.log_softmax(x.double(), 1)[[0, 1, 2], [1, 2, 3]].cpu().numpy()
    s = torch.cuda.Stream()
    pn.set_stream(s.cuda_stream)
    try:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            rcs = [lib.neural_token_logprobs_forward(LP._ptr, None, None, None, None, 0, X._ptr, tok.ctypes.data, 1.0),
                   lib.neural_token_logprobs_forward(LP._ptr, None, None, ids.ctypes.data, None, 2, X._ptr,
                                                     dev.data_ptr(), 1.0),
                   lib.neural_token_logprobs_backward(DX._ptr, LP._ptr, None, X._ptr, tok.ctypes.data, LP._ptr, None, 1.0),
                   lib.neural_quantize_rows(codes.ctypes.data, 100, LP._ptr, X._ptr),
                   lib.neural_rms_norm_forward_q8(codes.ctypes.data, 100, LP._ptr, None, X._ptr, None, None, 0.1),
                   lib.neural_linear_q8(DX._ptr, codes.ctypes.data, 100, LP._ptr, w.data_ptr(), 100, SW._ptr, 100, None, 0,
                                        0.0, None),
                   lib.neural_linear_q8(DX._ptr, w.data_ptr(), 100, LP._ptr, hw.ctypes.data, 100, SW._ptr, 100, None, 0,
                                        0.0, None)]
            assert lib.neural_token_logprobs_forward(LP._ptr, None, None, None, None, 0, X._ptr, dev.data_ptr(), 1.0) == 0
        assert rcs == [pn.NeuralError.INVALID_ARGUMENT] * 7, rcs
        for _ in range(2):
            lp.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert np.abs(lp.cpu().numpy() - want).max() < 1e-5
        assert (ids == 7).all() and (codes == 7).all()
    finally:
        pn.set_stream(None)


def test_strided_tokens(pn, rng):
    """In host memory they are copied; in device memory refused, as torch's copy would be on a stream
    of its own."""
    import torch
    x, _ = _case(rng, 3, 50, np.float32)
    m, tok = pn.TokenLogProbs(), torch.tensor([4, 0, 7, 0, 9, 0])
    got = m(pn.Tensor.from_numpy(x), tok[::2]).logprob.numpy()
    same_bits(got, _forward(pn, x, np.array([4, 7, 9]))["logprob"])
    with pytest.raises(ValueError):
        m(pn.Tensor.from_numpy(x), tok.cuda()[::2])


def test_threads(pn, rng):
    import threading
    cases = [_case(rng, 3 + i, 20011 + 7000 * i, np.float32) for i in range(4)]
    want = [_forward(pn, x, t, 12) for x, t in cases]
    bad = []

    def work(i):
        for _ in range(5):
            got = _forward(pn, *cases[i], 12)
            if not all(np.array_equal(got[n], want[i][n]) for n in got):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_many_elements(pn):
    """More than 2^32 logits: the first and last rows have what they have alone."""
    import torch
    V, rows = 50257, 86001
    torch.cuda.empty_cache()
    pn.core._lib.neural_hip_empty_cache()
    if torch.cuda.mem_get_info()[0] < 4 * rows * V + (4 << 30):
        pytest.skip("not enough free device memory")
    lib, T = pn.core._lib, pn.Tensor
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    one = torch.randn(3, V, device="cuda", generator=gen)
    x = torch.zeros(rows, V, device="cuda")
    x[-3:] = one
    tok = torch.arange(rows, device="cuda") % V
    o = {n: torch.empty(rows, device="cuda") for n in ("logprob", "entropy", "lse")}
    g = torch.ones(rows, device="cuda")
    ids, top = torch.empty(rows, 4, dtype=torch.int64, device="cuda"), torch.empty(rows, 4, device="cuda")
    w = {n: T.from_torch(v) for n, v in {**o, "x": x, "g": g, "top": top}.items()}
    P = lambda n: w[n]._ptr  # noqa: E731
    torch.cuda.synchronize()
    assert lib.neural_token_logprobs_forward(P("logprob"), P("entropy"), P("lse"), ids.data_ptr(), P("top"), 4, P("x"),
                                             tok.data_ptr(), 1.0) == 0
    assert lib.neural_token_logprobs_backward(P("x"), P("g"), P("g"), P("x"), tok.data_ptr(), P("lse"), P("entropy"),
                                              1.0) == 0
    pn.synchronize()
    small, tokens = one.cpu().numpy(), tok[-3:].cpu().numpy()
    want, bound = ref.logprobs(small, tokens, 4, 1.0)
    for n in o:
        within(o[n][-3:].cpu().numpy(), want[n], bound[n], n)
    assert np.array_equal(ids[-3:].cpu().numpy(), want["ids"]) and ids[0].tolist() == [0, 1, 2, 3]
    gn = np.ones(3, np.float32)
    wg, bg = ref.logprobs_grad(small, tokens, gn, gn, o["lse"][-3:].cpu().numpy(), o["entropy"][-3:].cpu().numpy(), 1.0)
    within(x[-3:].cpu().numpy(), wg, bg, "dx")
    del x
    w.clear()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", DT)
def test_module(pn, rng, dt):
    T = pn.Tensor
    x, tokens = _case(rng, 12, 500, dt)
    m = pn.TokenLogProbs(temperature=0.9, top_k=6)
    o = m(T.from_numpy(x.reshape(3, 4, 500)), tokens)
    want = _forward(pn, x, tokens, 6, 0.9)
    same_bits(o.logprob.numpy(), want["logprob"])
    same_bits(o.entropy.numpy(), want["entropy"])
    same_bits(o.top_logprobs.numpy(), want["top"])
    assert np.array_equal(o.top_ids, want["ids"])
    g, e = rng.normal(0, 1, 12).astype(dt), rng.normal(0, 1, 12).astype(dt)
    dx = m.backward(T.from_numpy(g), T.from_numpy(e))
    same_bits(dx.numpy().reshape(12, 500), _backward(pn, x, tokens, g, e, want["lse"], want["entropy"], 0.9))
    o = pn.TokenLogProbs()(T.from_numpy(x))
    assert o.logprob is None and o.top_ids is None
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            pn.TokenLogProbs(bad)
    with pytest.raises(ValueError):
        pn.TokenLogProbs(top_k=65)
    with pytest.raises(ValueError):
        m(T.from_numpy(x), tokens[:5])


@pytest.mark.parametrize("rows", [1, 5, 70])
def test_a_layers_path_to_its_answer(pn, rng, rows):
    """The operators in a row, as a serving program has them: residual add and norm to 8 bits,
    the wide product with its activation, the narrow one back onto the residual stream, the
    last norm, the vocabulary's product, log probabilities and alternatives.  Every stage is
    checked from what the stage before it left, in long double and whole numbers."""
    d, wide, V = 96, 260, 1003
    T = pn.Tensor
    n1, n2 = pn.RMSNorm(d), pn.RMSNorm(d)
    n1.gamma, n2.gamma = (T.from_numpy(rng.normal(1, 0.2, d).astype(np.float32)) for _ in range(2))
    weights = [rng.normal(0, a ** -0.5, (b, a)).astype(np.float32) for a, b in ((d, wide), (wide, d), (d, V))]
    bias = rng.normal(0, 0.1, wide).astype(np.float32)
    up = pn.QuantizedLinear(T.from_numpy(weights[0]), T.from_numpy(bias), activation="swish")
    down, head = pn.QuantizedLinear(T.from_numpy(weights[1])), pn.QuantizedLinear(T.from_numpy(weights[2]))
    x, res = rng.normal(0, 1, (rows, d)).astype(np.float32), rng.normal(0, 1, (rows, d)).astype(np.float32)
    q1, hidden = n1.forward_q8(T.from_numpy(x), T.from_numpy(res))
    mid = up(q1)
    stream = down(mid, hidden)
    q2 = n2.forward_q8(stream)
    logits = head(q2)
    tokens = rng.integers(0, V, rows)
    out = pn.TokenLogProbs(top_k=5)(logits, tokens)
    u = 2.0 ** -24
    h = res + x
    same_bits(hidden.numpy(), h)
    wn = h.astype(np.float64) * n1.gamma.numpy().astype(np.float64)
    assert np.array_equal(q1.codes(), ref.codes(wn)[0])
    L = np.longdouble

    def product(q, lin):
        acc = q.codes().astype(np.float64) @ lin.weight.codes().astype(np.float64).T
        return acc.astype(L) * q.scale.numpy().astype(L)[:, None] * lin.weight.scale.numpy().astype(L)

    z = product(q1, up) + bias
    s = z / (1 + np.exp(-z))
    # one rounding of z (swish's slope is below 1.1), then the float formula: three of its results'
    lim = 1.2 * u * np.abs(z) + 4 * u * np.abs(s) + 1e-12
    assert (np.abs(mid.numpy() - s) <= lim).all()
    qm = pn.QuantizedRows(mid)
    want = product(qm, down) + h
    assert (np.abs(stream.numpy() - want) <= 1.01 * u * (np.abs(want) + np.abs(want - h))).all()
    assert np.array_equal(q2.codes(), ref.codes(stream.numpy().astype(np.float64) * n2.gamma.numpy())[0])
    want = product(q2, head)
    assert (np.abs(logits.numpy() - want) <= 1.01 * u * np.abs(want)).all()
    want, bound = ref.logprobs(logits.numpy(), tokens, 5, 1.0)
    within(out.logprob.numpy(), want["logprob"], bound["logprob"], "logprob")
    assert np.array_equal(out.top_ids, want["ids"])
    # and all of it against the layer without quantization: within the codes' steps (127 levels)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6) * n1.gamma.numpy()
    zf = y @ weights[0].T + bias
    sf = h + (zf / (1 + np.exp(-zf))) @ weights[1].T
    yf = sf / np.sqrt((sf * sf).mean(-1, keepdims=True) + 1e-6) * n2.gamma.numpy()
    lf = yf @ weights[2].T
    assert np.sqrt(np.mean((logits.numpy() - lf) ** 2)) <= 0.05 * np.sqrt(np.mean(lf ** 2))
