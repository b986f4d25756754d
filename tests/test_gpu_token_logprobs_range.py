"""Token log probabilities over the whole range of temperatures and logits: the gradient against
a softmax in long double from the logits alone, not from the saved log-sum-exp."""

import numpy as np
import pytest

import serving_ref as ref
from conftest import GPU, same_bits
from sublayer_ref import D, U, within
from test_gpu_token_logprobs import _backward, _forward

pytestmark = GPU

DT = [np.float32, np.float64]
L = np.longdouble


def _grad_of_logits(x, tokens, g, e, temperature, four=False):
    """The gradient, and its bound for a call from the lse and entropy that forward leaves (four: from
    its four values, log s rounded to the type: u log s more).

    s is off by es of itself (serving_ref.logprobs: each exponential to 8 u, each term's rounding in
    double).  log p = (x - m) / T - log s: off by es and by 4 D of its terms.  Where |lse| < 64 it may be
    x / T - lse instead, with lse rounded to the type: u |lse| more.  p: its exponential, 8 u, beside
    that; the entropy: the forward call's bound; then as serving_ref.logprobs_grad."""
    rows, V = x.shape
    u, inv = U[x.dtype], 1 / L(temperature)
    with np.errstate(all="ignore"):
        xl = x.astype(L)
        m = xl.max(1, keepdims=True)
        masked = np.isneginf(m)
        d = np.where(masked, L(0), xl - np.where(masked, L(0), m)) * inv
        p = np.exp(d)
        p = np.where(np.isneginf(xl), L(0), p)
        dz = np.where(np.isneginf(d), L(0), d)
        s = p.sum(1, keepdims=True)
        mine = np.where(dz == 0, L(0), p)
        es = u * (mine * (8 + np.abs(dz))).sum(1, keepdims=True) / s + (V + 8) * D * 2
        ls = np.log(s)
        lse = m * inv + ls
        p, lp = p / s, dz - ls
        want, bound = ref.logprobs(x, tokens, 0, temperature)
        h, bh = want["entropy"][:, None], bound["entropy"][:, None]
        at = (np.arange(V) == tokens[:, None]).astype(L)
        gl = np.zeros((rows, 1), L) if g is None else g.astype(L)[:, None]
        el = np.zeros((rows, 1), L) if e is None else e.astype(L)[:, None]
        lz = np.where(p == 0, L(0), lp + h)
        grad = (gl * (at - p) - el * p * lz) * inv
        off = es + 4 * D * (np.abs(dz) + np.abs(ls)) + (u * np.abs(ls) if four else 0)
        off = off + np.where(np.abs(lse) < 65, u * np.abs(lse) + 4 * D * (np.abs(m * inv) + np.abs(dz) + np.abs(lse)), 0)
        dp = np.where(p == 0, L(0), p * (8 * u + off))
        dl = off + bh + u * np.abs(lz)
        err = np.abs(gl) * (dp + 2 * u * np.abs(at - p)) + np.abs(el) * (dp * np.abs(lz) + p * dl + 3 * u * p * np.abs(lz))
        tiny = ref.tiny_of(x.dtype) * (1 + inv) * (1 + np.abs(gl) + np.abs(el) * (1 + np.abs(lz)))
        limit = 1.02 * inv * err + 2 * u * np.abs(grad) + 4 * tiny
        zero = masked | (tokens < 0)[:, None]
    return np.where(zero, L(0), grad), np.where(zero, L(0), limit)


def _rows(rng, V, dt, temperature):
    """Rows whose lse lies anywhere: sure ones with the likeliest token and another, ties, rivals within
    a few temperatures, masks, rows that are not used, large and huge logits of both signs."""
    x = rng.normal(0, 2.5, (14, V))
    tokens = rng.integers(0, V, 14)
    top = rng.integers(0, V, 14)
    x[np.arange(14), top] += 22.7
    tokens[0] = top[0]
    x[2, tokens[2]] = x[2, top[2]]
    near = rng.integers(0, V, 9)
    x[3, near] = x[3, top[3]] - temperature * np.arange(9) / 2
    tokens[3] = near[1]
    x[4] = np.clip(temperature * rng.normal(0, 2.5, V), -1e30, 1e30)
    x[5, rng.random(V) < 0.9] = -np.inf
    tokens[5] = int(np.argmax(x[5]))
    x[6] = -np.inf
    tokens[7] = -1
    x[8] = 1e5 * rng.normal(0, 1, V)
    tokens[8] = int(np.argmax(x[8]))
    x[9] = 1e30 * rng.normal(0, 1, V)
    tokens[9] = int(np.argmax(x[9]))
    x[10] = -1e30
    x[11] = rng.normal(0, 1, V)
    x[12] = -300.0 + x[12]
    tokens[12] = top[12]
    return x.astype(dt), tokens.astype(np.int64)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [3, 300, 1000, 2000, 4096, 5003, 40001])
@pytest.mark.parametrize("temperature", [1e-10, 1e-6, 1e-4, 1e-3, 0.01, 0.3, 1.0, 30.0, 1e4, 1e10])
def test_gradient_of_the_logits(pn, rng, dt, V, temperature):
    x, tokens = _rows(rng, V, dt, temperature)
    got = _forward(pn, x, tokens, 0, temperature)
    g, e = rng.normal(0, 1, 14).astype(dt), rng.normal(0, 1, 14).astype(dt)
    for a, b in ((g, None), (None, e), (g, e)):
        dx = _backward(pn, x, tokens, a, b, got["lse"], got["entropy"], temperature)
        want, bound = _grad_of_logits(x, tokens, a, b, temperature)
        within(dx, want, bound, "dx")
    assert not dx[[6, 7]].any()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [300, 2000, 4096, 4097, 5003, 40001])
@pytest.mark.parametrize("shift", [0, 1, 5])
def test_gradient_over_the_logits(pn, rng, dt, V, shift):
    """In place, from any address, rows of both kinds side by side: the bits of a gradient elsewhere,
    and nothing beside it touched."""
    import torch
    temperature, rows = 0.01, 14
    x, tokens = _rows(rng, V, dt, temperature)
    x[::3] *= dt(0.01)  # |lse| < 64 in every third row
    got = _forward(pn, x, tokens, 0, temperature)
    near = np.abs(got["lse"]) < 64
    assert near.any() and not near.all()
    g, e = rng.normal(0, 1, rows).astype(dt), rng.normal(0, 1, rows).astype(dt)
    want = _backward(pn, x, tokens, g, e, got["lse"], got["entropy"], temperature)
    big = torch.full((x.size + 64,), 5, dtype=torch.float32 if dt == np.float32 else torch.float64, device="cuda")
    view = big[16 + shift:16 + shift + x.size].view(x.shape)
    view.copy_(torch.from_numpy(x))
    T = pn.Tensor
    X, tok = T.from_torch(view), torch.from_numpy(tokens).cuda()
    t = [T.from_numpy(v) for v in (g, e, got["lse"], got["entropy"])]
    torch.cuda.synchronize()
    assert pn.core._lib.neural_token_logprobs_backward(X._ptr, t[0]._ptr, t[1]._ptr, X._ptr, tok.data_ptr(), t[2]._ptr,
                                                       t[3]._ptr, temperature) == 0
    pn.synchronize()
    same_bits(view.cpu().numpy(), want)
    assert bool((big[:16 + shift] == 5).all()) and bool((big[16 + shift + x.size:] == 5).all())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 0.7])
def test_gradient_of_a_sure_token_by_module(pn, rng, dt, temperature):
    """The likeliest token's own gradient is g (1 - p) / T: nothing where nothing else is likely."""
    x, tokens = _rows(rng, 1000, dt, temperature)
    x, tokens = x[:1].copy(), tokens[:1]
    m = pn.TokenLogProbs(temperature=temperature)
    m(pn.Tensor.from_numpy(x), tokens)
    g = np.ones(1, dt)
    dx = m.backward(pn.Tensor.from_numpy(g)).numpy()
    want, bound = _grad_of_logits(x, tokens, g, None, temperature, True)
    within(dx, want, bound, "dx")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [3, 300, 513, 700, 3000, 5003, 20011, 40001])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 1e10])
def test_masks_of_the_lowest_value(pn, rng, dt, V, temperature):
    """Logits ruled out by the type's lowest value, or others far from the largest, in whole waves and
    parts: sums, alternatives, and the gradient."""
    low = np.finfo(dt).min
    x, tokens = _rows(rng, V, dt, 1.0)
    x[9:11] = x[3:5]
    tokens[9:11] = V // 2
    keep = {r: rng.integers(0, V, 3) for r in range(9)}
    for r, at in keep.items():
        row = np.full(V, (low, low / 2, -1e300 if dt == np.float64 else -1e30)[r % 3], dt)
        row[at], row[tokens[r]] = x[r, at], x[r, tokens[r]]
        x[r] = row
    x[6] = low
    x[11] = np.where(np.arange(V) < V // 2, low, -np.inf)
    x[11, V - 1] = 2.0
    got = _forward(pn, x, tokens, 5, temperature)
    want, bound = ref.logprobs(x, tokens, 5, temperature)
    for n in ("logprob", "entropy", "lse", "top"):
        with np.errstate(all="ignore"):
            rounded = want[n].astype(dt)
        within(got[n], np.where(np.isinf(rounded), rounded, want[n]), bound[n], n)  # (past the type's range)
    assert np.array_equal(got["ids"], want["ids"]) and not np.isnan(got["entropy"]).any()
    g, e = rng.normal(0, 1, 14).astype(dt), rng.normal(0, 1, 14).astype(dt)
    dx = _backward(pn, x, tokens, g, e, got["lse"], got["entropy"], temperature)
    want, bound = _grad_of_logits(x, tokens, g, e, temperature)
    within(dx, want, bound, "dx")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [40, 700, 40001])
@pytest.mark.parametrize("temperature", [2.0, 50.0, 1e10])
def test_differences_past_the_range(pn, rng, dt, V, temperature):
    """Logits of both signs near the type's largest value: (x - m) / T is within its range where x - m
    is not."""
    big = dt(0.9) * np.finfo(dt).max
    x = (rng.uniform(-1, 1, (6, V)) * big).astype(dt)
    x[:, V // 3] = big
    tokens = np.argmin(x, 1)
    tokens[4:] = np.argmax(x[4:], 1)
    x[3, 1:] = -big
    x[3, V // 3] = big
    got = _forward(pn, x, tokens, 7, temperature)
    want, bound = ref.logprobs(x, tokens, 7, temperature)
    assert np.isfinite(got["logprob"]).all()
    for n in ("logprob", "entropy", "lse", "top"):
        within(got[n], want[n], bound[n], n)
    assert np.array_equal(got["ids"], want["ids"])


@pytest.mark.parametrize("dt", DT)
def test_module_between_the_calls(pn, rng, dt):
    """What a caller does to the returned entropy and to the module's temperature between forward and
    backward does not reach the gradient."""
    T = pn.Tensor
    x, tokens = _rows(rng, 600, dt, 0.8)
    g, e = T.from_numpy(rng.normal(0, 1, 14).astype(dt)), T.from_numpy(rng.normal(0, 1, 14).astype(dt))
    m = pn.TokenLogProbs(temperature=0.8)
    m(T.from_numpy(x), tokens)
    want = m.backward(g, e).numpy()
    o = m(T.from_numpy(x), tokens)
    o.entropy.fill(7.0)
    o.logprob.fill(7.0)
    m.temperature = 3.0
    same_bits(m.backward(g, e).numpy(), want)


def _four(pn, x, tokens, temperature):
    """lse of four values per row, alone."""
    import torch
    T = pn.Tensor
    X, tok = T.from_numpy(x), torch.from_numpy(tokens).cuda()
    saved = T.create([x.shape[0], 4], X.dtype)
    torch.cuda.synchronize()
    assert pn.core._lib.neural_token_logprobs_forward(None, None, saved._ptr, None, None, 0, X._ptr, tok.data_ptr(),
                                                      temperature) == 0
    return saved.numpy()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [3, 300, 2000, 4096, 5003, 40001])
@pytest.mark.parametrize("temperature", [1e-10, 1e-4, 0.01, 1.0, 1e10])
def test_four_saved_values(pn, rng, dt, V, temperature):
    """What they hold; the gradient from them, with the bits that one value gives where |lse| < 64."""
    x, tokens = _rows(rng, V, dt, temperature)
    got = _forward(pn, x, tokens, 0, temperature)
    four = _four(pn, x, tokens, temperature)
    same_bits(four[:, 0], got["lse"])
    same_bits(four[:, 3], got["entropy"])
    used = tokens >= 0
    top = x.max(1)
    masked = np.isneginf(top)
    assert np.array_equal(four[used, 1], np.where(masked, dt(0), top)[used]) and not four[~used].any()
    assert np.isneginf(four[masked & used, 2]).all() and np.isfinite(four[~masked, 2]).all()
    g, e = rng.normal(0, 1, 14).astype(dt), rng.normal(0, 1, 14).astype(dt)
    near = np.abs(got["lse"]) < 64
    for a, b in ((g, None), (None, e), (g, e)):
        one = _backward(pn, x, tokens, a, b, got["lse"], got["entropy"], temperature)
        dx = _backward(pn, x, tokens, a, b, four, None, temperature)
        same_bits(dx[near], one[near])
        want, bound = _grad_of_logits(x, tokens, a, b, temperature, True)
        within(dx, want, bound, "dx")


def test_four_saved_values_refused(pn):
    """Counts other than one and four a row, and no entropy beside one."""
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    x, dx, g, tok = T.zeros([3, 9]), T.zeros([3, 9]), T.zeros([3]), np.zeros(3, np.int64)
    forward, backward = lib.neural_token_logprobs_forward, lib.neural_token_logprobs_backward
    for n in (0, 1, 6, 9, 13):
        s = T.create([n])
        assert forward(None, None, s._ptr, None, None, 0, x._ptr, tok.ctypes.data, 1.0) == E.SHAPE_MISMATCH
        assert backward(dx._ptr, g._ptr, None, x._ptr, tok.ctypes.data, s._ptr, None, 1.0) == E.SHAPE_MISMATCH
    one, four, five = T.zeros([3]), T.zeros([3, 4]), T.zeros([5])
    assert backward(dx._ptr, g._ptr, g._ptr, x._ptr, tok.ctypes.data, one._ptr, None, 1.0) == E.NULL_POINTER
    assert backward(dx._ptr, g._ptr, g._ptr, x._ptr, tok.ctypes.data, four._ptr, five._ptr, 1.0) == E.SHAPE_MISMATCH
    assert forward(None, four._ptr, None, None, None, 0, x._ptr, tok.ctypes.data, 1.0) == E.SHAPE_MISMATCH
    assert forward(None, None, x._ptr, None, None, 0, x._ptr, tok.ctypes.data, 1.0) == E.SHAPE_MISMATCH
    for v in (four, dx, g):
        assert not v.numpy().any()
    assert forward(None, None, four._ptr, None, None, 0, x._ptr, tok.ctypes.data, 1.0) == E.OK
    assert backward(dx._ptr, g._ptr, g._ptr, x._ptr, tok.ctypes.data, four._ptr, None, 1.0) == E.OK


@pytest.mark.parametrize("four", [False, True])
def test_graph_at_a_low_temperature(pn, rng, four):
    """Forward and gradient captured, replayed over changed logits and tokens, eager calls in between."""
    import torch
    rows, V, temperature, lib, T = 14, 5003, 0.01, pn.core._lib, pn.Tensor
    t = {"x": torch.zeros(rows, V, device="cuda"), "dx": torch.zeros(rows, V, device="cuda"),
         "lse": torch.zeros(rows, 4 if four else 1, device="cuda"),
         **{n: torch.zeros(rows, device="cuda") for n in ("entropy", "g", "e")}}
    tok = torch.zeros(rows, dtype=torch.int64, device="cuda")
    w = {n: T.from_torch(v) for n, v in t.items()}
    P = lambda n: w[n]._ptr  # noqa: E731
    stream = torch.cuda.Stream()
    pn.set_stream(stream.cuda_stream)
    try:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert lib.neural_token_logprobs_forward(None, P("entropy"), P("lse"), None, None, 0, P("x"), tok.data_ptr(),
                                                     temperature) == 0
            assert lib.neural_token_logprobs_backward(P("dx"), P("g"), P("e"), P("x"), tok.data_ptr(), P("lse"),
                                                      None if four else P("entropy"), temperature) == 0
        for _ in range(3):
            x, tokens = _rows(rng, V, np.float32, temperature)
            x[::4] *= np.float32(0.01)
            g, e = rng.normal(0, 1, rows).astype(np.float32), rng.normal(0, 1, rows).astype(np.float32)
            for n, v in (("x", x), ("g", g), ("e", e)):
                t[n].copy_(torch.from_numpy(v))
            tok.copy_(torch.from_numpy(tokens))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            saved = _four(pn, x, tokens, temperature)
            want = _backward(pn, x, tokens, g, e, saved if four else saved[:, 0].copy(),
                             None if four else saved[:, 3].copy(), temperature)
            same_bits(t["dx"].cpu().numpy(), want)
    finally:
        pn.set_stream(None)
