"""Counter-based dropout (neural_counter_dropout_forward / _backward): every
element equal, bit for bit, to the one product or +0 that its draw calls for
(tests/sublayer_ref.py), at sizes around the groups of 8, the vectors and the
blocks, at any alignment, p from 0 to 1, in both dtypes; keys in host and device
memory, captured graphs, element counts past 2^32, and the refusals."""

import ctypes

import numpy as np
import pytest

import sublayer_ref as ref
from conftest import GPU, same_bits

pytestmark = GPU

DT = [np.float32, np.float64]


def _key(pn, seed, offset):
    return ctypes.byref(pn.core.DropoutKeyC(seed, offset))


def _run(pn, x, p, seed, offset, fn="neural_counter_dropout_forward"):
    t = pn.Tensor.from_numpy(x)
    out = pn.Tensor.create(x.shape, t.dtype)
    assert getattr(pn.core._lib, fn)(out._ptr, t._ptr, p, _key(pn, seed, offset)) == 0
    return out.numpy()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 255, 256, 257, 1023, 2047, 2048, 2049, 4099,
                               100003])
def test_sizes(pn, rng, dt, n):
    x = rng.normal(0, 2, n).astype(dt)
    same_bits(_run(pn, x, 0.3, 11, 22), ref.dropout(x, 0.3, 11, 22))


@pytest.mark.parametrize("dt", DT)
# exact multiples of 2^-16 need no lower halves; 2^-20 and 1 - 2^-20 decide by them alone; 1e-12 rounds to 0
@pytest.mark.parametrize("p", [0.0, 1e-12, 2.0 ** -20, 0.1, 0.25, 0.5, 0.9, 1 - 2.0 ** -16, 1 - 2.0 ** -20, 1 - 2.0 ** -40, 1.0])
def test_probabilities(pn, rng, dt, p):
    x = rng.normal(0, 2, 1 << 19).astype(dt)
    x[::7] = -0.0
    same_bits(_run(pn, x, p, 3, 4), ref.dropout(x, p, 3, 4))


def test_lower_halves_decide(pn):
    """Elements whose upper 16 bits equal the threshold's: kept and dropped ones
    among them, as their lower halves say."""
    n, p, seed, offset = 1 << 21, 0.1, 8, 9
    r = ref.draws(0, n, seed, offset)
    thr = round(p * 2 ** 32)
    tie = (r >> np.uint64(16)) == thr >> 16
    assert (r[tie] >= thr).any() and (r[tie] < thr).any()  # about 32 of them
    got = _run(pn, np.ones(n, np.float32), p, seed, offset)
    assert np.array_equal(got != 0, r >= thr)


@pytest.mark.parametrize("key", [(0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (1 << 32, 0), (0, 1 << 32), (0x0123456789ABCDEF, 5)])
def test_keys(pn, key):
    x = np.ones(5000, np.float32)
    same_bits(_run(pn, x, 0.5, *key), ref.dropout(x, 0.5, *key))


def test_backward_takes_the_forward_mask(pn, rng):
    x = rng.normal(0, 1, (37, 53)).astype(np.float32) + 10  # no zeros
    y = _run(pn, x, 0.4, 1, 2)
    g = rng.normal(0, 1, x.shape).astype(np.float32)
    gi = _run(pn, g, 0.4, 1, 2, "neural_counter_dropout_backward")
    same_bits(gi, np.where(y != 0, g * np.float32(1 / 0.6), np.float32(0)))


def test_dropped_values_do_not_matter(pn):
    """NaN and infinities: +0 where dropped, themselves where kept."""
    for dt in DT:
        x = np.tile(np.array([np.nan, np.inf, -np.inf, 1e-45, -0.0], dt), 1000)
        same_bits(_run(pn, x, 0.5, 6, 7), ref.dropout(x, 0.5, 6, 7))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("start", [1, 2, 3, 5])
def test_alignment_guards_and_in_place(pn, rng, dt, start):
    """Buffers that start inside a vector; nothing outside them is written;
    in place gives the same."""
    import torch
    n = 3001
    base = torch.from_numpy(rng.normal(0, 1, n + 64).astype(dt)).cuda()
    out = torch.full((n + 64,), 7.0, dtype=base.dtype, device="cuda")
    x = base[start:start + n]
    o = out[start + 2:start + 2 + n]
    want = ref.dropout(x.cpu().numpy(), 0.2, 1, 1)
    lib = pn.core._lib
    T = pn.Tensor.from_torch
    tx, to = T(x), T(o)
    torch.cuda.synchronize()
    assert lib.neural_counter_dropout_forward(to._ptr, tx._ptr, 0.2, _key(pn, 1, 1)) == 0
    pn.synchronize()
    same_bits(o.cpu().numpy(), want)
    assert bool((out[:start + 2] == 7).all()) and bool((out[start + 2 + n:] == 7).all())
    before = base.clone()
    torch.cuda.synchronize()
    assert lib.neural_counter_dropout_forward(tx._ptr, tx._ptr, 0.2, _key(pn, 1, 1)) == 0
    pn.synchronize()
    same_bits(x.cpu().numpy(), want)
    assert torch.equal(base[:start], before[:start]) and torch.equal(base[start + n:], before[start + n:])


def test_host_buffers(pn, rng):
    """Tensors over host memory (zero copy)."""
    x = rng.normal(0, 1, 777).astype(np.float32)
    out = np.zeros_like(x)
    tx, to = pn.Tensor.from_numpy_zero_copy(x), pn.Tensor.from_numpy_zero_copy(out)
    assert pn.core._lib.neural_counter_dropout_forward(to._ptr, tx._ptr, 0.5, _key(pn, 2, 3)) == 0
    same_bits(out, ref.dropout(x, 0.5, 2, 3))


def test_empty(pn):
    x = pn.Tensor.create([0, 5])
    assert pn.core._lib.neural_counter_dropout_forward(x._ptr, x._ptr, 0.5, _key(pn, 0, 0)) == 0


def test_refusals(pn):
    E, lib, T = pn.NeuralError, pn.core._lib, pn.Tensor
    f = lib.neural_counter_dropout_forward
    a, b = T.zeros([4, 6]), T.zeros([4, 6])
    k = _key(pn, 0, 0)
    assert f(None, a._ptr, 0.5, k) == E.NULL_POINTER
    assert f(b._ptr, None, 0.5, k) == E.NULL_POINTER
    assert f(b._ptr, a._ptr, 0.5, None) == E.NULL_POINTER
    d, s = T.zeros([4, 6], pn.float64), T.zeros([4, 7])
    assert f(d._ptr, a._ptr, 0.5, k) == E.DTYPE_MISMATCH
    assert f(s._ptr, a._ptr, 0.5, k) == E.SHAPE_MISMATCH
    for p in (-1e-9, 1 + 1e-9, float("nan"), float("inf")):
        assert f(b._ptr, a._ptr, p, k) == E.INVALID_ARGUMENT
    buf = (ctypes.c_uint64 * 4)()
    assert f(b._ptr, a._ptr, 0.5, ctypes.addressof(buf) + 4) == E.INVALID_ARGUMENT
    import torch
    t = torch.zeros(8, 6, device="cuda")
    strided, tight = T.from_torch(t[::2]), T.from_torch(t[:4])
    assert f(strided._ptr, a._ptr, 0.5, k) == E.INVALID_ARGUMENT
    assert f(a._ptr, strided._ptr, 0.5, k) == E.INVALID_ARGUMENT
    shifted = T.from_torch(t[1:5])
    assert f(shifted._ptr, tight._ptr, 0.5, k) == E.INVALID_ARGUMENT
    assert np.array_equal(b.numpy(), np.zeros((4, 6), np.float32))


def test_device_key_and_graph_replays(pn, rng):
    """A key in device memory gives the mask of the words it holds when the
    kernel runs: a captured graph takes a new one in every replay."""
    import torch
    lib = pn.core._lib
    x = rng.normal(0, 1, 20000).astype(np.float32)
    tx = torch.from_numpy(x).cuda()
    out = torch.empty_like(tx)
    key = torch.tensor([5, 0], dtype=torch.int64, device="cuda")
    X, O = pn.Tensor.from_torch(tx), pn.Tensor.from_torch(out)
    s = torch.cuda.Stream()
    try:
        pn.set_stream(s.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert lib.neural_counter_dropout_forward(O._ptr, X._ptr, 0.3, key.data_ptr()) == 0
            key[1] += 1
        for i in range(4):
            graph.replay()
            torch.cuda.synchronize()
            same_bits(out.cpu().numpy(), ref.dropout(x, 0.3, 5, i))
            out.fill_(3.0)  # the program's own work between replays
            torch.cuda.synchronize()
            assert lib.neural_counter_dropout_forward(O._ptr, X._ptr, 0.3, _key(pn, 1, i)) == 0
            pn.synchronize()
            same_bits(out.cpu().numpy(), ref.dropout(x, 0.3, 1, i))
    finally:
        pn.set_stream(None)


def test_misaligned_device_key(pn):
    import torch
    key = torch.zeros(16, dtype=torch.uint8, device="cuda")
    a = pn.Tensor.zeros([8])
    f = pn.core._lib.neural_counter_dropout_forward
    assert f(a._ptr, a._ptr, 0.5, key.data_ptr() + 4) == pn.NeuralError.INVALID_ARGUMENT


@pytest.mark.parametrize("log2", [32, 34])
def test_many_elements(pn, log2):
    """Indexes past 2^32 elements, block numbers past 2^32 (2^34 elements)."""
    import torch
    n = (1 << log2) + 13
    if torch.cuda.mem_get_info()[0] < 4 * n + (8 << 30):
        torch.cuda.empty_cache()
        pn.core._lib.neural_hip_empty_cache()
    if torch.cuda.mem_get_info()[0] < 4 * n + (2 << 30):
        pytest.skip("not enough free device memory")
    x = torch.ones(n, dtype=torch.float32, device="cuda")
    X = pn.Tensor.from_torch(x)
    torch.cuda.synchronize()
    assert pn.core._lib.neural_counter_dropout_forward(X._ptr, X._ptr, 0.5, _key(pn, 3, 1)) == 0
    pn.synchronize()
    for first in (0, n // 2 - 5, (1 << log2) - 4096, n - 2061):
        m = 2061
        want = ref.dropout(np.ones(m, np.float32), 0.5, 3, 1, first=first)
        same_bits(x[first:first + m].cpu().numpy(), want)
    del X, x
    torch.cuda.empty_cache()


def test_module(pn, rng):
    x = rng.normal(0, 1, (33, 65)).astype(np.float32)
    m = pn.CounterDropout(0.25, seed=7, offset=40)
    t = pn.Tensor.from_numpy(x)
    for call in range(3):
        same_bits(m(t).numpy(), ref.dropout(x, 0.25, 7, 40 + call))
        same_bits(m.backward(t).numpy(), ref.dropout(x, 0.25, 7, 40 + call))
    m.eval()
    same_bits(m(t).numpy(), x)
    same_bits(m.backward(t).numpy(), x)
    assert m.offset == 43
    m.train()
    same_bits(m(t).numpy(), ref.dropout(x, 0.25, 7, 43))


def test_threads(pn, rng):
    """Calls from several host threads at once."""
    import threading
    x = rng.normal(0, 1, 40000).astype(np.float32)
    bad = []

    def work(i):
        for k in range(5):
            if not np.array_equal(_run(pn, x, 0.3, i, k), ref.dropout(x, 0.3, i, k)):
                bad.append((i, k))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad
