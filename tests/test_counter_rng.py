"""The tests' own Philox4x32-10 and the draws made from it, without a GPU: the
generator's published known answers, the layout of the draws, and the modules' own argument
checks."""

import numpy as np
import pytest

import sublayer_ref as ref


@pytest.mark.parametrize("counter,key,want", [
    # known answers that the generator's authors publish with it
    ((0, 0), 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((2 ** 64 - 1, 2 ** 64 - 1), 2 ** 64 - 1, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x85A308D3243F6A88, 0x0370734413198A2E), 0x299F31D0A4093822, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_known_answers(counter, key, want):
    got = ref.philox(np.array([counter[0]], dtype=np.uint64), counter[1], key)[0]
    assert tuple(int(v) for v in got) == want


def test_draws_layout():
    """Element 13 is place 5 of group 1: the upper half of word 2 of blocks 2 and 3."""
    seed, offset = 0x123456789ABCDEF0, 77
    hi = int(ref.philox(np.array([2], dtype=np.uint64), offset, seed)[0][2]) >> 16
    lo = int(ref.philox(np.array([3], dtype=np.uint64), offset, seed)[0][2]) >> 16
    assert int(ref.draws(13, 1, seed, offset)[0]) == hi << 16 | lo
    assert np.array_equal(ref.draws(13, 40, seed, offset), ref.draws(0, 64, seed, offset)[13:53])


def test_keep_rate():
    n = 1 << 20
    for p in (0.0, 0.1, 0.5, 1.0):
        k = ref.keep(n, p, 5, 9).mean()
        assert abs(k - (1 - p)) <= 6 * np.sqrt(p * (1 - p) / n)  # six standard deviations


def test_bounds_catch_a_wrong_result():
    """The forms' bounds let a double computation pass and a float one, or a
    variance over C - 1, fail."""
    rng = np.random.default_rng(0)
    x = rng.normal(3, 1, (5, 100))
    (y, mean, rstd), (by, bm, br) = ref.norm(x, None, None, 1e-5)
    d = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((d * d).mean(-1) + 1e-5)
    ref.within(d * r[:, None], y, by)
    ref.within(r, rstd, br)
    with pytest.raises(AssertionError):
        ref.within((d * r[:, None]).astype(np.float32).astype(np.float64), y, by)
    with pytest.raises(AssertionError):
        ref.within(1 / np.sqrt(x.var(-1, ddof=1) + 1e-5), rstd, br)


def test_module_arguments():
    import pyneural as pn
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            pn.CounterDropout(p)
    with pytest.raises(ValueError):
        pn.LayerNorm(0)
    with pytest.raises(RuntimeError):
        pn.CounterDropout(0.5).backward(None)


def test_refused_without_a_gpu():
    """Without a device the entry points return the initialisation's error and
    touch nothing, whatever the arguments (in a child process: with a GPU they
    report the null pointers)."""
    import ctypes
    import subprocess
    import sys
    from pathlib import Path
    lib = Path(__file__).resolve().parent.parent / "neural-assembly_amd" / "libneural_hip.so"
    code = ("import ctypes,sys; l=ctypes.CDLL(sys.argv[1]); v=ctypes.c_void_p; d=ctypes.c_double\n"
            "def f(n,*a):\n"
            "    f=getattr(l,n); f.argtypes=list(a); return f(*[0.5 if t is d else None for t in a])\n"
            "print(f('neural_counter_dropout_forward',v,v,d,v), f('neural_counter_dropout_backward',v,v,d,v),"
            " f('neural_layer_norm_forward',v,v,v,v,d,v,v), f('neural_layer_norm_backward',*[v]*8),"
            " f('neural_dropout_add_layer_norm_forward',*[v]*6,d,v,d,v,v),"
            " f('neural_dropout_add_layer_norm_backward',*[v]*10,d,v))")
    out = subprocess.run([sys.executable, "-c", code, str(lib)], capture_output=True, text=True, timeout=120)
    rcs = [int(v) for v in out.stdout.split()[-6:]]
    assert rcs in ([15] * 6, [1] * 6), (out.stdout, out.stderr)
    assert ctypes.sizeof(ctypes.c_void_p) == 8
