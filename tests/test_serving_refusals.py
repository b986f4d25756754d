"""What the norm to 8 bits, the 8-bit product and the token log probabilities refuse before
they reach a device: without one, the initialisation's error whatever the arguments, and
the modules' own checks."""

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

LIB = Path(__file__).resolve().parent.parent / "neural-assembly_amd" / "libneural_hip.so"


def test_refused_without_a_gpu():
    """In a child process: with a GPU the null pointers are reported."""
    code = ("import ctypes,sys; l=ctypes.CDLL(sys.argv[1]); v=ctypes.c_void_p; d=ctypes.c_double; i=ctypes.c_int64\n"
            "c=ctypes.c_int; give={d: 0.5, i: 1, c: 0, v: None}\n"
            "def f(n,*a):\n"
            "    f=getattr(l,n); f.argtypes=list(a); return f(*[give[t] for t in a])\n"
            "print(f('neural_rms_norm_forward',*[v]*5,d,v), f('neural_rms_norm_backward',*[v]*7),"
            " f('neural_rms_norm_forward_q8',v,i,*[v]*5,d), f('neural_quantize_rows',v,i,v,v),"
            " f('neural_linear_q8',v,v,i,v,v,i,v,i,v,c,d,v),"
            " f('neural_token_logprobs_forward',*[v]*5,i,v,v,d), f('neural_token_logprobs_backward',*[v]*7,d))")
    out = subprocess.run([sys.executable, "-c", code, str(LIB)], capture_output=True, text=True, timeout=120)
    rcs = [int(v) for v in out.stdout.split()[-7:]]
    assert rcs in ([15] * 7, [1] * 7), (out.stdout, out.stderr)


def test_module_arguments():
    import pyneural as pn
    from pyneural import nn
    with pytest.raises(ValueError):
        pn.RMSNorm(0)
    for bad in (0.0, -1.0, 9e-11, 1.1e10, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            pn.TokenLogProbs(temperature=bad)
    for k in (-1, 65):
        with pytest.raises(ValueError):
            pn.TokenLogProbs(top_k=k)
    with pytest.raises(RuntimeError):
        pn.TokenLogProbs().backward()
    for bad in (np.zeros(3), np.zeros(2, np.int64), [1, 2], ["a", "b", "c"]):
        with pytest.raises(ValueError):
            nn._int64_rows(bad, 3)
    assert nn._int64_rows(None, 3) == (None, None)
    held, at = nn._int64_rows(np.array([1, -1, 5], np.int32), 3)
    assert held.dtype == np.int64 and at == held.ctypes.data and held.tolist() == [1, -1, 5]
    import torch
    with pytest.raises(ValueError):
        nn._int64_rows(torch.zeros(3, dtype=torch.int32), 3)
    with pytest.raises(ValueError):
        nn._int64_rows(torch.zeros(4, dtype=torch.int64), 3)
    step = torch.arange(6)[::2]
    held, at = nn._int64_rows(step, 3)
    assert held.tolist() == [0, 2, 4] and at == held.data_ptr()
