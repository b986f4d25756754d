"""RMS norm to 8 bits with eps = 0: a row of zeros, whose rstd is infinite, has codes and scale 0."""

import numpy as np
import pytest

import serving_ref as ref
from conftest import GPU, same_bits

pytestmark = GPU


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("cols", [1, 24, 300, 2050, 20000, 70001])
@pytest.mark.parametrize("add", [False, True])
def test_codes_of_zeros(pn, rng, dt, cols, add):
    import torch
    T, lib = pn.Tensor, pn.core._lib
    x = rng.normal(0, 1, (9, cols)).astype(dt)
    gamma = rng.normal(1, 0.2, cols).astype(dt)
    x[1] = 0.0
    x[4] = -0.0
    x[5, cols - 1] = np.nan
    x[6] = np.inf
    x[7] = 0.0
    x[7, 0] = np.inf
    half = rng.integers(-4, 5, x.shape).astype(dt)
    half[1] = 0.0
    a, b = (x - half, half) if add else (x, None)
    if add:
        x = (b + a).astype(dt)
        assert not x[1].any()
    for g in (gamma, None):
        X, R, G = (T.from_numpy(v) if v is not None else None for v in (a, b, g))
        H = T.create(x.shape, X.dtype) if add else None
        scale, codes = T.create([9], X.dtype), torch.full((9, cols), 9, dtype=torch.int8, device="cuda")
        torch.cuda.synchronize()
        P = lambda t: t._ptr if t is not None else None  # noqa: E731
        assert lib.neural_rms_norm_forward_q8(codes.data_ptr(), cols, scale._ptr, P(H), X._ptr, P(R), P(G), 0.0) == 0
        pn.synchronize()
        s, c = scale.numpy(), codes.cpu().numpy()
        assert not s[[1, 4]].any() and not np.signbit(s[[1, 4]]).any() and not c[[1, 4]].any()
        assert np.isnan(s[5:8]).all() and not c[5:8].any()
        w = x.astype(np.float64) * (1.0 if g is None else g.astype(np.float64))
        live = [0, 2, 3, 8]
        assert np.array_equal(c[live], ref.codes(w[live])[0])
        assert np.isfinite(s[live]).all() and (s[live] > 0).all()
        if not add:  # the product of such a row is the bias
            W, sw = torch.ones(5, cols, dtype=torch.int8, device="cuda"), T.ones([5], X.dtype)
            bias, out = T.from_numpy(np.arange(5).astype(dt)), T.create([9, 5], X.dtype)
            torch.cuda.synchronize()
            assert lib.neural_linear_q8(out._ptr, codes.data_ptr(), cols, scale._ptr, W.data_ptr(), cols, sw._ptr, cols,
                                        bias._ptr, 0, 0.0, None) == 0
            same_bits(out.numpy()[1], np.arange(5).astype(dt))
