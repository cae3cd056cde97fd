"""The torch references of the 4-bit operators and the router against the numpy ones, on the CPU."""
import numpy as np
import pytest
import torch

import mx4_gpu_ref as M
import mx4_ref as R


@pytest.mark.parametrize("T,E,k,align,renorm", [(50, 7, 3, 4, True), (40, 20, 5, 1, False), (9, 4, 4, 8, True), (30, 3, 1, 32, False)])
def test_route(T, E, k, align, renorm):
    rng = np.random.default_rng(T)
    x = np.round(rng.standard_normal((T, E)) * 8) / 4           # ties
    x[rng.random((T, E)) < 0.3] = -np.inf
    mask = (rng.random(T) < 0.8).astype(np.uint8)
    a, b = R.route(x, mask, k, align, renorm, 0.3), M.route(torch.from_numpy(x), torch.from_numpy(mask), k, align, renorm, 0.3)
    for n in ("ids", "counts", "offsets", "pos", "order", "on"):
        assert np.array_equal(a[n], b[n].numpy()), n
    for n in ("gates", "probs", "p"):
        assert np.allclose(a[n], b[n].numpy(), rtol=1e-13, atol=0), n
    assert a["used"] == b["used"] and np.isclose(a["loss"], b["loss"], rtol=1e-13, atol=0)
    dg = rng.standard_normal((T, k))
    for got, want in zip(M.route_gradient(b, k, renorm, 0.3, torch.from_numpy(dg), 1.7), R.route_gradient(a, k, renorm, 0.3, dg, 1.7)):
        assert np.allclose(got.numpy(), want, rtol=1e-12, atol=1e-15)


def test_quantise_and_values():
    rng = np.random.default_rng(1)
    x = np.round(rng.standard_normal((20, 77)) * np.exp(3 * rng.standard_normal((20, 1))) * 8) / 8      # ties
    x[3], x[4, :32] = 0.0, -0.0
    code, s = R.quantise(x)
    codes, scales = M.quantise(torch.from_numpy(x))
    assert np.array_equal(R.pack(code), codes.numpy()) and np.array_equal(s, scales.numpy())
    scales[5, 1] = 255
    assert np.array_equal(R.values(codes.numpy(), scales.numpy())[:, :77], M.values(codes, scales, 77).numpy(), equal_nan=True)
