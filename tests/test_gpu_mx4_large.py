"""The 4-bit operators on calls large enough for the paths that small ones do not take, and on empty ones; exact against
references on the GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
import mx4_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_layer_without_tokens(dtype):
    """No tokens: the router's order holds padding only, the matrix that it picks rows from has none (and no address)."""
    say(f"no tokens {dtype}")
    E, d, f, align = 5, 200, 96, 32
    rows = E * (align - 1)
    _, o, _ = R.gpu_route(torch.zeros(0, E, device="cuda"), None, 2, align, True, 0.5)
    x = torch.zeros(0, d, dtype=R.TORCH[dtype], device="cuda")
    assert x.data_ptr() == 0 and o["order"].shape[0] == rows
    c, s, ct, st = R.gpu_quantise(x, index=o["order"], down=True)
    nb, nr = R.up(d, 32) // 32, R.up(rows, 32) // 32
    assert (c == 0).all() and (s[:, :nb] == 0).all() and (ct == 0).all() and (st[:, :nr] == 0).all()
    a, at = (R.dev(c), R.dev(s)), (R.dev(ct), R.dev(st))
    w = torch.full((E * f, 16 * nb), 0x22, dtype=torch.uint8, device="cuda"), torch.full((E * f, R.up(nb, 4)), 127, dtype=torch.uint8, device="cuda")
    out = R.gemm(G.MX4_ROWS, a, w, rows, f, d, torch.full((rows, f), 5.0, device="cuda"), o["offsets"], E,
                 b_strides=(f * w[0].shape[1], f * w[1].shape[1]))
    assert bool((out == 5.0).all())
    out = R.gemm(G.MX4_INNER, at, at, d, d, rows, torch.full((E, d, d), 5.0, device="cuda"), o["offsets"], E, c_stride=d * d)
    assert bool((out == 0.0).all())
