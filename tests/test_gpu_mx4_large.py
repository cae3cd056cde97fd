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


def test_older_error_is_not_the_calls():
    """An error that an earlier call of the program left behind (here: a device that does not exist) is not reported as a
    failed launch."""
    say("older error")
    hip = C.CDLL("libamdhip64.so")
    x = torch.randn(70, 96, device="cuda")
    y = torch.zeros(70, 96, device="cuda")
    c, s = torch.zeros(70, 48, dtype=torch.uint8, device="cuda"), torch.zeros(70, 4, dtype=torch.uint8, device="cuda")
    out = torch.zeros(70, 70, device="cuda")
    q = G.Mx4Quant(70, 96, G.F32, 70, x.data_ptr(), 96, None, c.data_ptr(), 48, s.data_ptr(), 4, None, 0, None, 0)
    d = G.Mx4Dequant(70, 96, G.F32, c.data_ptr(), 48, s.data_ptr(), 4, y.data_ptr(), 96)
    p = G.Mx4Gemm(G.MX4_ROWS, 1, 70, 70, 96, G.F32, 1.0, 0.0, c.data_ptr(), 48, s.data_ptr(), 4, c.data_ptr(), 48, 0,
                  s.data_ptr(), 4, 0, None, out.data_ptr(), 70, 0)
    ws = torch.zeros(max(16, G.lib().ggemm_mx4_gemm_workspace(C.byref(p))), dtype=torch.uint8, device="cuda")
    r, o, rws = R.gpu_route(x, None, 2, 1, True, 0.1)
    dx = torch.zeros(70, 96, device="cuda")
    calls = {"quantize": lambda: G.lib().ggemm_mx4_quantize(C.byref(q), R.stream()),
             "dequantize": lambda: G.lib().ggemm_mx4_dequantize(C.byref(d), R.stream()),
             "gemm": lambda: G.lib().ggemm_mx4_gemm(C.byref(p), ws.data_ptr(), ws.numel(), R.stream()),
             "route": lambda: G.lib().ggemm_route(C.byref(r), rws.data_ptr(), rws.numel(), R.stream()),
             "route_backward": lambda: G.lib().ggemm_route_backward(C.byref(r), None, None, dx.data_ptr(), 96, R.stream())}
    torch.cuda.synchronize()
    rc = {}
    for name, call in calls.items():
        assert hip.hipSetDevice(9999) != 0
        rc[name] = call()
        hip.hipGetLastError()
    torch.cuda.synchronize()
    assert rc == {name: G.GGEMM_OK for name in calls}
    assert bool(((y - x).abs() <= 0.5 * x.abs().amax(1, keepdim=True)).all()) and bool(out.any())


@pytest.mark.parametrize("m", [3, 100, 9000])
def test_products_of_subnormal_size(m):
    """A single product of 1.5 2^e, and two that leave 2^(e - 1), down to e = -152: exact where a 32-bit number holds it
    (multiples of 2^-149), rounded there below."""
    say(f"subnormal products {m}")
    n, k = 64, 64
    e = np.arange(-152, -152 + n)
    ac = torch.zeros(m, 32, dtype=torch.uint8, device="cuda")
    asc = torch.full((m, 4), 127 - 60, dtype=torch.uint8, device="cuda")
    bsc = R.dev(np.repeat((e + 60 + 127).astype(np.uint8)[:, None], 4, 1))
    for a0, b0, want in ((0x02, 0x03, np.ldexp(1.5, e)), (0x22, 0xA3, np.ldexp(0.5, e))):      # 1, 1.5;  1 1, 1.5 -1
        ac[:, 0] = a0
        bc = torch.zeros(n, 32, dtype=torch.uint8, device="cuda")
        bc[:, 0] = b0
        out = R.gemm(G.MX4_ROWS, (ac, asc), (bc, bsc), m, n, k, torch.zeros(m, n, device="cuda"))
        got = out.double().cpu().numpy()
        held = np.ldexp(np.round(np.ldexp(want, 149)), -149) == want
        assert (got[:, held] == want[held]).all() and held.sum() >= 60
        assert (np.abs(got - want) <= 2.0 ** -149).all()
