"""The activations (include/ggemm_glu.h) value by value in 32 bits, through a gated integer product whose sums are 1: c = act(v) 1 with v the
scale of b's row."""
import ctypes as C
import math

import pytest
import torch

import ggemm as G
import glu_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def activation(v, act):
    n = v.numel()
    one = torch.zeros(n, 16, dtype=torch.int8, device="cuda")
    one[:, 0] = 1
    ones, out = torch.ones(n, device="cuda"), torch.empty(1, n, device="cuda")
    p = G.W8Gemm(1, 1, n, 1, G.F32, G.ACTS[act], one.data_ptr(), 16, ones.data_ptr(), one.data_ptr(), one.data_ptr(), 16, 0, v.data_ptr(),
                 ones.data_ptr(), 0, None, out.data_ptr(), n)
    G.check(G.lib().ggemm_w8_gemm(C.byref(p), None, 0, torch.cuda.current_stream().cuda_stream), "ggemm_w8_gemm")
    return out[0]


def values():
    near = torch.linspace(-12, 12, 400001, dtype=torch.float64)
    far = torch.exp(torch.linspace(math.log(1e-30), math.log(1e30), 20001, dtype=torch.float64))
    return torch.cat([near, far, -far]).float().cuda()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_values(act):
    """silu, gelu_tanh: logistic(a) = 1 / (1 + exp(-a)) with an argument rounded k times (silu 1, gelu_tanh 5) is off by k |a| 2^-24 of itself
    where a < 0 and by less where a > 0; exponential, sum, reciprocal and the product with v by at most four units of 2^-23.  Below
    exp(-87) it may be 0.  gelu: the polynomial is within 1.5e-7 of the error function, half of which times |v| <= 4 is 3e-7, and the 32-bit
    roundings (seven of 2^-24 of at most 1, times |v| / 2, and those of the exponential's argument) 2e-7; past 4 the exponential
    leaves only the two roundings of 1 - p and the product."""
    say("activation", act)
    v = values()
    got, x = activation(v, act).double(), v.double()
    want = x * R.act_parts(x, act)[0]
    want = torch.where(x > 1e3, x, torch.where(x < -1e3, 0.0, want))      # where 64 bits overflow in x^3
    if act == "gelu":
        bound = 5e-7 + 2.0 ** -23 * want.abs()
    else:
        a = (x if act == "silu" else math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3)).clamp(-100, 0)
        bound = ((1 if act == "silu" else 5) * a.abs() * 2.0 ** -24 + 4 * 2.0 ** -23) * want.abs() + 1e-35
    bad = ((got - want).abs() / bound)
    say(float(bad.max()), float(v[bad.argmax()]))
    assert float(bad.max()) <= 1.0
    assert bool((got[x > 100] == x[x > 100]).all()) and bool((got[x < -200] == 0).all())


def test_zero_and_infinity():
    say("zero and infinity")
    v = torch.tensor([0.0, -0.0, float("inf"), 3.4e38, -3.4e38, float("nan")], device="cuda")
    for act in ("silu", "gelu", "gelu_tanh"):
        got = activation(v, act)
        assert got[:5].tolist()[:2] == [0.0, 0.0] and got[2] == float("inf") and got[3] == v[3] and got[4] == 0 and torch.isnan(got[5])
