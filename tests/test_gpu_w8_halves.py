"""Row quantisation next to halves (include/ggemm_w8.h) where 32-bit numbers run out of bits: 32-bit rows whose scale lies just
above the least one, and every 16-bit row maximum with every value below it; bit for bit."""
import numpy as np
import pytest
import torch

import glu_ref as R
from gpu_util import say
from test_gpu_w8 import quantise, same

pytestmark = pytest.mark.gpu


def rows_at_halves(rng, n, low, high):
    """Rows with maxima of low .. high and, for each half up to 126.5 of their scale, the value there and its neighbours."""
    rows = []
    for _ in range(n):
        top = np.float32(rng.uniform(low, high))
        s = np.float64(np.maximum(np.float32(np.float64(top) / 127), np.float32(2.0 ** -126)))
        h = ((np.arange(0, 127) + 0.5) * s).astype(np.float32)
        h = np.concatenate([h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(0))])
        rows.append(np.concatenate([[top], np.minimum(h, top) * rng.choice([-1, 1], h.shape).astype(np.float32)]))
    return torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()


@pytest.mark.parametrize("low,high", [(127 * 2.0 ** -126, 127 * 2.0 ** -125), (127 * 2.0 ** -125, 127 * 2.0 ** -123), (100 * 2.0 ** -126, 130 * 2.0 ** -126),
                                      (2.0 ** 127, 3.4028234e38)])
def test_halves_of_32_bit_rows(low, high):
    say("halves between", low, high)
    x = rows_at_halves(np.random.default_rng(1), 4000, low, high)
    same(quantise(x), R.quantise64(x))


def test_a_half_below_the_least_normal_number():
    """x / s = 35.499999957 with s = 0x1.64dc6ep-126: 35."""
    say("one half")
    x = torch.tensor([[float.fromhex("0x1.6212b6p-119"), float.fromhex("0x1.8be48ap-121")]], device="cuda")
    assert quantise(x)[0].tolist() == [[127, 35]]


def test_half_of_a_small_bf16_maximum():
    """a = 222 2^-126, x = a / 2: x / s = 63.499999966, 63."""
    say("bf16 half")
    x = torch.tensor([[222 * 2.0 ** -126, 111 * 2.0 ** -126]], device="cuda").bfloat16()
    assert quantise(x)[0].tolist() == [[127, 63]]


@pytest.mark.parametrize("dtype,top", [("bf16", 0x7f80), ("f16", 0x7c00)])
def test_every_16_bit_maximum_with_every_value(dtype, top):
    """Rows: every positive finite maximum; columns: every value up to it (the maximum itself instead of larger ones)."""
    say("every", dtype)
    every = torch.arange(0, top, dtype=torch.int16, device="cuda")
    for i in range(1, top, 1024):
        a = torch.arange(i, min(i + 1024, top), dtype=torch.int16, device="cuda")
        x = torch.minimum(every[None], a[:, None]).view(R.TORCH[dtype])      # positive values order as their bits
        same(quantise(x), R.quantise64(x))
