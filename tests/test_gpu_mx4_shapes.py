"""Grouped 4-bit products at sizes that take each of the kernel's tile shapes, split inner dimensions and long group
lists, against 64-bit products on the GPU."""
import numpy as np
import pytest
import torch

import ggemm as G
import mx4_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def _operand(rng, rows, cols):
    """Random codes and scales (the last block filled up with zeros): torch bytes and float64 values, on the GPU."""
    nb = R.up(max(cols, 1), 32) // 32
    codes = torch.from_numpy(rng.integers(0, 256, (rows, 16 * nb), dtype=np.uint8)).cuda()
    if cols % 32:
        keep = torch.arange(32 * nb, device="cuda") < cols
        codes &= (keep[0::2].to(torch.uint8) * 15) | (keep[1::2].to(torch.uint8) * 240)
    scales = torch.full((rows, R.up(nb, 4)), 255, dtype=torch.uint8, device="cuda")
    scales[:, :nb] = torch.from_numpy(rng.integers(123, 132, (rows, nb), dtype=np.uint8)).cuda()
    grid = torch.tensor(list(R.GRID) + [-v for v in R.GRID], dtype=torch.float64, device="cuda")
    nib = torch.stack((codes & 15, codes >> 4), -1).view(rows, nb, 32).int()
    scale = ((scales[:, :nb].long() + 896) << 52).view(torch.float64)    # 2^(s - 127) from its bits
    return (codes, scales), (grid[nib] * scale[..., None]).view(rows, -1)[:, :cols].contiguous()


def _check(got, want, mass, k, dtype, what):
    tol = (k + 4) * 2.0 ** -23 * mass + 2 * R.UNIT[dtype] * want.abs() + R.TINY[dtype]
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (what, int((err > tol).sum()), float((err / tol).max()))


def _split(rng, total, groups, step=1):
    cut = np.sort(rng.integers(0, total // step + 1, groups - 1)) if groups > 1 else np.array([], dtype=np.int64)
    return np.concatenate([[0], cut, [total // step]]) * step


ROWS = [  # m, n, k, groups
    (5000, 6000, 300, 1), (5000, 6001, 96, 7), (9000, 4100, 544, 3),        # 256 x 256 tiles
    (3000, 900, 1100, 5), (20000, 130, 64, 200), (2000, 515, 288, 9),       # 128 x 128
    (5000, 1030, 200, 100), (700, 4100, 320, 30), (4000, 257, 32, 500),     # 32 x 128
    (3, 200, 5000, 1), (16, 40, 16384, 1), (5, 77, 8200, 4), (4, 300, 512, 900),   # 16 x 32
    (17, 130, 16384, 1), (64, 1024, 8192, 2), (300, 260, 20000, 1),         # parts of the inner dimension
]


@pytest.mark.parametrize("m,n,k,groups", ROWS)
def test_rows(m, n, k, groups):
    rng = np.random.default_rng(m + 3 * n + 7 * k)
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, groups * n, k)
    off = _split(rng, m, groups)
    offs = R.dev(off.astype(np.int32))
    want, mass = torch.zeros(m, n, dtype=torch.float64, device="cuda"), torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for g in range(groups):
        lo, hi = int(off[g]), int(off[g + 1])
        if lo < hi:
            w = bv[g * n:(g + 1) * n].t().contiguous()
            want[lo:hi], mass[lo:hi] = av[lo:hi] @ w, av[lo:hi].abs() @ w.abs()
    for dtype in ("f32", "bf16"):
        for pad in (0, 3):
            say(f"rows {m} {n} {k} {groups} {dtype} {pad}")
            out = torch.full((m, n + pad), 5.0, dtype=R.TORCH[dtype], device="cuda")
            R.gemm(G.MX4_ROWS, a, b, m, n, k, out, offs, groups, b_strides=(n * b[0].shape[1], n * b[1].shape[1]), ldc=n + pad)
            _check(out[:, :n], want, mass, k, dtype, (m, n, k, groups, dtype, pad))
            assert bool((out[:, n:] == 5.0).all())
    c0 = torch.randn(m, n, device="cuda")
    out = c0.clone()
    R.gemm(G.MX4_ROWS, a, b, m, n, k, out, offs, groups, alpha=0.5, beta=-2.0, b_strides=(n * b[0].shape[1], n * b[1].shape[1]))
    _check(out, 0.5 * want - 2.0 * c0.double(), 0.5 * mass + 2.0 * c0.double().abs(), k, "f32", ("beta", m, n, k, groups))


INNER = [  # m, n, total k, groups
    (4100, 3000, 3200, 3), (2048, 4096, 4000, 4),            # 256 x 256
    (1000, 700, 5000, 6), (129, 4000, 2080, 2),              # 128 x 128
    (20, 500, 3000, 5), (64, 64, 2000, 70),                  # 32 x 128
    (7, 90, 4100, 3), (16, 33, 640, 1),                      # 16 x 32
    (128, 128, 30000, 1), (1000, 130, 20000, 2), (40, 60, 40000, 3),   # parts of the inner dimension
]


@pytest.mark.parametrize("m,n,k,groups", INNER)
def test_inner(m, n, k, groups):
    rng = np.random.default_rng(m + 5 * n + 11 * k)
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, n, k)
    off = _split(rng, k, groups, 32)
    off[-1] = k                      # the last group may end inside a block
    want, mass = (torch.zeros(groups, m, n, dtype=torch.float64, device="cuda") for _ in range(2))
    for g in range(groups):
        s = slice(int(off[g]), int(off[g + 1]))
        w = bv[:, s].t().contiguous()
        want[g], mass[g] = av[:, s] @ w, av[:, s].abs() @ w.abs()
    for dtype, pad in (("f32", 0), ("bf16", 0), ("f32", 1)):
        say(f"inner {m} {n} {k} {groups} {dtype} {pad}")
        out = torch.full((groups, m, n + pad), 5.0, dtype=R.TORCH[dtype], device="cuda")
        R.gemm(G.MX4_INNER, a, b, m, n, k, out, R.dev(off.astype(np.int32)), groups, ldc=n + pad, c_stride=m * (n + pad))
        _check(out[..., :n], want, mass, k, dtype, (m, n, k, groups, dtype, pad))
        assert bool((out[..., n:] == 5.0).all())


def test_same_bits_every_time():
    say("same bits")
    rng = np.random.default_rng(1)
    for m, n, k, groups in ((5000, 6000, 300, 4), (300, 260, 20000, 1), (16, 40, 16384, 1), (700, 4100, 320, 30)):
        a, _ = _operand(rng, m, k)
        b, _ = _operand(rng, groups * n, k)
        offs = R.dev(_split(rng, m, groups).astype(np.int32))
        runs = [R.gemm(G.MX4_ROWS, a, b, m, n, k, torch.zeros(m, n, device="cuda"), offs, groups,
                       b_strides=(n * b[0].shape[1], n * b[1].shape[1])) for _ in range(3)]
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2]), (m, n, k, groups)


def test_long_rows():
    """Leading dimensions of more than 2^23 bytes: offsets past 32 bits from the first row on."""
    say("long rows")
    rng = np.random.default_rng(2)
    k, m, n, ld = 500, 300, 40, 2 ** 24 + 16
    buf = torch.zeros(m * ld, dtype=torch.uint8, device="cuda")
    a, av = _operand(rng, m, k)
    b, bv = _operand(rng, n, k)
    wide = buf.view(m, ld)
    wide[:, :a[0].shape[1]] = a[0]
    out = torch.zeros(m, n, device="cuda")
    R.gemm(G.MX4_ROWS, (wide, a[1]), b, m, n, k, out)
    w = bv.t().contiguous()
    _check(out, av @ w, av.abs() @ w.abs(), k, "f32", "long rows")


def test_inner_order_of_groups():
    """More than two runs of 64 groups of different lengths, empty ones among them."""
    test_inner(130, 200, 6400, 150)
    test_inner(300, 260, 3200, 64)
