"""The gated block and the integer operators (include/ggemm_glu.h, include/ggemm_w8.h) at the ends of their documented ranges: the largest
gathered x, widths of 2^22, 4096 groups, weights that groups share, millions of rows and columns."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
import glu_ref as R
from gpu_util import say
from test_gpu_glu import check_backward, check_forward, cut, kept
from test_gpu_w8 import Operands, check, quantise, same, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,ldx", [(8, 8), (20, 24), (40, G.GLU_MAX_LD)])
@pytest.mark.parametrize("rows", [12, 300, 5000])
def test_gathered_x_of_nearly_two_gib(d, ldx, rows):
    """x_rows ldx just below 2^30: rows at byte offsets up to 2^31."""
    say("2 GiB of x", d, ldx, rows)
    x_rows = (2 ** 30 - 1) // ldx
    rng = np.random.default_rng(rows)
    index = np.where(rng.random(rows) < 0.5, x_rows - 1 - rng.integers(0, 9, rows), rng.integers(0, x_rows, rows))
    index[0], index[1], index[2] = x_rows - 1, -1, x_rows
    # the reference holds the rows that are picked, and an index of its own into them
    order = np.arange(rows)
    order[[1, 2]] = -1
    b = R.Block([0, rows // 3, rows], rows, d, 24, "bf16", "silu", order, rows, seed=rows + d)
    x = torch.empty(x_rows * ldx, dtype=torch.bfloat16, device="cuda").view(x_rows, ldx)
    at = torch.from_numpy(index).cuda()
    for i in range(rows):      # rows picked twice: the same values in the reference
        if 0 <= index[i] < x_rows:
            x[int(index[i]), :b.x.shape[1]] = b.x[i]
    live = b.live()
    b.x[live] = x[at[live]][:, :b.x.shape[1]]
    ref_f, (gate, u) = b.forward64(), kept(b)
    ref_b = b.backward64(gate.double(), u.double())
    small = b.x, b.index, b.x_rows
    b.x, b.index, b.x_rows = x, at.int(), x_rows
    g2, u2, y = b.forward()
    got = b.backward(gate, u)
    b.x, b.index, b.x_rows = small
    for n, t in (("gate", g2), ("up", u2), ("y", y)):
        assert R.worst(t, *ref_f[n]) <= 1.0, n
    for n, (v, e) in ref_b.items():
        assert R.worst(got[n].reshape(v.shape), v, e) <= 1.0, n


@pytest.mark.parametrize("rows,d,f", [(3, 8, 2 ** 22), (3, 2 ** 22, 8), (70, 2 ** 20 + 3, 5), (70, 5, 2 ** 20 + 3)])
def test_widths(rows, d, f):
    say("widths", rows, d, f)
    b = R.Block([0, rows], rows, d, f, "bf16", "gelu", seed=30)
    check_forward(b)
    check_backward(b, *kept(b), dw_dtype="bf16")


@pytest.mark.parametrize("rows", [5, 4096, 30000])
def test_4096_groups(rows):
    say("4096 groups", rows)
    rng = np.random.default_rng(rows)
    b = R.Block(cut(rng, rows, 4096), rows, 16, 24, "f16", "silu", seed=31)
    check_forward(b)
    check_backward(b, *kept(b))
    o = Operands(32, rows, 24, 40, 4096, True)
    check(o, cut(rng, rows, 4096), "bf16", "silu")


def test_groups_that_share_weights():
    """w_stride = d_stride = 0."""
    say("shared weights")
    for rows, d, f in ((40, 24, 40), (900, 136, 264)):
        one = R.Block([0, rows], rows, d, f, seed=33)
        b = R.Block([0, rows // 4, rows], rows, d, f, seed=33)
        b.x, b.dy = one.x, one.dy
        for n, r in (("wg", f), ("wu", f), ("wd", d)):
            setattr(b, n, getattr(one, n).repeat(2, 1))     # the reference's copies
        gate, u, y = b.out(rows, f), b.out(rows, f), b.out(rows, d)
        p = b.struct(gate, u, y)
        p.w_gate, p.w_up, p.w_down, p.w_stride, p.d_stride = one.wg.data_ptr(), one.wu.data_ptr(), one.wd.data_ptr(), 0, 0
        R.run_forward(p)
        for n, t in (("gate", gate), ("up", u), ("y", y)):
            assert R.worst(t, *b.forward64()[n]) <= 1.0, n
        dx, dwg, dwu, dwd = b.out(rows, d), b.out(2 * f, d, "f32"), b.out(2 * f, d, "f32"), b.out(2 * d, f, "f32")
        R.run_backward(p, R.grad_struct(b, dx, dwg, dwu, dwd))
        for n, t in (("dx", dx), ("dwg", dwg), ("dwu", dwu), ("dwd", dwd)):
            v, e = b.backward64(gate.double(), u.double())[n]
            assert R.worst(t.reshape(v.shape), v, e) <= 1.0, n


def test_millions_of_columns():
    say("columns")
    for m in (1, 20):
        check(Operands(34, m, 5000011, 16, 1, False), [0, m], "bf16", None)
    check(Operands(35, 2, 1000003, 32, 1, True), [0, 2], "f32", "silu")


def test_millions_of_rows():
    say("rows")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(36)
    for rows, cols in ((20000003, 1), (5000001, 9)):
        x = torch.randn(rows, cols, device="cuda", generator=gen).bfloat16()
        q, s = quantise(x)
        same((q, s), R.quantise64(x))
        q = q.contiguous()
        y = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
        p = G.W8Dequant(rows, cols, G.BF16, q.data_ptr(), cols, s.data_ptr(), y.data_ptr(), cols)
        G.check(G.lib().ggemm_w8_dequantize(C.byref(p), stream()), "ggemm_w8_dequantize")
        assert torch.equal(y, (q.float() * s[:, None]).bfloat16())
    m, n, k = 3000017, 8, 16
    check(Operands(37, m, n, k, 3, False), [0, 5, 2000000, m], "bf16", None)
