"""Rows of the gated block (include/ggemm_glu.h) whose index names none, with weights that are not finite: zeros all the same, in every
kernel that computes them."""
import pytest
import torch

import glu_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu

# rows, groups' ends, d, f: the kernel for few rows; tiles of 64, 128 and 256 rows, whole and partial
SIZES = [(12, [5, 12], 40, 24), (200, [90, 200], 72, 136), (700, [200, 700], 328, 264), (8192, [8192], 520, 2048), (8192, [4096, 8192], 2048, 264)]


def block(rows, ends, d, f, dtype, act, dead):
    gen = torch.Generator()
    gen.manual_seed(rows + d)
    index = torch.randint(0, rows, (rows,), generator=gen)
    index[torch.rand(rows, generator=gen) < dead] = -1
    index[rows // 2] = rows if dead else 0
    b = R.Block([0, *ends], rows, d, f, dtype, act, index.numpy(), rows, seed=rows + f)
    return b


def spoil(b, values):
    """Every matrix gets one of the values in each row that it has, at columns that differ."""
    for n, t in (("wg", b.wg), ("wu", b.wu), ("wd", b.wd)):
        cols = b.f if n == "wd" else b.d
        for i, v in enumerate(values):
            r = torch.arange(i, t.shape[0], len(values), device="cuda")
            t[r, (r * 7 + i) % cols] = v


@pytest.mark.parametrize("rows,ends,d,f", SIZES)
@pytest.mark.parametrize("dtype,act", [("bf16", "silu"), ("f16", "gelu"), ("bf16", "gelu_tanh")])
def test_dead_rows_with_weights_that_are_not_finite(rows, ends, d, f, dtype, act):
    say("dead rows, infinite weights", rows, d, f, dtype, act)
    b = block(rows, ends, d, f, dtype, act, 0.3)
    spoil(b, [float("inf"), float("nan"), float("-inf")])
    dead = ~b.live()
    gate, u, y = b.forward()
    for n, t in (("gate", gate), ("up", u), ("y", y)):
        assert bool((t[:rows][dead] == 0).all()), n
        assert not bool(torch.isfinite(t[:rows][~dead]).all()), n     # the weights do reach the others
    y2 = b.forward(keep=False)[2]
    assert bool((y2[:rows][dead] == 0).all())
    got = b.backward(gate, u)
    assert bool((got["dx"][:rows][dead] == 0).all())


def test_no_live_row_at_all():
    """Then the weights' gradients are zeros too."""
    say("all dead")
    for rows, ends, d, f in SIZES:
        b = block(rows, ends, d, f, "bf16", "silu", 1.1)
        spoil(b, [float("inf"), float("nan")])
        gate, u, y = b.forward()
        got = b.backward(gate, u)
        for n, t in (("gate", gate), ("up", u), ("y", y), *got.items()):
            assert bool((t[:rows] == 0).all() if n in ("gate", "up", "y", "dx") else (t == 0).all()), n
