"""Rows of the gated block (include/ggemm_glu.h) whose index names none, with weights that are not finite: zeros all the same, in every
kernel that computes them, also from a captured graph."""
import ctypes as C

import pytest
import torch

import ggemm as G
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


def test_captured_with_an_index_that_changes():
    """Forward and backward in one graph; index, offsets and inputs are other ones at every replay, eager calls in between."""
    say("graph")
    rows, d, f = 700, 136, 264
    b = block(rows, [200, 450, rows], d, f, "bf16", "silu", 0.3)
    y, gate, u, dx = b.out(rows, d), b.out(rows, f), b.out(rows, f), b.out(rows, d)
    dwg, dwu, dwd = b.out(3 * f, d, "f32"), b.out(3 * f, d, "f32"), b.out(3 * d, f, "f32")
    out = (y, gate, u, dx, dwg, dwu, dwd)
    p, q = b.struct(gate, u, y), R.grad_struct(b, dx, dwg, dwu, dwd)
    n1, n2 = G.lib().ggemm_glu_workspace(C.byref(p)), G.lib().ggemm_glu_backward_workspace(C.byref(p), C.byref(q))
    ws = torch.empty(max(n1, n2), dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        G.check(G.lib().ggemm_glu(C.byref(p), ws.data_ptr(), n1, s), "ggemm_glu")
        G.check(G.lib().ggemm_glu_backward(C.byref(p), C.byref(q), ws.data_ptr(), n2, s), "ggemm_glu_backward")
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    gen = torch.Generator()
    for i in range(5):
        gen.manual_seed(i)
        b.index.copy_(torch.randint(-rows // 4, rows + 20, (rows,), generator=gen).int())
        b.offs.copy_(torch.tensor([0, *sorted(torch.randint(0, rows + 1, (2,), generator=gen).tolist()), rows]).int())
        b.x[:, :d] = torch.randn(rows, d, device="cuda", generator=b.gen).to(b.x.dtype)
        for t in out:
            t.fill_(3.0)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for t in out:
            t.fill_(3.0)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(g, t) for g, t in zip(got, out)), i
        dead = ~b.live()
        assert bool(dead.any()) and all(bool((t[:rows][dead] == 0).all()) for t in (y, gate, u, dx))
        b.offsets = b.offs.tolist()
        want = b.forward64()
        for n, t in (("gate", gate), ("up", u), ("y", y)):
            assert R.worst(t, *want[n]) <= 1.0, (i, n)
        for n, (v, e) in b.backward64(gate.double(), u.double()).items():
            assert R.worst({"dx": dx, "dwg": dwg, "dwu": dwu, "dwd": dwd}[n].reshape(v.shape), v, e) <= 1.0, (i, n)
