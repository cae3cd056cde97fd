"""The gated feed-forward block and its gradients (include/ggemm_glu.h) against 64-bit forms, every entry within the
bound that the roundings of its own sums give (glu_ref.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

import ggemm as G
import glu_ref as R
from gpu_util import say

pytestmark = pytest.mark.gpu


def cut(rng, rows, groups, empty=0.3):
    """Ascending offsets, some groups without rows."""
    c = np.sort(rng.integers(0, rows + 1, max(groups - 1, 0)))
    for i in range(1, len(c)):
        if rng.random() < empty:
            c[i] = c[i - 1]
    return [0, *map(int, c), rows]


def check_forward(b, keep=True, pad=0):
    gate, u, y = b.forward(keep, pad)
    want, cov = b.forward64(), b.covered()
    for n, t, w in (("gate", gate, b.f), ("up", u, b.f), ("y", y, b.d)):
        if t is None:
            continue
        t = t[:b.rows]
        bad = R.worst(t[cov, :w], want[n][0][cov], want[n][1][cov])
        assert bad <= 1.0, (n, bad)
        assert bool((t[~cov] == 7.0).all()) and bool((t[:, w:] == 7.0).all()), n    # rows of no group, the padding of rows
    return gate, u, y


def kept(b, gen_seed=5):
    """Kept projections of a backward call: random ones of the forward pass's size."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(gen_seed)
    new = lambda: torch.randn(max(b.rows, 1), b.f, device="cuda", generator=gen).to(R.TORCH[b.dtype])   # noqa: E731
    return new(), new()


def check_backward(b, gate, u, dw_dtype="f32", beta=0.0, pad=0, want=("dx", "dw", "dwd")):
    dw0 = None
    if beta:
        gen = torch.Generator(device="cuda")
        gen.manual_seed(9)
        dw0 = {n: torch.randn(b.E, r, c, device="cuda", generator=gen).to(R.TORCH[dw_dtype]).double()
               for n, r, c in (("dwg", b.f, b.d), ("dwu", b.f, b.d), ("dwd", b.d, b.f))}
    got = b.backward(gate, u, want, dw_dtype, beta, dw0, pad)
    ref = b.backward64(gate[:b.rows].double(), u[:b.rows].double(), dw_dtype, beta, dw0)
    cov = b.covered()
    for n, (v, e) in ref.items():
        if got[n] is None:
            continue
        w = v.shape[-1]
        if n == "dx":
            t = got[n][:b.rows]
            bad = R.worst(t[cov, :w], v[cov], e[cov])
            assert bool((t[~cov] == 7.0).all()), n
        else:
            t = got[n]
            bad = R.worst(t[:, :w].reshape(v.shape), v, e)
        assert bad <= 1.0, (n, bad)
        if beta == 0.0 or n == "dx":
            assert bool((got[n][:, w:] == 7.0).all()), n
    return got


def index_for(rng, rows, x_rows, dead=0.15):
    i = rng.integers(0, max(x_rows, 1), rows).astype(np.int64)
    i[rng.random(rows) < dead] = -1
    if rows > 2:
        i[rows // 2] = x_rows            # just past the last row of x
    return i


SHAPES = [  # rows, groups, d, f
    (1, 1, 8, 8), (1, 1, 1, 1), (3, 1, 7, 5), (1, 3, 64, 64), (16, 1, 128, 64), (17, 2, 65, 63), (33, 4, 96, 33),
    (5, 9, 200, 72), (64, 1, 128, 256), (100, 3, 129, 257), (130, 1, 333, 191), (257, 2, 256, 128), (300, 5, 100, 300),
    (700, 70, 40, 48), (600, 1, 512, 640), (513, 3, 264, 1000),
]


@pytest.mark.parametrize("rows,groups,d,f", SHAPES)
@pytest.mark.parametrize("dtype,act", [("bf16", "silu"), ("f16", "gelu"), ("bf16", "gelu_tanh"), ("f16", "silu")])
def test_block(rows, groups, d, f, dtype, act):
    say("block", rows, groups, d, f, dtype, act)
    rng = np.random.default_rng(rows + 3 * d + 7 * f)
    b = R.Block(cut(rng, rows, groups), rows, d, f, dtype, act, seed=rows + d)
    check_forward(b)
    gate, u = kept(b)
    check_backward(b, gate, u)
    b = R.Block(cut(rng, rows, groups), rows, d, f, dtype, act, index_for(rng, rows, 2 * rows), 2 * rows, seed=rows + f, pad=8)
    check_forward(b, keep=rows % 2 == 0, pad=3)
    check_backward(b, gate, u, dw_dtype=dtype, pad=5)


LARGE = [  # rows, groups, d, f: tiles of the largest kind, several rounds of them, long inner dimensions
    (5000, 3, 1024, 1536), (4100, 1, 520, 2056), (9000, 8, 768, 1000), (40, 1, 4096, 8200), (2048, 40, 512, 768), (20000, 2, 264, 520),
]


@pytest.mark.parametrize("rows,groups,d,f", LARGE)
@pytest.mark.parametrize("gather", [False, True])
def test_large(rows, groups, d, f, gather):
    say("large", rows, groups, d, f, gather)
    rng = np.random.default_rng(rows)
    index = index_for(rng, rows, rows // 2 + 1) if gather else None
    b = R.Block(cut(rng, rows, groups, 0.1), rows, d, f, "bf16", "silu", index, rows // 2 + 1, seed=rows)
    check_forward(b)
    gate, u = kept(b)
    check_backward(b, gate, u, dw_dtype="bf16" if gather else "f32")


@pytest.mark.parametrize("rows,groups,d,f", [(8192, 1, 4096, 2048), (8200, 3, 4096, 2056), (3000, 2, 1500, 1000)])
@pytest.mark.parametrize("dtype,act", [("f16", "gelu_tanh"), ("bf16", "gelu")])
def test_every_product_in_large_tiles(rows, groups, d, f, dtype, act):
    say("large tiles", rows, groups, d, f, dtype, act)
    rng = np.random.default_rng(rows)
    b = R.Block(cut(rng, rows, groups, 0.0), rows, d, f, dtype, act, seed=22)
    check_forward(b)
    gate, u = kept(b)
    # gradients of 1 / 16, so that sums over 8192 rows of f16 factors stay within its range
    b.dy *= 0.0625
    check_backward(b, gate, u, dw_dtype=dtype)


def test_rows_of_no_group_are_left_alone():
    say("rows of no group")
    b = R.Block([3, 20, 20, 300], 350, 72, 136, seed=3)      # rows 0 .. 2 and 300 .. 349
    gate, u, _ = check_forward(b)
    check_backward(b, gate, u)


@pytest.mark.parametrize("offsets", [[0, 500, 40], [-5, 10, 40], [0, 2 ** 31 - 1, 2 ** 31 - 1], [30, 10, 40]])
def test_offsets_out_of_range(offsets):
    """Clamped: only the rows that the clamped offsets name may be touched."""
    say("offsets", offsets)
    b = R.Block(offsets, 40, 64, 72, seed=4)
    if offsets == [0, 500, 40] or offsets == [30, 10, 40]:   # a descending pair names no rows; rows of both groups clash nowhere
        gate, u, y = b.forward()
        cov = b.covered()
        assert bool((y[~cov] == 7.0).all()) and bool((gate[~cov] == 7.0).all())
        if offsets[0] == 30:
            want = b.forward64()["y"]
            assert R.worst(y[cov], want[0][cov], want[1][cov]) <= 1.0
    else:
        gate, u, _ = check_forward(b)
        check_backward(b, gate, u)


def test_no_offsets_and_no_rows():
    say("no offsets")
    b = R.Block([0, 70], 70, 48, 80, seed=5)
    y0 = b.forward()[2]
    y1 = b.forward(keep=False, offsets=None)[2]
    assert torch.equal(y0, y1)
    empty = R.Block([0, 0, 0], 0, 48, 80, seed=6)
    gate, u = kept(empty)
    for beta in (0.0, 0.5):
        check_backward(empty, gate, u, beta=beta)
    none = R.Block([0, 0, 0, 0], 30, 48, 80, seed=6)         # rows, but of no group
    gate, u = kept(none)
    check_forward(none)
    check_backward(none, gate, u, beta=1.0)


@pytest.mark.parametrize("beta", [1.0, -0.5])
@pytest.mark.parametrize("dw_dtype", ["f32", "bf16", "f16"])
def test_gradients_accumulate(beta, dw_dtype):
    say("beta", beta, dw_dtype)
    rng = np.random.default_rng(8)
    for rows, groups, d, f in ((90, 3, 72, 40), (600, 2, 520, 264)):
        b = R.Block(cut(rng, rows, groups), rows, d, f, "bf16", "silu", seed=8)
        check_backward(b, *kept(b), dw_dtype=dw_dtype, beta=beta)


def test_gradients_by_themselves():
    say("some gradients")
    b = R.Block([0, 40, 200], 200, 72, 136, seed=10)
    gate, u = kept(b)
    full = check_backward(b, gate, u)
    for want in (("dx",), ("dw",), ("dwd",), ("dx", "dwd"), ()):
        part = check_backward(b, gate, u, want=want)
        for n, t in part.items():
            assert t is None or torch.equal(t, full[n]), n


def test_dead_rows_hold_anything():
    """NaN and Inf in rows of x that no index names, in dy, gate and up of rows whose index names none: nothing comes of it."""
    say("dead rows")
    rng = np.random.default_rng(11)
    for rows, d, f in ((70, 40, 72), (900, 264, 520)):
        index = index_for(rng, rows, rows, 0.4)
        used = np.zeros(rows + 1, dtype=bool)
        used[index[(index >= 0) & (index < rows)]] = True
        b = R.Block([0, rows // 3, rows], rows, d, f, "bf16", "gelu", index, rows, seed=12)
        b.x[torch.from_numpy(~used[:rows]).cuda()] = float("inf")
        gate, u = kept(b)
        dead = ~b.live()
        for t, v in ((gate, float("nan")), (u, float("-inf")), (b.dy, float("nan"))):
            t[:rows][dead] = v
        check_forward(b)
        got = check_backward(b, gate, u)
        assert bool((got["dx"][:rows][dead] == 0).all())


def test_no_row_of_x_exists():
    say("no x")
    b = R.Block([0, 3, 9], 9, 24, 40, index=[-1, 0, 5, 3, -7, 2 ** 31 - 1, 1, 2, -2 ** 31], x_rows=0, seed=13)
    p = b.struct(None, None, y := b.out(9, 24))
    p.x = None
    R.run_forward(p)
    assert bool((y == 0).all())
    got = b.backward(*kept(b))
    assert all(bool((t == 0).all()) for t in got.values())


def test_nonfinite_values_stay_in_their_rows():
    """A NaN in a row of x reaches that row of y and no other; an Inf weight the columns that it feeds."""
    say("nonfinite")
    for rows, d, f in ((50, 72, 136), (520, 264, 264)):
        b = R.Block([0, rows // 2, rows], rows, d, f, seed=14)
        b.x[3, 5] = float("nan")
        b.x[rows - 1, d - 1] = float("inf")
        gate, u, y = b.forward()
        bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        bad[3] = bad[rows - 1] = True
        assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all())
        assert bool(torch.isfinite(gate[~bad]).all())


def test_gradients_against_differences():
    """Along a direction v of each input: (L(+t v) - L(-t v)) / 2 t of the 64-bit form, L = sum dy y; its own error is of
    order t^2 times third derivatives of order one, 1e-8 relative at t = 1e-4.  The kernel's gradient, at the
    kept projections (rounded: their effect on the slope, at most UNIT |a| (|a''| + ..) an entry, enters with random signs), is
    off by a part of 2^-7 of the norms' product over the square root of the entries; 2^-6 of it is allowed without that root."""
    say("differences")
    for dtype, act in (("bf16", "silu"), ("f16", "gelu"), ("f16", "gelu_tanh")):
        b = R.Block([0, 30, 30, 90], 90, 48, 72, dtype, act, seed=15)
        gate, u, _ = b.forward()
        got = b.backward(gate, u)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(1)
        base = {"x": b.x64(), **{n: getattr(b, n)[:, :c].double() for n, c in (("wg", b.d), ("wu", b.d), ("wd", b.f))}}
        dy = b.dy[:, :b.d].double()

        def loss(t):
            tot = 0.0
            for g, r in b.spans():
                f, d = b.f, b.d
                a, c = R.mm(t["x"][r], t["wg"][g * f:(g + 1) * f].t()), R.mm(t["x"][r], t["wu"][g * f:(g + 1) * f].t())
                tot = tot + float((R.mm(a * R.act_parts(a, act)[0] * c, t["wd"][g * d:(g + 1) * d].t()) * dy[r]).sum())
            return tot
        for n, grad in (("x", "dx"), ("wg", "dwg"), ("wu", "dwu"), ("wd", "dwd")):
            v = torch.randn(base[n].shape, device="cuda", generator=gen, dtype=torch.float64)
            t = 1e-4
            slope = (loss({**base, n: base[n] + t * v}) - loss({**base, n: base[n] - t * v})) / (2 * t)
            mine = float((got[grad].double()[:v.shape[0], :v.shape[1]] * v).sum())
            assert abs(slope - mine) <= 2.0 ** -6 * float(got[grad].double().norm() * v.norm()), (dtype, act, n, slope, mine)


def test_same_bits_every_time():
    say("same bits")
    rng = np.random.default_rng(16)
    for rows, groups, d, f in ((3, 1, 4096, 512), (300, 4, 520, 264), (3000, 2, 520, 1032)):
        b = R.Block(cut(rng, rows, groups), rows, d, f, seed=17)
        first = b.forward()
        grads = b.backward(first[0], first[1])
        for _ in range(2):
            again = b.forward()
            assert all(torch.equal(x, y) for x, y in zip(first, again))
            g2 = b.backward(first[0], first[1])
            assert all(torch.equal(grads[n], g2[n]) for n in grads)


def test_other_streams_at_once():
    """Two calls on two streams, each with a workspace of its own."""
    say("streams")
    blocks = [R.Block([0, 150, 400], 400, 264, 520, seed=s) for s in (1, 2)]
    want = [b.forward() for b in blocks]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    got = []
    for b, s in zip(blocks, streams):
        with torch.cuda.stream(s):
            got.append([b.forward() for _ in range(4)])
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(x, y) for r in runs for x, y in zip(w, r))


def test_captured_into_a_graph():
    """Forward and backward captured together; replayed with new inputs, eager work in between, checked every time."""
    say("graph")
    b = R.Block([0, 100, 260], 260, 136, 264, seed=18)
    y, gate, u = b.out(260, 136), b.out(260, 264), b.out(260, 264)
    grads = [b.out(260, 136), b.out(2 * 264, 136, "f32"), b.out(2 * 264, 136, "f32"), b.out(2 * 136, 264, "f32")]
    p, p2 = b.struct(gate, u, y), b.struct(gate, u, None)
    q = R.grad_struct(b, *grads)
    lib = G.lib()
    n1, n2 = lib.ggemm_glu_workspace(C.byref(p)), lib.ggemm_glu_backward_workspace(C.byref(p2), C.byref(q))
    ws = torch.empty(max(n1, n2), dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        G.check(lib.ggemm_glu(C.byref(p), ws.data_ptr(), n1, s), "ggemm_glu")
        G.check(lib.ggemm_glu_backward(C.byref(p2), C.byref(q), ws.data_ptr(), n2, s), "ggemm_glu_backward")
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        b.x[:, :136] = torch.randn(260, 136, device="cuda", generator=b.gen).to(b.x.dtype)
        for t in (y, gate, u, *grads):
            t.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, gate, u, *grads)]
        g1, u1, y1 = b.forward()
        e = b.backward(g1, u1)
        for t, w in zip(got, (y1, g1, u1, e["dx"], e["dwg"], e["dwu"], e["dwd"])):
            assert torch.equal(t, w), i


def test_large_values():
    """Projections far out: the activation is 0 or the identity there, and no slope is NaN."""
    say("large values")
    for act in ("silu", "gelu", "gelu_tanh"):
        b = R.Block([0, 64], 64, 64, 64, "bf16", act, seed=19)
        gate, u = kept(b)
        gate[:, ::3] *= 1e18
        gate[:, 1::3] *= -1e30
        u.fill_(1.0)
        got = b.backward(gate, u, want=("dx", "dw"))
        assert bool(torch.isfinite(got["dx"]).all()) and bool(torch.isfinite(got["dwg"]).all())
        want = b.backward64(gate.double().clamp(-1e4, 1e4), u.double())   # the same slopes
        assert R.worst(got["dwg"].view(1, 64, 64), want["dwg"][0], want["dwg"][1] + 1e-3 * want["dwg"][0].abs()) <= 1.0


def test_long_rows():
    """Rows of x, dy and the weights 2^23 bytes apart: offsets past 32 bits from the 512th row on, and past 31 within a tile's."""
    say("long rows")
    for rows, d, f in ((300, 40, 24), (9, 24, 300), (600, 40, 40)):
        b = R.Block([0, rows], rows, d, f, seed=20)
        for n in ("x", "dy", "wg", "wu", "wd"):
            t = getattr(b, n)
            wide = torch.empty(t.shape[0], G.GLU_MAX_LD, dtype=t.dtype, device="cuda")
            wide[:, :t.shape[1]] = t
            setattr(b, n, wide)
        check_forward(b)
        check_backward(b, *kept(b))
        del b


def test_offsets_that_name_rows_many_times():
    """Not ascending: results of rows named twice are anybody's, but nothing outside the results is touched and the calls end."""
    say("offsets over and over")
    for rows, groups in ((40, 9), (3000, 201)):
        b = R.Block([0 if g % 2 == 0 else rows for g in range(groups + 1)], rows, 16, 24, seed=21)
        y, gate, u, dx = (torch.full((rows + 64, w), 7.0, dtype=torch.bfloat16, device="cuda") for w in (16, 24, 24, 16))
        R.run_forward(b.struct(gate[32:], u[32:], y[32:]))
        dwg, dwu, dwd = b.out(groups * 24, 16, "f32"), b.out(groups * 24, 16, "f32"), b.out(groups * 16, 24, "f32")
        R.run_backward(b.struct(gate[32:], u[32:], None), R.grad_struct(b, dx[32:], dwg, dwu, dwd))
        torch.cuda.synchronize()
        for t in (y, gate, u, dx):
            assert bool((t[:32] == 7.0).all()) and bool((t[rows + 32:] == 7.0).all())
